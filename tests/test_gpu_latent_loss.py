"""The softmax loss over the catalogue (blp.latent.softmax_loss*) against its definition in 64 bits.

Bounds, from the operator's own roundings (u = 2^-23, a 32-bit step: products are added inside the matrix
instruction, whose inner rounding may truncate):
  a score         dz_i  = (k + 4) u S_i, S_i = max_j scale sum |x w|
  log-sum-exp     dz_i + (depth + 8) u + 4 u |lse|     depth: additions in a chain of partial sums
  a probability   relative r_i = 2 dz_i + (depth + 16) u + 4 u (S_i + |lse_i|)
  dS              h |dS| more for its rounding to the type (h half a step; halves hold 2^-14 less than
                  2^-25 of the largest row gradient)
  a gradient      scale sum (error of dS) |w| + (n + 8) u sum |dS w|, then h of the result
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -23


def _torch():
    return pytest.importorskip("torch")


def _half_step(t):
    import torch

    return torch.finfo(t).eps / 2


def make(m, n, k, dtype, seed=0, ignored=0.0, spread=3.0, scale=1.0, device="cuda"):
    import torch

    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k, generator=g).to(dtype)
    w = (torch.randn(n, k, generator=g) * (spread / scale / k ** 0.5)).to(dtype)
    t = torch.randint(0, n, (m,), generator=g)
    t[torch.rand(m, generator=g) < ignored] = -1
    return x.to(device), w.to(device), t.to(device)


def reference(x, w, t, scale, g=None, reduction="mean"):
    """-> dict of the definition's values and error bounds, on the inputs' device in 64 bits."""
    import torch

    X, W = x.double(), w.double()
    n, k = W.shape
    ok = (t >= 0) & (t < n)
    X = torch.where(ok[:, None], X, 0.0)
    at = t.clamp(0, n - 1).long()[:, None]
    z = scale * (X @ W.t().contiguous())
    S = abs(scale) * (X.abs() @ W.abs().t().contiguous()).amax(1)
    lse = torch.logsumexp(z, 1)
    loss = torch.where(ok, lse - z.gather(1, at)[:, 0], 0.0)
    depth = 64 + n / 64  # within a tile, then along the tiles' pairs
    dz = (k + 4) * U * S
    bl = 2 * dz + (depth + 8) * U + 8 * U * (lse.abs() + S)
    count = max(int(ok.sum()), 1)
    gi = torch.ones_like(lse) if g is None else g.double().expand(len(lse))
    if reduction == "mean":
        gi = gi / count
    gi = torch.where(ok, gi, 0.0)
    p = torch.exp(z - lse[:, None])
    hit = torch.zeros_like(p).scatter_(1, at, 1.0)
    d = gi[:, None] * (p - hit)
    h = _half_step(x.dtype)
    r = 2 * dz + (depth + 16) * U + 4 * U * (S + lse.abs())
    # bound on dS: the probability's, a 32-bit step of the difference, the rounding to the type
    e = gi.abs()[:, None] * (p * r[:, None] + 2 * U) + h * d.abs()
    if x.dtype == torch.float16:
        e = e + gi.abs().max() * 2.0 ** -39
    out = {"loss": loss, "b_loss": bl, "ok": ok, "count": count, "lse": lse}
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    mm = lambda a, b: a @ b.contiguous()
    out["dx"] = scale * mm(d, W)
    out["b_dx"] = abs(scale) * (mm(e, W.abs()) + (n + 8) * U * mm(d.abs(), W.abs()))
    out["dw"] = scale * mm(d.t(), X)
    out["b_dw"] = abs(scale) * (mm(e.t(), X.abs()) + (len(lse) + 8) * U * mm(d.t().abs(), X.abs()))
    for q in ("dx", "dw"):
        out["b_" + q] = out["b_" + q] * (1 + 2 * h) + h * out[q].abs() + tiny
    return out


def near(got, want, bound):
    import torch

    assert tuple(got.shape) == tuple(want.shape)
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), "off by %.3g more than %.3g" % (float(off.max()), float(bound.flatten()[off.argmax()]))
    assert bool(torch.isfinite(got).all())


SIZES = [(1, 1, 1), (1, 7, 3), (2, 100, 50), (31, 33, 8), (32, 257, 64), (33, 64, 65), (130, 1000, 64), (257, 513, 72),
         (64, 5003, 128), (300, 300, 200), (700, 129, 24)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_loss_and_gradients(gpu, m, n, k, dtype):
    torch = _torch()
    from blp import latent

    x, w, t = make(m, n, k, getattr(torch, dtype), seed=m + n, ignored=0.2 if m > 5 else 0.0, scale=1.5)
    ref = reference(x, w, t, 1.5)
    loss = latent.softmax_loss(x, w, t, scale=1.5, reduction="none")
    near(loss, ref["loss"], ref["b_loss"])
    total, dx, dw = latent.softmax_loss_grad(x, w, t, scale=1.5)
    near(total, ref["loss"].sum() / ref["count"], ref["b_loss"].mean() * m / ref["count"] + U * abs(float(total)))
    near(dx, ref["dx"], ref["b_dx"])
    near(dw, ref["dw"], ref["b_dw"])
    assert dx.dtype == x.dtype and dw.dtype == w.dtype and total.dtype == torch.float32


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", [(2100, 3000, 64), (600, 9001, 328), (1500, 2500, 1000)])
def test_large_tiles(gpu, m, n, k, dtype):
    torch = _torch()
    from blp import latent

    x, w, t = make(m, n, k, getattr(torch, dtype), seed=k, ignored=0.1)
    ref = reference(x, w, t, 1.0)
    total, dx, dw = latent.softmax_loss_grad(x, w, t)
    near(total, ref["loss"].sum() / ref["count"], ref["b_loss"].mean() * m / ref["count"] + U * abs(float(total)))
    near(dx, ref["dx"], ref["b_dx"])
    near(dw, ref["dw"], ref["b_dw"])


@pytest.mark.parametrize("dtype,m,n,k", [("float32", 12000, 24011, 20), ("float32", 9000, 24011, 72), ("bfloat16", 16000, 20011, 136)])
def test_pieces_of_the_catalogue(gpu, dtype, m, n, k):
    """More scores than one workspace piece holds (256 MiB: 134M halves, 45M floats of three halves), and as many where
    nothing is kept."""
    torch = _torch()
    from blp import latent

    x, w, t = make(m, n, k, getattr(torch, dtype), seed=3, ignored=0.02)
    ref = reference(x, w, t, 1.0)
    total, dx, dw = latent.softmax_loss_grad(x, w, t, reduction="sum")
    near(dx.double() / ref["count"], ref["dx"], ref["b_dx"])
    near(dw.double() / ref["count"], ref["dw"], ref["b_dw"])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_autograd_gradients_per_row(gpu, dtype):
    """reduction none: every row's own gradient, of both signs and very different sizes, zero among them."""
    torch = _torch()
    from blp import latent

    x, w, t = make(140, 700, 56, getattr(torch, dtype), seed=9, ignored=0.1)
    g = torch.logspace(-4, 3, 140, device="cuda") * torch.where(torch.arange(140, device="cuda") % 2 == 0, 1.0, -1.0)
    g[7] = 0.0
    ref = reference(x, w, t, 0.75, g, "none")
    x.requires_grad_(True)
    w.requires_grad_(True)
    loss = latent.softmax_loss(x, w, t, scale=0.75, reduction="none")
    dx, dw = torch.autograd.grad(loss, (x, w), g)
    near(dx, ref["dx"], ref["b_dx"])
    near(dw, ref["dw"], ref["b_dw"])
    # one of the two only
    (dx2,) = torch.autograd.grad(latent.softmax_loss(x, w.detach(), t, scale=0.75, reduction="none"), (x,), g)
    assert torch.equal(dx, dx2)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", [(300, 700, 30), (300, 700, 64), (131, 1000, 96), (131, 1000, 128), (131, 1000, 160)])
def test_scales_and_row_gradients(gpu, m, n, k, dtype):
    """Negative scales, a scale of 0 (every business equally likely), gradients of their own for the rows."""
    torch = _torch()
    from blp import latent

    x, w, t = make(m, n, k, getattr(torch, dtype), seed=k, ignored=0.1)
    g = torch.linspace(-2, 3, m, device="cuda")
    x.requires_grad_(True)
    w.requires_grad_(True)
    for scale in (-0.7, 0.0, 1e-30):
        ref = reference(x.detach(), w.detach(), t, scale, g, "none")
        loss = latent.softmax_loss(x, w, t, scale=scale, reduction="none")
        near(loss.detach(), ref["loss"], ref["b_loss"])
        dx, dw = torch.autograd.grad(loss, (x, w), g)
        near(dx, ref["dx"], ref["b_dx"])
        near(dw, ref["dw"], ref["b_dw"])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_confident_rows(gpu, dtype):
    """Targets that take nearly all of the softmax, and targets far below the rest: 1 - p keeps its digits, and the reference
    score that the sums start from lies far from the maximum."""
    torch = _torch()
    from blp import latent

    for k in (64, 200):
        g = torch.Generator().manual_seed(k)
        w = torch.randn(900, k, generator=g)
        w = (w / w.norm(dim=1, keepdim=True)).to(getattr(torch, dtype)).cuda()
        t = torch.randint(0, 900, (64,), generator=g).cuda()
        x = w[t] * torch.tensor([12.0, 90.0, -60.0, 0.5], device="cuda").repeat(16)[:, None].to(w.dtype)
        ref = reference(x, w, t, 1.0)
        loss, dx, dw = latent.softmax_loss_grad(x, w, t)
        near(latent.softmax_loss(x, w, t, reduction="none"), ref["loss"], ref["b_loss"])
        near(dx, ref["dx"], ref["b_dx"])
        near(dw, ref["dw"], ref["b_dw"])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", [(70, 77, 40), (150, 700, 64), (1537, 3001, 33), (150, 700, 200), (70, 3001, 128)])
def test_catalogues_of_low_scores(gpu, m, n, k, dtype):
    """Every score far below zero, so exp(0 - lse) of the rows past the catalogue's end (zeros) is infinite in the type."""
    torch = _torch()
    from blp import latent

    dtype = getattr(torch, dtype)
    g = torch.Generator().manual_seed(k)
    x = (0.5 + torch.rand(m, k, generator=g)).to(dtype).cuda()
    w = (-(0.5 + torch.rand(n, k, generator=g)) * (200 / k)).to(dtype).cuda()
    t = torch.randint(0, n, (m,), generator=g).cuda()
    ref = reference(x, w, t, 1.0)
    total, dx, dw = latent.softmax_loss_grad(x, w, t)
    near(total, ref["loss"].sum() / ref["count"], ref["b_loss"].mean() * m / ref["count"] + U * abs(float(total)))
    near(dx, ref["dx"], ref["b_dx"])
    near(dw, ref["dw"], ref["b_dw"])
    lse = torch.logsumexp(x.double() @ w.double().t().contiguous(), 1).float()
    dx, dw = latent.softmax_loss_backward(torch.full((m,), 1 / m, device="cuda"), lse, None, x, w, t)
    assert dx.isfinite().all() and dw.isfinite().all()


def test_scores_that_rise_along_the_catalogue(gpu):
    """Sorted scores, over 300 in all: the running reference is overtaken again and again, by more than 2^60 at a time."""
    torch = _torch()
    from blp import latent

    for dtype in (torch.float32, torch.bfloat16):
        for k in (8, 200):
            for flip in (1, -1):
                w = torch.zeros(3000, k)
                w[:, 0] = torch.linspace(-150, 150, 3000) * flip
                x = torch.zeros(40, k)
                x[:, 0] = 1.0
                t = torch.arange(40) * 70
                x, w, t = x.to(dtype).cuda(), w.to(dtype).cuda(), t.cuda()
                ref = reference(x, w, t, 1.0)
                near(latent.softmax_loss(x, w, t, reduction="none"), ref["loss"], ref["b_loss"])


def test_autograd_in_a_capture_is_refused(gpu):
    torch = _torch()
    from blp import latent

    x, w, t = make(10, 30, 8, torch.float32)
    x.requires_grad_(True)
    latent.softmax_loss(x, w, t).backward()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="softmax_loss_grad"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            latent.softmax_loss(x, w, t)
    with pytest.raises(RuntimeError, match="lookup_grad"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            latent.lookup(x, t)
    torch.cuda.synchronize()
    assert torch.isfinite(latent.softmax_loss(x, w, t))


def test_against_differences(gpu):
    """The gradient against the loss's own differences, taken in 64 bits."""
    torch = _torch()
    from blp import latent

    x, w, t = make(9, 40, 6, torch.float32, seed=4)
    _, dx, dw = latent.softmax_loss_grad(x, w, t)

    def f(X, W):
        z = X @ W.t()
        return float((torch.logsumexp(z, 1) - z.gather(1, t[:, None])[:, 0]).mean())

    X, W, step = x.double().cpu(), w.double().cpu(), 1e-5
    t = t.cpu()
    for A, got in ((X, dx), (W, dw)):
        for i, j in ((0, 0), (3, 5), (8, 2)):
            keep = float(A[i, j])
            A[i, j] = keep + step
            hi = f(X, W)
            A[i, j] = keep - step
            lo = f(X, W)
            A[i, j] = keep
            # differences: third derivatives below 10 times step^2, and 1e-16 / step; 32-bit gradient
            assert abs((hi - lo) / (2 * step) - float(got[i, j])) < 10 * step ** 2 + 1e-10 + 1e-5 * float(got.abs().max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_more_rows_than_the_pairs_have_room_for(gpu, dtype):
    """391 tiles of the catalogue leave 782 pairs a row, of which 256 MiB hold 42,752 rows."""
    torch = _torch()
    from blp import latent

    m, n, k = 43100, 100000, 136
    x, w, t = make(m, n, k, getattr(torch, dtype), seed=11, ignored=0.1)
    at = torch.cat([torch.arange(0, 43), torch.arange(42700, 42800), torch.arange(m - 20, m), torch.arange(0, m, 997)]).cuda()
    ref = reference(x[at], w, t[at], 1.0)
    for tt in (t, t.to(torch.int32)):
        loss = latent.softmax_loss(x, w, tt, reduction="none")
        near(loss[at], ref["loss"], ref["b_loss"])
        total = latent.softmax_loss(x, w, tt, reduction="sum")
        assert abs(float(total) - float(loss.double().sum())) <= U * float(total)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_ignored_rows_hold_anything(gpu, dtype):
    torch = _torch()
    from blp import latent

    x, w, t = make(70, 300, 40, getattr(torch, dtype), seed=5)
    t[3], t[20], t[69] = -1, 300, -100
    for wide in (True, False):
        tt = t if wide else t.to(torch.int32)
        clean = latent.softmax_loss_grad(x, w, tt)
        bad = x.clone()
        bad[3], bad[20], bad[69] = float("nan"), float("inf"), float("-inf")
        got = latent.softmax_loss_grad(bad, w, tt)
        for a, b in zip(clean, got):
            assert torch.equal(a, b)
        loss = latent.softmax_loss(bad, w, tt, reduction="none")
        assert loss[3] == 0 and loss[20] == 0 and loss[69] == 0
        assert not got[1][3].any() and not got[1][20].any() and not got[1][69].any()


def test_no_row_left_and_no_rows(gpu):
    torch = _torch()
    from blp import latent

    x, w, t = make(40, 90, 16, torch.bfloat16, seed=6)
    loss, dx, dw = latent.softmax_loss_grad(x, w, torch.full_like(t, -1))
    assert float(loss) == 0 and not dx.any() and not dw.any()
    loss, dx, dw = latent.softmax_loss_grad(x[:0], w, t[:0])
    assert float(loss) == 0 and dx.shape == (0, 16) and not dw.any()
    assert latent.softmax_loss(x[:0], w, t[:0], reduction="none").shape == (0,)


def test_infinite_and_nan_scores_stay_in_their_rows(gpu):
    torch = _torch()
    from blp import latent

    x, w, t = make(20, 50, 8, torch.float32, seed=7)
    want = latent.softmax_loss(x, w, t, reduction="none")
    x[4, 0] = float("nan")
    x[5] = 1e30  # scores beyond 32 bits' exponents: infinite
    x[5, 0] = -1e38
    got = latent.softmax_loss(x, w, t, reduction="none")
    keep = [i for i in range(20) if i not in (4, 5)]
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[4])
    # large equal scores: the running maximum keeps exp in range
    big = torch.full((3, 4), 100.0, device="cuda")
    loss = latent.softmax_loss(big, torch.full((1000, 4), 50.0, device="cuda"), t[:3], reduction="none")
    np.testing.assert_allclose(loss.cpu().numpy(), np.log(1000.0), rtol=0, atol=20000 * 4 * U)


@pytest.mark.parametrize("k", [40, 200])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_infinite_and_nan_row_gradients_stay_in_their_rows(gpu, dtype, k):
    """Row gradients that are infinite or NaN: their rows of dx and all of dtable; the other rows of dx are those of
    row gradients of 0 in these places. Finite ones next to the largest float are taken as they are."""
    torch = _torch()
    from blp import latent

    x, w, t = make(150, 700, k, getattr(torch, dtype), seed=8)
    t[9] = -1
    g = torch.randn(150, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    lse = torch.logsumexp(x.float() @ w.float().t().contiguous(), 1)
    bad = {3: float("inf"), 9: float("nan"), 77: float("nan"), 149: float("-inf")}
    zeroed = g.clone()
    for i, v in bad.items():
        g[i], zeroed[i] = v, 0.0
    want, _ = latent.softmax_loss_backward(zeroed, lse, None, x, w, t)
    dx, dw = latent.softmax_loss_backward(g, lse, None, x, w, t)
    keep = [i for i in range(150) if i not in (3, 77, 149)]  # row 9 is ignored
    assert torch.equal(dx[keep], want[keep]) and want[keep].isfinite().all()
    assert not dx[[3, 77, 149]].isfinite().any() and not dw.isfinite().any()
    if dtype != "float16":  # whose gradients end at 65,504
        dw = latent.softmax_loss_backward(torch.full_like(g, 3.2e38), lse, None, x * 2.0 ** -20, w, t)[1]
        assert dw.isfinite().all() and dw.any()


def test_strided_and_unaligned_rows(gpu):
    """Slices of wider tensors: row strides, and starts that no 16-byte load can take."""
    torch = _torch()
    from blp import latent

    for dtype in (torch.bfloat16, torch.float32):
        X, W, t = make(50, 400, 96, dtype, seed=8)
        for lo, hi in ((0, 64), (8, 72), (1, 65), (3, 90)):
            x, w = X[:, lo:hi], W[:, lo:hi]
            a = latent.softmax_loss_grad(x, w, t)
            b = latent.softmax_loss_grad(x.contiguous(), w.contiguous(), t)
            for p, q in zip(a, b):
                assert torch.equal(p, q)


def test_same_result_twice_and_on_another_stream(gpu):
    torch = _torch()
    from blp import latent

    x, w, t = make(500, 3000, 64, torch.bfloat16, seed=10)
    a = latent.softmax_loss_grad(x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = latent.softmax_loss_grad(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_captured_and_replayed(gpu):
    """Two captured graphs and eager calls between their replays, on changing inputs."""
    torch = _torch()
    from blp import latent

    x, w, t = make(90, 500, 50, torch.bfloat16, seed=11)
    x2, w2, t2 = make(90, 500, 50, torch.bfloat16, seed=12)
    latent.softmax_loss_grad(x, w, t)
    torch.cuda.synchronize()
    graphs = []
    for args in ((x, w, t), (x2, w2, t2)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = latent.softmax_loss_grad(*args)
        graphs.append((g, out, args))
    for i in range(4):
        for g, out, args in graphs:
            fresh = make(90, 500, 50, torch.bfloat16, seed=20 + i)
            for dst, src in zip(args, fresh):
                dst.copy_(src)
            g.replay()
            want = latent.softmax_loss_grad(*fresh)
            for p, q in zip(out, want):
                assert torch.equal(p, q)


@pytest.mark.parametrize("dtype,m,n,k", [("bfloat16", 600, 3000, 200), ("float32", 600, 1300, 40), ("float32", 300, 900, 100),
                                         ("float16", 20, 3000, 500)])
def test_every_path_captured_and_replayed(gpu, dtype, m, n, k):
    """Forward and backward with row gradients, beside the step in one call; eager calls between the replays."""
    torch = _torch()
    from blp import latent

    dtype = getattr(torch, dtype)
    x, w, t = make(m, n, k, dtype, seed=1, ignored=0.1)
    g = torch.randn(m, device="cuda")
    lse = torch.logsumexp(x.float() @ w.float().t().contiguous(), 1)

    def step():
        return (latent.softmax_loss(x, w, t, reduction="none"), *latent.softmax_loss_grad(x, w, t, reduction="sum"),
                *latent.softmax_loss_backward(g, lse, None, x, w, t, need_x=True))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        for dst, src in zip((x, w, t), make(m, n, k, dtype, seed=30 + i, ignored=0.1)):
            dst.copy_(src)
        g.normal_()
        lse.copy_(torch.logsumexp(x.float() @ w.float().t().contiguous(), 1))
        graph.replay()
        for p, q in zip(out, step()):
            assert torch.equal(p, q)


def test_two_calls_at_once(gpu):
    """The same step on two streams side by side, many times over: each call has its own workspace."""
    torch = _torch()
    from blp import latent

    sets = [make(500, 2000, k, torch.bfloat16, seed=40 + k) for k in (64, 200)]
    want = [latent.softmax_loss_grad(*a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[] for _ in sets]
    for _ in range(20):
        for s, a, to in zip(streams, sets, got):
            with torch.cuda.stream(s):
                to.append(latent.softmax_loss_grad(*a))
    torch.cuda.synchronize()
    for w, all_of in zip(want, got):
        for out in all_of:
            assert all(torch.equal(p, q) for p, q in zip(out, w))


def test_refusals(gpu):
    torch = _torch()
    from blp import latent

    x, w, t = make(10, 20, 8, torch.float32)
    for bad in (lambda: latent.softmax_loss(x.double(), w, t), lambda: latent.softmax_loss(x, w.half(), t),
                lambda: latent.softmax_loss(x[:, :4], w, t), lambda: latent.softmax_loss(x, w, t[:5]),
                lambda: latent.softmax_loss(x, w, t.float()), lambda: latent.softmax_loss(x, w, t.cpu()),
                lambda: latent.softmax_loss(x.cpu(), w, t), lambda: latent.softmax_loss(x, w[:0], t),
                lambda: latent.softmax_loss(x.t(), w, t), lambda: latent.softmax_loss(x[0], w, t),
                lambda: latent.softmax_loss(x[:1].expand(10, 8), w, t), lambda: latent.softmax_loss(x, w, t, reduction="max"),
                lambda: latent.softmax_loss(x, w, t, scale=float("nan")),
                lambda: latent.softmax_loss_grad(x, w, t, reduction="none"),
                lambda: latent.softmax_loss_backward(torch.ones(3, device="cuda"), torch.ones(10, device="cuda"), None, x, w, t)):
        with pytest.raises(ValueError):
            bad()
