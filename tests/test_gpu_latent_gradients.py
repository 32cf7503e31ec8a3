"""The softmax loss's gradients keep 32-bit accuracy up to their one rounding (blp.latent.softmax_loss*).

dS is held as a sum of halves (two of them where the factors are halves, three where they are floats), so what its
rounding leaves is the half step of the type squared, h^2 (bfloat16 2^-16, float16 2^-22), or 2^-24. The bounds are those of
test_gpu_latent_loss.py with h^2 in the place of h: a gradient is off by
  scale sum_j (|g_i| (p_ij r_i + 2 u) + h2 |dS_ij|) |w_j| + (n + 8) u scale sum |dS w|, then h of the result,
  r_i = 2 dz_i + (depth + 16) u + 4 u (S_i + |lse_i|)
u = 2^-23. Catalogues are small, so that (n + 8) u stays far below h.
float16 holds dS times 2^14: its lowest step leaves 2^-25 2^-14 = 2^-39 of the largest row gradient.
"""
import pytest

from test_gpu_latent_loss import U, _half_step, _torch, make, near, reference

pytestmark = pytest.mark.gpu


def gradients(x, w, t, scale, gi, floor_dx, floor_dw=None):
    """-> ((dx, bound), (dw, bound)) of row gradients gi (64 bits); floor_dx, floor_dw: what float16's lowest step leaves of dS, in
    units of 2^-39 (dw: of the largest gi)."""
    import torch

    X, W = x.double(), w.double()
    n, k = W.shape
    ok = (t >= 0) & (t < n)
    X = torch.where(ok[:, None], X, 0.0)
    at = t.clamp(0, n - 1).long()[:, None]
    z = scale * (X @ W.t().contiguous())
    S = abs(scale) * (X.abs() @ W.abs().t().contiguous()).amax(1)
    lse = torch.logsumexp(z, 1)
    gi = torch.where(ok, gi, 0.0)
    p = torch.exp(z - lse[:, None])
    d = gi[:, None] * (p - torch.zeros_like(p).scatter_(1, at, 1.0))
    h = _half_step(x.dtype)
    h2 = 2.0 ** -24 if x.dtype == torch.float32 else h * h
    r = 2 * (k + 4) * U * S + (64 + n / 64 + 16) * U + 4 * U * (S + lse.abs())
    e = gi.abs()[:, None] * (p * r[:, None] + 2 * U) + h2 * d.abs()
    half = x.dtype == torch.float16
    tiny = torch.finfo(x.dtype).tiny * torch.finfo(x.dtype).eps / 2  # half the lowest step: results below the normal numbers

    def mm(a, b):
        return a @ b.contiguous()

    out = []
    for a, b, floor in ((lambda v: v, W, floor_dx), (lambda v: v.t(), X, gi.abs().max() if floor_dw is None else floor_dw)):
        want = scale * mm(a(d), b)
        bound = abs(scale) * (mm(a(e + floor * (2.0 ** -39 if half else 0.0)), b.abs()) + (max(x.shape[0], n) + 8) * U * mm(a(d).abs(), b.abs()))
        out.append((want, bound * (1 + 2 * h) + h * want.abs() + tiny))
    return out


@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "float32"])
@pytest.mark.parametrize("m,n,k", [(200, 260, 24), (300, 150, 64), (130, 333, 100), (129, 257, 128), (150, 300, 136), (300, 200, 328),
                                   (40, 90, 700), (600, 700, 200)])
def test_gradients_are_rounded_once(gpu, m, n, k, dtype):
    torch = _torch()
    from blp import latent

    x, w, t = make(m, n, k, getattr(torch, dtype), seed=m + k, ignored=0.1, scale=1.25)
    _, dx, dw = latent.softmax_loss_grad(x, w, t, scale=1.25, reduction="sum")
    one = torch.ones(m, dtype=torch.float64, device="cuda")
    for got, (want, bound) in zip((dx, dw), gradients(x, w, t, 1.25, one, one[:, None])):
        near(got, want, bound)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("k", [64, 200])
def test_backward_of_row_gradients_is_rounded_once(gpu, k, dtype):
    """The same through autograd, with gradients of their own for the rows."""
    torch = _torch()
    from blp import latent

    x, w, t = make(140, 300, k, getattr(torch, dtype), seed=k, ignored=0.1)
    g = torch.linspace(-2, 3, 140, device="cuda")
    x.requires_grad_(True)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(latent.softmax_loss(x, w, t, reduction="none"), (x, w), g)
    for got, (want, bound) in zip((dx, dw), gradients(x.detach(), w.detach(), t, 1.0, g.double(), g.double().abs().max())):
        near(got, want, bound)


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_pieces_of_the_catalogue_add_up(gpu, dtype):
    """dx of a catalogue of several pieces: 131,072 rows leave room for 1,024 columns of two halves each, 1,100 columns are two pieces."""
    torch = _torch()
    from blp import latent

    m, n, k = 131072, 1100, 136
    x, w, t = make(m, n, k, getattr(torch, dtype), seed=2, ignored=0.05)
    _, dx, dw = latent.softmax_loss_grad(x, w, t, reduction="sum")
    at = torch.cat([torch.arange(0, 200), torch.arange(m - 100, m)]).cuda()
    one = torch.ones(len(at), dtype=torch.float64, device="cuda")
    (want, bound), _ = gradients(x[at], w, t[at], 1.0, one, one[:, None])
    near(dx[at], want, bound)
    assert dw.isfinite().all()


@pytest.mark.parametrize("dtype,m,n,k", [("bfloat16", 16384, 87300, 200), ("float32", 15162, 62966, 104)])
def test_a_last_piece_of_fewer_slices(gpu, dtype, m, n, k):
    """A catalogue whose last piece has fewer stages than the slices of the others take: the row gradient's parts add up."""
    torch = _torch()
    from blp import latent

    x, w, t = make(m, n, k, getattr(torch, dtype), seed=4)
    _, dx, _ = latent.softmax_loss_grad(x, w, t, reduction="sum")
    at = torch.cat([torch.arange(0, 100), torch.arange(m - 60, m)]).cuda()
    one = torch.ones(len(at), dtype=torch.float64, device="cuda")
    (want, bound), _ = gradients(x[at], w, t[at], 1.0, one, one[:, None])
    near(dx[at], want, bound)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("k", [40, 64, 100, 160, 328])
def test_row_gradients_of_very_different_sizes(gpu, k, dtype):
    """Three decades of row gradients beside some 10^9 times larger, of rows whose target has all of the softmax: these have no part
    in dx or (but for component 0) in dtable, and the other rows' are as accurate as if they were alone."""
    torch = _torch()
    from blp import latent

    m, n = 150, 400
    x, w, t = make(m, n, k, getattr(torch, dtype), seed=k)
    t %= n - 1
    sure = torch.arange(m, device="cuda") % 10 == 3
    x[:, 0], w[:, 0] = 0, 0
    w[n - 1] = 0
    w[n - 1, 0] = 30  # the row that the sure ones are sure of: a score of 240 there, 0 everywhere else
    x[sure] = 0
    x[sure, 0] = 8
    t[sure] = n - 1
    g = torch.logspace(-3, 0, m, device="cuda") * torch.where(torch.arange(m, device="cuda") % 2 == 0, 1.0, -1.0)
    g[sure] *= 1e9
    lse = torch.logsumexp(x.double() @ w.double().t().contiguous(), 1).float()
    got = latent.softmax_loss_backward(g, lse, None, x, w, t)
    zero = torch.zeros((), dtype=torch.float64, device="cuda")
    (want_x, bound_x), (want_w, bound_w) = gradients(x, w, t, 1.0, g.double(), zero, zero)
    near(got[0][~sure], want_x[~sure], bound_x[~sure])
    near(got[1][:, 1:], want_w[:, 1:], bound_w[:, 1:])
    # without the sure rows: the same row gradients of x
    alone = latent.softmax_loss_backward(torch.where(sure, 0.0, g), lse, None, x, w, t)
    near(alone[0][~sure], want_x[~sure], bound_x[~sure])


@pytest.mark.parametrize("k", [8, 64, 72, 200])
def test_workspace_of_row_gradients(gpu, k):
    """float16 with one gradient and with one a row, of the same sizes, on strided rows."""
    torch = _torch()
    from blp import latent

    m, n = 90, 700
    x, w, t = make(m, n, k + 5, torch.float16, seed=k)
    x, w = x[:, 3:3 + k], w[:, 2:2 + k]
    lse = torch.logsumexp(x.double() @ w.double().t().contiguous(), 1).float()
    for g in (torch.full((), 0.5, device="cuda"), torch.full((m,), 0.5, device="cuda")):
        half = torch.full((m,), 0.5, dtype=torch.float64, device="cuda")
        for got, (want, bound) in zip(latent.softmax_loss_backward(g, lse, None, x, w, t), gradients(x, w, t, 1.0, half, half[:, None])):
            near(got, want, bound)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("k", [8, 64, 128, 200])
def test_gradients_where_scale_and_gradient_pass_the_floats(gpu, k, dtype):
    """scale / count is no normal number, or scale times the loss's gradient is infinite; the gradients themselves are floats."""
    torch = _torch()
    from blp import latent

    m, n = 12, 20
    x, w, t = make(m, n, k, getattr(torch, dtype), seed=k)
    one = torch.ones(m, dtype=torch.float64, device="cuda")
    X, W = x * 2.0 ** 50, w * 2.0 ** 50
    for scale in (2.0 ** -130, 2.0 ** -127, -(2.0 ** -128)):
        for p, (want, bound) in zip(latent.softmax_loss_grad(X, W, t, scale=scale)[1:], gradients(X, W, t, scale, one / m, one[:, None])):
            near(p, want, bound)
    X, W, top = x * 2.0 ** -20, w * 2.0 ** -100, torch.full((), 2.0 ** 100, device="cuda")
    lse = torch.logsumexp(2.0 ** 100 * (X.double() @ W.double().t().contiguous()), 1).float()
    dx, _ = latent.softmax_loss_backward(top, lse, None, X, W, t, scale=2.0 ** 100, need_table=False)
    near(dx, *gradients(X, W, t, 2.0 ** 100, one * 2.0 ** 100, one[:, None])[0])


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("k", [8, 64, 128, 200])
def test_scales_next_to_zero(gpu, k, dtype):
    """Products next to the largest float times scales next to its smallest: 0 is 0, and 2^-130 is itself."""
    torch = _torch()
    from blp import latent
    m, n = 40, 333
    x, w, t = make(m, n, k, getattr(torch, dtype), seed=k)
    x, w = x * 2.0 ** 62, w * (2.0 ** 62 * k ** 0.5 / k)
    for scale in (0.0, 2.0 ** -130, 2.0 ** -126, -(2.0 ** -128)):
        ref = reference(x, w, t, scale)
        near(latent.softmax_loss(x, w, t, scale=scale, reduction="none"), ref["loss"], ref["b_loss"])
        total, dx, dw = latent.softmax_loss_grad(x, w, t, scale=scale)
        near(dx, ref["dx"], ref["b_dx"] + 2.0 ** -133)
        near(dw, ref["dw"], ref["b_dw"] + 2.0 ** -133)


def test_more_rows_than_a_launch_joins(gpu):
    """2^28 rows and some more, whose pairs are joined in two launches; forward alone and with gradients."""
    torch = _torch()
    from blp import latent

    m, n, k, edge = (1 << 28) + 300, 50, 8, 1 << 28
    torch.cuda.empty_cache()
    x = torch.empty(m, k, dtype=torch.bfloat16, device="cuda")
    for at in range(0, m, 1 << 25):
        x[at:at + (1 << 25)].normal_()
    w = torch.randn(n, k, device="cuda").to(torch.bfloat16)
    t = torch.randint(-1, n, (m,), device="cuda", dtype=torch.int32)
    loss = latent.softmax_loss(x, w, t, reduction="none")
    total, dx, dw = latent.softmax_loss_grad(x, w, t, reduction="sum")
    for lo, hi in ((0, 200), (edge - 200, edge + 300)):
        ref = reference(x[lo:hi], w, t[lo:hi], 1.0)
        near(loss[lo:hi], ref["loss"], ref["b_loss"])
        one = torch.ones(hi - lo, dtype=torch.float64, device="cuda")
        near(dx[lo:hi], *gradients(x[lo:hi], w, t[lo:hi], 1.0, one, one[:, None])[0])
    assert abs(float(total) - float(loss.double().sum())) <= U * float(total) and dw.isfinite().all()
    del x, loss, dx
    torch.cuda.empty_cache()


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
@pytest.mark.parametrize("k", [40, 200])
def test_forward_leaves_what_backward_takes(gpu, k, reduction):
    """softmax_loss_forward, then softmax_loss_backward: the loss and the gradients of softmax_loss, also captured and replayed."""
    torch = _torch()
    from blp import latent

    m, n = 70, 300
    x, w, t = make(m, n, k, torch.bfloat16, seed=k, ignored=0.2)
    g = torch.randn(m, device="cuda") if reduction == "none" else torch.full((), 1.5, device="cuda")

    def step():
        loss, lse, count = latent.softmax_loss_forward(x, w, t, 0.5, reduction)
        return (loss, lse, *latent.softmax_loss_backward(g, lse, count, x, w, t, 0.5))

    def check(got):
        ref = reference(x, w, t, 0.5)
        scale = {"mean": 1.5 / ref["count"], "sum": 1.5, "none": 1.0}[reduction]
        per_row = g.double() if reduction == "none" else torch.full((m,), scale, dtype=torch.float64, device="cuda")
        near(got[1][ref["ok"]], ref["lse"][ref["ok"]], ref["b_loss"][ref["ok"]])
        xr, wr = x.clone().requires_grad_(), w.clone().requires_grad_()
        loss = latent.softmax_loss(xr, wr, t, 0.5, reduction)
        assert torch.equal(got[0], loss) and not got[0].requires_grad
        for p, (want, bound) in zip(got[2:], gradients(x, w, t, 0.5, per_row, per_row.abs().max())):
            near(p, want, bound)
        for p, q in zip(got[2:], torch.autograd.grad(loss, (xr, wr), g)):
            assert torch.equal(p, q)

    check(step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        for dst, src in zip((x, w, t), make(m, n, k, torch.bfloat16, seed=50 + i, ignored=0.2)):
            dst.copy_(src)
        graph.replay()
        check(out)
