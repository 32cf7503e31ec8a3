"""8-bit factor rows and their scores of the catalogue (blp.latent.quantize_rows, int8_scores), and the latent
operators together.

The sum of a score is a whole number and exact; its conversion and the two scales round three times in 32
bits (2^-24 each), then to the output's type (half a step). Quantised values equal their definition.
"""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    return pytest.importorskip("torch")


def quantize(x):
    """The definition in 64 bits: (whole numbers, float32 scales)."""
    import torch

    x = x.double()
    s = (x.abs().amax(1) / 127).float()
    q = torch.where(s[:, None] > 0, torch.round(x / s.double()[:, None]), 0.0).clamp(-127, 127)
    return q.to(torch.int8), s


def check_scores(got, q, s, p, t):
    import torch

    want = (q.double() @ p.double().t().contiguous()) * s.double()[:, None] * t.double()[None, :]
    h = torch.finfo(got.dtype).eps / 2
    # Below the type's smallest normal number roundings are off by half of its last place at most, whatever the value:
    # float16 2^-24 / 2; float32 2^-149 / 2 (the product with t; sum times s is a multiple of s, so it is a multiple of
    # 2^-149 and exact there); bfloat16 2^-133 / 2 after that float32 rounding.
    tiny = {torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134 + 2.0 ** -150}[got.dtype]
    off = (got.double() - want).abs() - (want.abs() * (3 * 2.0 ** -24 + h) * 1.001 + tiny)
    assert got.shape == want.shape and bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 5), (100, 64), (257, 50), (33, 1000), (7, 8200)])
def test_quantized_rows(gpu, n, k, dtype):
    torch = _torch()
    from blp import latent

    g = torch.Generator(device="cuda").manual_seed(n * k)
    x = (torch.randn(n, k, device="cuda", generator=g) * 10.0 ** torch.randint(-3, 3, (n, 1), device="cuda", generator=g)).to(
        getattr(torch, dtype))
    x[n // 2] = 0
    q, s = latent.quantize_rows(x)
    wq, ws = quantize(x)
    assert torch.equal(s, ws) and torch.equal(q, wq)
    assert q.stride(0) % 16 == 0


def test_quotients_on_a_border(gpu):
    """Values that lie on or next to halves of the scale, tiny rows and rows that are not finite."""
    torch = _torch()
    from blp import latent

    s0 = torch.tensor([1.0, 0.3, 1e-30, 3e38 / 127, 7.77], device="cuda")
    half = (torch.arange(-126, 127, device="cuda") + 0.5)[None, :] * s0[:, None]
    x = torch.cat([half, torch.nextafter(half, half * 2), torch.nextafter(half, half * 0), 127 * s0[:, None]], 1)
    q, s = latent.quantize_rows(x)
    wq, ws = quantize(x)
    assert torch.equal(s, ws) and torch.equal(q, wq)
    x = torch.zeros(5, 20, device="cuda")
    x[0, 3] = 1e-44
    x[1, 19] = float("inf")
    x[2, 0] = float("nan")
    x[3, 1] = -1e-39
    q, s = latent.quantize_rows(x)
    assert not q[1].any() and not q[2].any() and torch.isnan(s[1:3]).all() and s[4] == 0 and not q[4].any()
    assert int(q[3, 1]) == -127 and s[3] > 0


@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 5003, 64), (7, 300, 50), (32, 1000, 200), (33, 129, 128), (130, 4099, 64),
                                   (300, 301, 1000), (3500, 4600, 272)])
def test_scores(gpu, m, n, k, out):
    torch = _torch()
    from blp import latent

    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    q = torch.randint(-128, 128, (m, k), device="cuda", generator=g).to(torch.int8)
    p = torch.randint(-128, 128, (n, k), device="cuda", generator=g).to(torch.int8)
    s = torch.rand(m, device="cuda", generator=g) * 1e-3
    t = torch.rand(n, device="cuda", generator=g) * 1e-2
    got = latent.int8_scores(q, s, p, t, dtype=getattr(torch, out))
    check_scores(got, q, s, p, t)


@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", [(5, 700, 64), (40, 300, 200), (300, 301, 1000)])
def test_scales_far_apart(gpu, m, n, k, out):
    """Large scales of rows against small ones of the catalogue: sum times row scale passes the largest float, the score
    does not."""
    torch = _torch()
    from blp import latent

    g = torch.Generator(device="cuda").manual_seed(m)
    q = torch.randint(-128, 128, (m, k), device="cuda", generator=g).to(torch.int8)
    p = torch.randint(-128, 128, (n, k), device="cuda", generator=g).to(torch.int8)
    q[0], p[0] = 127, 127
    s = (0.5 + torch.rand(m, device="cuda", generator=g)) * 2.0 ** 126
    t = (0.5 + torch.rand(n, device="cuda", generator=g)) * 2.0 ** -120
    s[-1], s[-2] = 2.0 ** -40, -2.0 ** 120
    if out == "float16":
        t *= 2.0 ** -6
        p[:, 1:] = 0
    check_scores(latent.int8_scores(q, s, p, t, dtype=getattr(torch, out)), q, s, p, t)


@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", [(300, 90001, 50), (129, 210002, 128), (37, 700003, 64), (1000, 27004, 100),
                                   (1400, 100001, 50), (130, 1100002, 128)])
def test_many_scores_in_rows_of_odd_lengths(gpu, m, n, k, out):
    """Rows that begin anywhere in a line, in outputs that the caches hold and past their 256 MB."""
    torch = _torch()
    from blp import latent

    g = torch.Generator(device="cuda").manual_seed(n)
    q = torch.randint(-128, 128, (m, k), device="cuda", generator=g).to(torch.int8)
    p = torch.randint(-128, 128, (n, k), device="cuda", generator=g).to(torch.int8)
    s = torch.rand(m, device="cuda", generator=g) * 1e-3
    t = torch.rand(n, device="cuda", generator=g) * 1e-2
    s[1] = 2.0 ** 100
    t[: n // 2] *= 2.0 ** -100 if out != "float16" else 1.0
    got = latent.int8_scores(q, s, p, t, dtype=getattr(torch, out))
    if out == "float16":  # row 1 passes its largest number
        got, q, s = got[2:], q[2:], s[2:]
    check_scores(got, q, s, p, t)


@pytest.mark.parametrize("m", [140, 700])
def test_rows_of_odd_lengths_leave_their_surroundings(gpu, m):
    """Into rows of a wider buffer: only the scores change."""
    torch = _torch()
    from blp import latent
    from blp._lib import check, lib

    n, k, ld = 200001, 64, 200013
    q, s = latent.quantize_rows(torch.randn(m, k, device="cuda"))
    p, t = latent.quantize_rows(torch.randn(n, k, device="cuda"))
    for dtype, code in ((torch.float32, 0), (torch.bfloat16, 1)):
        want = latent.int8_scores(q, s, p, t, dtype=dtype)
        buf = torch.full((m + 2, ld), 77.0, device="cuda", dtype=dtype)
        check(lib().blp_scores8(0, torch.cuda.current_stream().cuda_stream, q.data_ptr(), k, s.data_ptr(), p.data_ptr(), k,
                                t.data_ptr(), m, n, k, code, buf[1:, 5:].data_ptr(), ld, None, 0))
        assert torch.equal(buf[1:-1, 5:5 + n], want)
        buf[1:-1, 5:5 + n] = 77.0
        assert bool((buf == 77.0).all())


@pytest.mark.parametrize("out", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("m,n,k", [(10, 1266, 6462), (1, 3, 5000), (100, 1001, 4100), (321, 2047, 6120), (40, 513, 272), (1, 40001, 513)])
def test_long_rows_of_few_tiles(gpu, m, n, k, out):
    """Where k is taken in slices, whose sums are joined."""
    torch = _torch()
    from blp import latent

    g = torch.Generator(device="cuda").manual_seed(k)
    q = torch.randint(-128, 128, (m, k), device="cuda", generator=g).to(torch.int8)
    p = torch.randint(-128, 128, (n, k), device="cuda", generator=g).to(torch.int8)
    s = torch.rand(m, device="cuda", generator=g) * 1e-3
    t = torch.rand(n, device="cuda", generator=g) * 1e-2
    if out != "float16":
        s[-1] = 2.0 ** 110
        t[n // 2:] *= 2.0 ** -110
    check_scores(latent.int8_scores(q, s, p, t, dtype=getattr(torch, out)), q, s, p, t)


@pytest.mark.parametrize("m,n,k", [(1, 700, 50), (5, 700, 50), (700, 60, 50), (40, 3000, 201), (300, 301, 1001), (9, 1266, 6462),
                                   (1400, 100001, 50)])
def test_rows_end_inside_a_granule_of_anything(gpu, m, n, k):
    """k not a multiple of 16, rows that begin at whole granules, anything in the bytes behind them."""
    torch = _torch()
    from blp import latent

    g = torch.Generator(device="cuda").manual_seed(k)
    wide = (k + 15) // 16 * 16
    q = torch.randint(-128, 128, (m, wide), device="cuda", generator=g).to(torch.int8)[:, :k]
    p = torch.randint(-128, 128, (n, wide + 16), device="cuda", generator=g).to(torch.int8)[:, :k]
    s = torch.rand(m, device="cuda", generator=g) * 1e-3
    t = torch.rand(n, device="cuda", generator=g) * 1e-2
    check_scores(latent.int8_scores(q, s, p, t), q, s, p, t)


def test_longest_sums(gpu):
    """The largest k: sums next to 2^31."""
    torch = _torch()
    from blp import latent

    k = (1 << 17) - 1
    q = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
    p = torch.full((5, k), -128, dtype=torch.int8, device="cuda")
    p[1] = 127
    one = torch.ones(5, device="cuda")
    got = latent.int8_scores(q, one[:3], p, one)
    assert float(got[0, 0]) == 2 ** 31 - 2 ** 14 and got[2, 1] == torch.tensor(-128.0 * 127 * k)
    with pytest.raises(ValueError):
        latent.int8_scores(torch.zeros(1, k + 1, dtype=torch.int8, device="cuda"), one[:1],
                           torch.zeros(1, k + 1, dtype=torch.int8, device="cuda"), one[:1])


def test_strides_padding_and_no_rows(gpu):
    torch = _torch()
    from blp import latent

    x, w = torch.randn(40, 70, device="cuda"), torch.randn(90, 70, device="cuda")
    q, s = latent.quantize_rows(x)
    p, t = latent.quantize_rows(w)
    a = latent.int8_scores(q, s, p, t)
    check_scores(a, q, s, p, t)
    # the padding's bytes are no part of a row
    wide = torch.full((90, 96), 77, dtype=torch.int8, device="cuda")
    wide[:, 5:75] = p
    assert torch.equal(a, latent.int8_scores(q.contiguous(), s, wide[:, 5:75], t))
    assert latent.int8_scores(q[:0], s[:0], p, t).shape == (0, 90)
    assert latent.quantize_rows(x[:0])[0].shape == (0, 70)
    s2 = s.clone()
    s2[3] = float("nan")
    b = latent.int8_scores(q, s2, p, t)
    assert torch.isnan(b[3]).all() and torch.equal(b[4:], a[4:])


def test_replayed(gpu):
    torch = _torch()
    from blp import latent

    x = torch.randn(33, 100, device="cuda")
    p, t = latent.quantize_rows(torch.randn(700, 100, device="cuda"))
    latent.int8_scores(*latent.quantize_rows(x), p, t)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = latent.int8_scores(*latent.quantize_rows(x), p, t)
    for _ in range(4):
        x.copy_(torch.randn(33, 100, device="cuda"))
        graph.replay()
        assert torch.equal(out, latent.int8_scores(*latent.quantize_rows(x), p, t))


@pytest.mark.parametrize("m,n,k", [(10, 1266, 6462), (300, 90001, 64), (600, 3000, 300), (1400, 100001, 64)])
def test_every_path_replayed(gpu, m, n, k):
    torch = _torch()
    from blp import latent

    x = torch.randn(m, k, device="cuda")
    p, t = latent.quantize_rows(torch.randn(n, k, device="cuda"))
    latent.int8_scores(*latent.quantize_rows(x), p, t, dtype=torch.bfloat16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = latent.int8_scores(*latent.quantize_rows(x), p, t, dtype=torch.bfloat16)
    for _ in range(4):
        x.normal_()
        graph.replay()
        assert torch.equal(out, latent.int8_scores(*latent.quantize_rows(x), p, t, dtype=torch.bfloat16))


def test_refusals(gpu):
    torch = _torch()
    from blp import latent

    q, s = latent.quantize_rows(torch.randn(4, 32, device="cuda"))
    for bad in (lambda: latent.quantize_rows(q), lambda: latent.quantize_rows(torch.randn(4, 8)),
                lambda: latent.quantize_rows(torch.randn(8, 4, device="cuda").t()),
                lambda: latent.int8_scores(q.float(), s, q, s), lambda: latent.int8_scores(q, s[:2], q, s),
                lambda: latent.int8_scores(q, s, q[:, :16], s), lambda: latent.int8_scores(q, s.double(), q, s),
                lambda: latent.int8_scores(q, s, q, s, dtype=torch.float64), lambda: latent.int8_scores(q, s, q[:0], s[:0])):
        with pytest.raises(ValueError):
            bad()


def test_training_step_then_scores(gpu):
    """As they are used together: the users' rows looked up, the softmax loss over the businesses, both tables'
    gradients, a step down them, then the 8-bit scores of the trained tables."""
    torch = _torch()
    from blp import latent

    g = torch.Generator(device="cuda").manual_seed(1)
    users = (torch.randn(500, 64, device="cuda", generator=g) * 0.1).requires_grad_(True)
    businesses = (torch.randn(900, 64, device="cuda", generator=g) * 0.1).requires_grad_(True)
    ids = torch.randint(0, 500, (300,), device="cuda", generator=g)
    ids[::10] = -1
    target = torch.randint(0, 900, (300,), device="cuda", generator=g)
    target[::10] = -1
    loss = latent.softmax_loss(latent.lookup(users, ids, 8.0), businesses, target)
    du, db = torch.autograd.grad(loss, (users, businesses))
    U, B = users.detach().double().requires_grad_(True), businesses.detach().double().requires_grad_(True)
    keep = ids >= 0
    z = (8.0 * U[ids[keep]]) @ B.t()
    want = torch.nn.functional.cross_entropy(z, target[keep])
    dU, dB = torch.autograd.grad(want, (U, B))
    loss, want = loss.detach(), want.detach()
    # 32-bit sums of 64 and 900 products of values below 1, relative to the gradients' size
    assert abs(float(loss) - float(want)) < 2e-6 * float(want)
    for got, ref in ((du, dU), (db, dB)):
        assert float((got.double() - ref).abs().max()) < 1e-5 * float(ref.abs().max())
    with torch.no_grad():
        users -= 50.0 * du
        businesses -= 50.0 * db
        q, s = latent.quantize_rows(latent.lookup(users, ids.clamp(min=0)))
        p, t = latent.quantize_rows(businesses)
        got = latent.int8_scores(q, s, p, t)
        full = users[ids.clamp(min=0)].double() @ businesses.double().t()
        # each factor is off by half a scale: sum (|x| t / 2 + |w| s / 2 + s t / 4)
        x, w = users[ids.clamp(min=0)].double().abs().sum(1), businesses.double().abs().sum(1)
        bound = 0.5 * x[:, None] * t.double() + 0.5 * s.double()[:, None] * w + 16.0 * s.double()[:, None] * t.double()
        assert bool(((got.double() - full).abs() <= bound * 1.0001).all())


def test_more_rows_than_a_launch_takes(gpu):
    """64 lanes a row: 2^25 rows are 2^31 threads, the most of a launch."""
    torch = _torch()
    from blp import latent

    n, k, edge = (1 << 25) + 70, 513, 1 << 25
    x = torch.empty(n, k, dtype=torch.bfloat16, device="cuda")
    for at in range(0, n, 1 << 22):
        x[at:at + (1 << 22)].normal_()
    q, s = latent.quantize_rows(x)
    for lo, hi in ((0, 100), (edge - 100, edge + 70), (n - 100, n)):
        want_q, want_s = latent.quantize_rows(x[lo:hi])
        assert torch.equal(q[lo:hi], want_q) and torch.equal(s[lo:hi], want_s)


def test_more_tiles_than_a_launch_takes(gpu):
    """2^23 tiles of 512 threads are 2^32: workgroups that take tile after tile. 139 GB of scores."""
    torch = _torch()
    from blp import latent

    m, n, k = 129, 1 << 29, 16
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 180e9:
        pytest.skip("needs 180 GB of device memory")
    q = torch.randint(-127, 128, (m, k), dtype=torch.int8, device="cuda")
    p = torch.empty(n, k, dtype=torch.int8, device="cuda")
    for at in range(0, n, 1 << 26):
        p[at:at + (1 << 26)].random_(-127, 128)
    s, t = torch.rand(m, device="cuda"), torch.rand(n, device="cuda")
    got = latent.int8_scores(q, s, p, t, dtype=torch.bfloat16)
    for lo in (0, 128 * 12345 - 50, (1 << 28) - 50, n - 1000):
        want = latent.int8_scores(q, s, p[lo:lo + 1000], t[lo:lo + 1000], dtype=torch.bfloat16)
        assert torch.equal(got[:, lo:lo + 1000], want)
    del got
    torch.cuda.empty_cache()
