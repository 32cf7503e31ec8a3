"""Row lookup and its gradient (blp.latent.lookup, lookup_grad) against their definitions.

A looked-up row is one 32-bit product rounded once: equal to the same in torch. A gradient's sum adds at
most 64 values and one partial sum in a chain in 32 bits (u = 2^-24 each), the partial sums in 64 bits,
then one product and one rounding to 32 bits: 68 u sum |g| scale; then half a step of the type.
"""
import pytest

pytestmark = pytest.mark.gpu


def _torch():
    return pytest.importorskip("torch")


def grad_reference(grad, ids, rows, scale, into=None):
    import torch

    k = grad.shape[-1]
    g = grad.reshape(-1, k).double()
    at = ids.reshape(-1).long()
    ok = (at >= 0) & (at < rows)
    out = torch.zeros(rows, k, dtype=torch.float64, device=grad.device)
    mag = torch.zeros_like(out)
    out.index_add_(0, at[ok], g[ok] * scale)
    mag.index_add_(0, at[ok], g[ok].abs() * abs(scale))
    bound = 68 * 2.0 ** -24 * mag
    if into is not None:
        out = out + into.double()
        bound = bound + 2.0 ** -24 * out.abs()
    h = torch.finfo(grad.dtype).eps / 2
    tiny = 2.0 ** -25 if grad.dtype == torch.float16 else 0.0
    return out, bound * (1 + h) + h * out.abs() + tiny


def check(got, want, bound):
    off = (got.double() - want).abs() - bound
    assert bool((off <= 0).all()), float(off.max())


CASES = [(1, 1, 1), (1, 300, 50), (20, 5000, 64), (63, 7, 3), (64, 7, 8), (65, 7, 130), (300, 1, 33), (2048, 100, 16),
         (2049, 100, 24), (5000, 3000, 64), (70001, 1500, 40), (30000, 70000, 7),
         (8192, 900, 20), (8193, 900, 20), (140001, 3000, 12)]


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("n,rows,k", CASES)
def test_lookup_and_gradient(gpu, n, rows, k, dtype):
    torch = _torch()
    from blp import latent

    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(n + rows)
    table = torch.randn(rows, k, device="cuda", generator=g).to(dt)
    # a few rows take most ids; some ids lie outside
    ids = (torch.rand(n, device="cuda", generator=g) ** 4 * (rows + 1)).long() - 1
    if n > 10:
        ids[3], ids[5], ids[7] = rows, -5, 2 ** 40
    for i in (ids, ids.clamp(-7, rows + 3).to(torch.int32)):
        ok = ((i >= 0) & (i < rows))[:, None]
        want = torch.where(ok, (table[i.clamp(0, rows - 1).long()].float() * 2.5), 0.0).to(dt)
        assert torch.equal(latent.lookup(table, i, 2.5), want)
        grad = torch.randn(n, k, device="cuda", generator=g).to(dt)
        got = latent.lookup_grad(grad, i, rows, scale=2.5)
        check(got, *grad_reference(grad, i, rows, 2.5))
        assert torch.equal(got, latent.lookup_grad(grad, i, rows, scale=2.5))


def test_three_sort_passes(gpu):
    """Row numbers of more than 20 bits."""
    torch = _torch()
    from blp import latent

    rows = (1 << 20) + 12345
    g = torch.Generator(device="cuda").manual_seed(1)
    ids = torch.randint(0, rows, (9000,), device="cuda", generator=g)
    ids[::3] = ids[0]
    ids[1::7] = rows - 1
    grad = torch.randn(9000, 5, device="cuda", generator=g)
    check(latent.lookup_grad(grad, ids, rows), *grad_reference(grad, ids, rows, 1.0))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_one_row_takes_all(gpu, dtype):
    torch = _torch()
    from blp import latent

    g = torch.Generator(device="cuda").manual_seed(2)
    grad = torch.randn(200000, 12, device="cuda", generator=g).to(getattr(torch, dtype))
    ids = torch.full((200000,), 4, dtype=torch.int32, device="cuda")
    got = latent.lookup_grad(grad, ids, 6)
    check(got, *grad_reference(grad, ids, 6, 1.0))
    assert not got[:4].any() and not got[5].any()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_added_to_a_gradient(gpu, dtype):
    torch = _torch()
    from blp import latent

    g = torch.Generator(device="cuda").manual_seed(3)
    dt = getattr(torch, dtype)
    for n in (100, 7000):
        grad = torch.randn(n, 20, device="cuda", generator=g).to(dt)
        ids = torch.randint(-1, 50, (n,), device="cuda", generator=g)
        ids[ids == 13] = -1
        wide = torch.randn(50, 32, device="cuda", generator=g).to(dt)
        into, before = wide[:, 4:24], wide.clone()
        assert latent.lookup_grad(grad, ids, 50, scale=0.5, into=into) is into
        check(into, *grad_reference(grad, ids, 50, 0.5, before[:, 4:24]))
        assert torch.equal(into[13], before[13, 4:24])  # a row without ids is left alone
        assert torch.equal(wide[:, :4], before[:, :4]) and torch.equal(wide[:, 24:], before[:, 24:])


def test_overlap_is_refused(gpu):
    torch = _torch()
    from blp import latent

    both = torch.zeros(20, 8, device="cuda")
    ids = torch.zeros(10, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError):
        latent.lookup_grad(both[:10], ids, 12, into=both[8:])
    latent.lookup_grad(both[:10], ids, 10, into=both[10:])


def test_shapes_strides_and_empty(gpu):
    torch = _torch()
    from blp import latent

    table = torch.randn(30, 40, device="cuda")
    ids = torch.randint(0, 30, (3, 5, 2), device="cuda")
    out = latent.lookup(table, ids)
    assert out.shape == (3, 5, 2, 40) and torch.equal(out, table[ids])
    part = table[:, 3:24]
    assert torch.equal(latent.lookup(part, ids), part[ids])
    check(latent.lookup_grad(out, ids, 30), *grad_reference(out, ids, 30, 1.0))
    none = ids[:0].reshape(0)
    assert latent.lookup(table, none).shape == (0, 40)
    z = latent.lookup_grad(torch.empty(0, 40, device="cuda"), none, 30)
    assert z.shape == (30, 40) and not z.any()


def test_nan_of_padded_entries_stays_out(gpu):
    torch = _torch()
    from blp import latent

    for n in (200, 5000):
        grad = torch.ones(n, 16, device="cuda")
        ids = torch.arange(n, device="cuda") % 9
        ids[::4] = -1
        grad[::4] = float("nan")
        got = latent.lookup_grad(grad, ids, 9)
        assert bool(torch.isfinite(got).all())
        check(got, *grad_reference(torch.nan_to_num(grad), ids, 9, 1.0))


def test_autograd_and_replay(gpu):
    torch = _torch()
    from blp import latent

    table = torch.randn(100, 24, device="cuda", requires_grad=True)
    ids = torch.randint(-1, 100, (6, 50), device="cuda")
    y = latent.lookup(table, ids, 1.5)
    (got,) = torch.autograd.grad((y * y).sum(), (table,))
    check(got, *grad_reference((2 * y).detach(), ids, 100, 1.5))
    grad, big = torch.randn(5000, 24, device="cuda"), torch.randint(0, 100, (5000,), device="cuda")
    latent.lookup_grad(grad, big, 100)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = latent.lookup_grad(grad, big, 100)
    for i in range(4):
        grad.copy_(torch.randn(5000, 24, device="cuda"))
        big.copy_(torch.randint(0, 100, (5000,), device="cuda"))
        graph.replay()
        assert torch.equal(out, latent.lookup_grad(grad, big, 100))


@pytest.mark.parametrize("n,rows", [(20000, 700), (300000, 2500)])
def test_long_lists_captured_and_replayed(gpu, n, rows):
    torch = _torch()
    from blp import latent

    grad, ids = torch.randn(n, 20, device="cuda"), torch.randint(-1, rows, (n,), device="cuda")
    into = torch.randn(rows, 20, device="cuda")
    held = into.clone()

    def step(into):
        return latent.lookup_grad(grad, ids, rows, 0.5), latent.lookup_grad(grad, ids, rows, 0.5, into=into)

    step(into.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(into)
    for i in range(4):
        grad.normal_()
        ids.copy_((torch.rand(n, device="cuda") ** 3 * (rows + 1)).long() - 1)
        into.copy_(held)
        graph.replay()
        for p, q in zip(out, step(held.clone())):
            assert torch.equal(p, q)


def test_refusals(gpu):
    torch = _torch()
    from blp import latent

    table, ids = torch.randn(10, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    grad = torch.ones(4, 8, device="cuda")
    for bad in (lambda: latent.lookup(table.double(), ids), lambda: latent.lookup(table, ids.float()),
                lambda: latent.lookup(table, ids.cpu()), lambda: latent.lookup(table.t(), ids), lambda: latent.lookup(table[:0], ids),
                lambda: latent.lookup(table, ids, float("inf")), lambda: latent.lookup(table, ids.repeat(2)[::2]),
                lambda: latent.lookup_grad(grad[:3], ids, 10), lambda: latent.lookup_grad(grad, ids, 0),
                lambda: latent.lookup_grad(grad.cpu(), ids.cpu(), 10),
                lambda: latent.lookup_grad(grad, ids, 10, into=torch.zeros(9, 8, device="cuda")),
                lambda: latent.lookup_grad(grad, ids, 10, into=torch.zeros(10, 8, device="cuda", dtype=torch.float16))):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("n", [100, 9000])
def test_into_counts_as_changed(gpu, n):
    torch = _torch()
    from blp import latent

    grad, ids = torch.randn(n, 8, device="cuda"), torch.randint(0, 20, (n,), device="cuda")
    into, p = torch.zeros(20, 8, device="cuda"), torch.randn(20, 8, device="cuda", requires_grad=True)
    loss = (into * p).sum()  # autograd keeps `into`
    before = into._version
    latent.lookup_grad(grad, ids, 20, into=into)
    assert into._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    wide = torch.zeros(20, 12, device="cuda")
    loss = (wide * torch.randn(20, 12, device="cuda", requires_grad=True)).sum()
    latent.lookup_grad(grad, ids, 20, into=wide[:, 2:10])  # a view: what it is a view of has changed
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    with pytest.raises(ValueError, match="require"):
        latent.lookup_grad(grad, ids, 20, into=p)
    with torch.no_grad():
        latent.lookup_grad(grad, ids, 20, into=p)
