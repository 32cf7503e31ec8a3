"""What blp.latent's calls refuse before they look at a device: transformations that would see only the allocation of their outputs,
and tensors whose memory is not their value."""
import pytest

from blp import latent

torch = pytest.importorskip("torch")


def calls(x, ids):
    """-> every entry point, as a call of the float tensor x (n, k)"""
    one = torch.ones(len(x))
    return {
        "softmax_loss": lambda: latent.softmax_loss(x, torch.ones_like(x.detach()), ids),
        "softmax_loss_forward": lambda: latent.softmax_loss_forward(x, x, ids),
        "softmax_loss_grad": lambda: latent.softmax_loss_grad(x, x, ids),
        "softmax_loss_backward": lambda: latent.softmax_loss_backward(one, one, None, x, x, ids),
        "lookup": lambda: latent.lookup(x, ids),
        "lookup_grad": lambda: latent.lookup_grad(x, ids, 5),
        "quantize_rows": lambda: latent.quantize_rows(x),
    }


NAMES = sorted(calls(torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)))


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name):
    """A dual tensor does not require a gradient: a result without its tangent would be a derivative of zero."""
    from torch.autograd import forward_ad

    x, ids = torch.randn(4, 8), torch.zeros(4, dtype=torch.int64)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward-mode"):
            calls(dual, ids)[name]()
    with pytest.raises(ValueError, match="GPU"):  # outside of it: a tensor on the host
        calls(x, ids)[name]()


def test_forward_mode_of_scales_is_refused():
    from torch.autograd import forward_ad

    with forward_ad.dual_level():
        dual = forward_ad.make_dual(torch.ones(4), torch.ones(4))
        with pytest.raises(RuntimeError, match="forward-mode"):
            latent._t()
            latent._floats(dual, "s", dual.device, ((4,),))


@pytest.mark.gpu
def test_forward_mode_is_refused_for_every_argument(gpu):
    from torch.autograd import forward_ad

    x, ids, q = torch.randn(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.ones(
        4, 8, dtype=torch.int8, device="cuda")
    one = torch.ones(4, device="cuda")
    with forward_ad.dual_level():
        d, done = forward_ad.make_dual(x, x), forward_ad.make_dual(one, one)
        for call in (lambda: latent.softmax_loss(x, d, ids), lambda: latent.softmax_loss(d.clone().requires_grad_(), x, ids),
                     lambda: latent.softmax_loss_grad(x, d, ids), lambda: latent.softmax_loss_backward(done, one, None, x, x, ids),
                     lambda: latent.softmax_loss_backward(one, done, None, x, x, ids), lambda: latent.lookup(d, ids),
                     lambda: latent.lookup_grad(x, ids, 4, into=d), lambda: latent.int8_scores(q, done, q, one),
                     lambda: latent.int8_scores(q, one, q, done)):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
        assert latent.lookup(x, ids).shape == (4, 8)  # others go through
    # the transformations that wrap their tensors refuse by themselves
    for call in (lambda: torch.func.jvp(lambda a: latent.lookup(a, ids), (x,), (x,)),
                 lambda: torch.func.vmap(lambda a: latent.softmax_loss(a, x, ids))(x[None]),
                 lambda: torch.func.grad(lambda a: latent.softmax_loss(a, x, ids))(x)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("name", NAMES)
def test_tracing_is_refused(name):
    """A trace would record the allocation of the outputs, and nothing that fills them."""
    ids = torch.zeros(4, dtype=torch.int64)

    def traced(x):
        with pytest.raises(RuntimeError, match="traced"):
            calls(x, ids)[name]()
        return x

    torch.jit.trace(traced, torch.randn(4, 8), check_trace=False)


@pytest.mark.gpu
def test_tracing_is_refused_on_the_device(gpu):
    x, ids, q = torch.randn(4, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), torch.ones(
        4, 8, dtype=torch.int8, device="cuda")
    for call in (lambda a: latent.lookup(a, ids), lambda a: latent.softmax_loss(a, x, ids), lambda a: latent.softmax_loss(x, a, ids),
                 lambda a: latent.int8_scores(q, a[:, 0].contiguous(), q, a[:, 0].contiguous())):
        for arg in (x, x.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="traced"):
                torch.jit.trace(call, arg, check_trace=False)
    fn = torch.compile(lambda a: latent.softmax_loss(a, x, ids) * 2, backend="eager")  # falls back to running the call
    assert torch.equal(fn(x), latent.softmax_loss(x, x, ids) * 2)


@pytest.mark.gpu
def test_negated_views_are_refused(gpu):
    ids = torch.zeros(4, dtype=torch.int64, device="cuda")
    neg = torch.complex(torch.zeros(4, 1, device="cuda"), torch.ones(4, 1, device="cuda")).conj().imag
    assert neg.is_neg() and neg[0] == -1
    one, q = torch.ones(1, device="cuda"), torch.ones(1, 8, dtype=torch.int8, device="cuda")
    for call in (lambda: latent.lookup(neg, ids), lambda: latent.lookup_grad(neg, ids, 4), lambda: latent.quantize_rows(neg),
                 lambda: latent.softmax_loss(neg, neg, ids), lambda: latent.int8_scores(q, neg[0], q, one)):
        with pytest.raises(ValueError, match="negat"):
            call()
    assert torch.equal(latent.lookup(neg.resolve_neg(), ids), -torch.ones(4, 1, device="cuda"))


def test_arguments_that_the_library_refuses_are_value_errors():
    from blp import _lib

    latent._t()
    for args in ((0, None, 0, 256, 8, 5, 8, 256, 0, 3, float("inf"), 256, 8), (0, None, 0, 256, 8, 1 << 31, 8, 256, 0, 3, 1.0, 256, 8)):
        with pytest.raises(ValueError) as e:
            latent.check(_lib.lib().blp_lookup(*args))
        assert isinstance(e.value, _lib.BLPError) and e.value.code == -1


@pytest.mark.gpu
def test_far_strides_are_value_errors(gpu):
    far = torch.zeros(2, (1 << 20) + 8, dtype=torch.float16, device="cuda")[:, :8]
    t = torch.zeros(2, dtype=torch.int64, device="cuda")
    w = torch.zeros(5, 8, dtype=torch.float16, device="cuda")
    with pytest.raises(ValueError, match="stride"):
        latent.softmax_loss(far, w, t)
    q = torch.zeros(2, (1 << 22) + 16, dtype=torch.int8, device="cuda")[:, :16]
    with pytest.raises(ValueError, match="stride"):
        latent.int8_scores(q, torch.ones(2, device="cuda"), q, torch.ones(2, device="cuda"))
    with pytest.raises(ValueError, match="scale"):
        latent.lookup(w, t, 1e39)


@pytest.mark.parametrize("name", NAMES)
def test_tracing_by_the_ids_is_refused(name):
    x = torch.randn(4, 8)

    def traced(ids):
        with pytest.raises(RuntimeError, match="traced"):
            calls(x, ids)[name]()
        return ids

    torch.jit.trace(traced, torch.zeros(4, dtype=torch.int64), check_trace=False)


def test_scales_whose_derivative_would_be_dropped_are_refused():
    """A scale is a number. One that requires a gradient, or is traced or dual, would lose it without an error."""
    from torch.autograd import forward_ad

    x, ids = torch.randn(4, 8), torch.zeros(4, dtype=torch.int64)
    uses = (lambda s: latent.softmax_loss(x, x, ids, scale=s), lambda s: latent.softmax_loss(x.requires_grad_(), x, ids, scale=s),
            lambda s: latent.softmax_loss_grad(x, x, ids, scale=s), lambda s: latent.lookup(x, ids, s),
            lambda s: latent.lookup_grad(x, ids, 4, scale=s))
    for use in uses:
        with pytest.raises(ValueError, match="scale must not require"):
            use(torch.tensor(2.0, requires_grad=True))
        with forward_ad.dual_level():
            with pytest.raises(RuntimeError, match="scale: forward-mode"):
                use(forward_ad.make_dual(torch.tensor(2.0), torch.tensor(1.0)))
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            use(torch.tensor(2.0, requires_grad=True))
