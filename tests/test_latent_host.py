"""The latent-factor entry points' refusals, on the host: every check comes before the device is touched."""
import ctypes

import pytest

import blp
from blp import _lib, latent

ONE = 1 << 20  # a stand-in for a device pointer that no refused call reads


def lib():
    latent._t()
    return _lib.lib()


def refused(rc, what):
    assert rc == -1, rc
    assert what in lib().blp_last_error().decode()


def loss(type=1, x=ONE, ldx=64, w=ONE, ldw=64, target=ONE, rows=10, cols=20, k=64, scale=1.0, loss=ONE, lse=ONE, grads=0, dx=None,
         lddx=64, dw=None, lddw=64, ws=ONE, ws_bytes=0):
    return lib().blp_softmax_loss(0, None, type, x, ldx, w, ldw, target, 1, rows, cols, k, scale, loss, lse, None, 0, grads, dx, lddx,
                                  dw, lddw, ws, ws_bytes)


@pytest.mark.parametrize("args,what", [
    ({"type": 3}, "type"), ({"rows": -1}, "rows"), ({"rows": 1 << 31}, "rows"), ({"cols": 0}, "catalogue"), ({"k": 0}, "k must"),
    ({"k": (1 << 20) + 1}, "k must"), ({"x": None}, "null"), ({"w": None}, "null"), ({"target": None}, "null"), ({"loss": None}, "null"),
    ({"ws": None}, "null"), ({"ldx": 63}, "stride"), ({"ldw": 63}, "stride"), ({"ldw": (1 << 20) + 1}, "strides"),
    ({"grads": 1, "dx": ONE, "lddx": 63}, "stride"), ({"grads": 1, "dw": ONE, "lddw": 63}, "stride"), ({"scale": float("nan")}, "scale"),
    ({"scale": float("inf")}, "scale"), ({}, "workspace is too small"), ({"ws": ONE + 16, "ws_bytes": 1 << 40}, "aligned")])
def test_softmax_loss_refuses(args, what):
    refused(loss(**args), what)


@pytest.mark.parametrize("args,what", [({"rows": (1 << 31) - (1 << 16) + 1}, "rows"), ({"cols": (1 << 31) - (1 << 16) + 1}, "catalogue")])
def test_softmax_loss_refuses_rows_whose_stages_pass_31_bits(args, what):
    refused(loss(**args), what)


def test_softmax_loss_backward_refuses():
    refused(lib().blp_softmax_loss_backward(0, None, 0, ONE, 8, ONE, 8, ONE, 0, 4, 4, 8, 1.0, ONE, ONE, 2, None, ONE, 8, ONE, 8, ONE,
                                            1 << 40), "grad_stride")


def workspace(type, rows, cols, k, forward=1, grads=1, x=ONE, ldx=None, w=ONE, ldw=None):
    n = ctypes.c_int64(-1)
    rc = lib().blp_softmax_loss_workspace(type, x, k if ldx is None else ldx, w, k if ldw is None else ldw, rows, cols, k, forward,
                                          grads, ctypes.byref(n))
    assert rc == 0
    return n.value


def test_softmax_loss_forward_workspace_is_bounded():
    """The forward pass alone: its pairs of as many rows as 256 MiB hold, a float a row, and the factors where packed."""
    for type, planes in ((0, 3), (1, 1), (2, 1)):
        for rows, cols, k in ((1 << 20, 1 << 20, 256), (1 << 24, 100000, 136), (300, 1 << 30, 136), (1 << 20, 40, 1000)):
            factors = 2 * planes * (rows + cols) * k if type == 0 else 0
            pairs = max(256 << 20, 8 * 512 * (cols // 32 + 4))
            assert workspace(type, rows, cols, k, grads=0, x=1 << 20, w=1 << 20) <= factors + pairs + 4 * rows + 4096


def test_softmax_loss_workspace_is_bounded():
    """The workspace never grows with rows x columns past one piece of the catalogue and the partial sums."""
    for type, es in ((0, 4), (1, 2), (2, 2)):
        for k in (1, 50, 64, 100, 129, 1000):
            for rows, cols in ((0, 1), (1, 1), (1, 200000), (10000, 100000), (16384, 200000), (100000, 77)):
                n = workspace(type, rows, cols, k)
                kp = -(-k // 8) * 8
                planes = 3 if type == 0 else 1
                factors = 2 * planes * (rows + cols) * kp
                parts = 64 * 4 * (rows + cols) * (k + 4) + 8 * rows * 2048
                assert 256 <= n <= factors + parts + (512 << 20) + 2 * planes * 256 * rows + (1 << 20), (type, k, rows, cols, n)
                assert workspace(type, rows, cols, k, grads=0) <= n + (1 << 20)
    # rows that are not whole 16-byte granules are packed: more workspace
    assert workspace(1, 100, 5000, 50) > workspace(1, 100, 5000, 56, grads=1)
    assert workspace(1, 100, 5000, 64, w=ONE + 2) > workspace(1, 100, 5000, 64)


def test_lookup_refuses():
    def look(type=0, table=ONE, ldt=8, rows=5, k=8, ids=ONE, n=3, scale=1.0, out=ONE, ldo=8):
        return lib().blp_lookup(0, None, type, table, ldt, rows, k, ids, 0, n, scale, out, ldo)

    for args, what in (({"type": -1}, "type"), ({"rows": 0}, "table"), ({"n": -1}, "ids"), ({"n": 1 << 31}, "ids"), ({"k": 0}, "k must"),
                       ({"table": None}, "null"), ({"ids": None}, "null"), ({"out": None}, "null"), ({"ldt": 7}, "stride"),
                       ({"ldo": 7}, "stride"), ({"scale": float("nan")}, "scale")):
        refused(look(**args), what)
    assert look(n=0, table=None, ids=None, out=None) == 0  # nothing to do: nothing is touched

    def grad(type=0, g=ONE, ldg=8, ids=ONE, n=3, rows=5, k=8, scale=1.0, out=ONE, ldo=8, ws=ONE, ws_bytes=1 << 30):
        return lib().blp_lookup_grad(0, None, type, g, ldg, ids, 0, n, rows, k, scale, out, ldo, 0, ws, ws_bytes)

    for args, what in (({"type": 9}, "type"), ({"g": None}, "null"), ({"ids": None}, "null"), ({"out": None}, "null"), ({"ws": None}, "null"),
                       ({"ldg": 7}, "stride"), ({"ldo": 7}, "stride"), ({"ws_bytes": 0}, "workspace"), ({"ws": ONE + 8}, "aligned"),
                       ({"scale": float("inf")}, "scale")):
        refused(grad(**args), what)


def test_scores8_refuses():
    def quantize(type=0, x=ONE, ldx=8, rows=2, k=8, q=ONE, ldq=16, s=ONE):
        return lib().blp_quantize_rows(0, None, type, x, ldx, rows, k, q, ldq, s)

    for args, what in (({"type": 3}, "type"), ({"rows": -1}, "rows"), ({"k": 0}, "rows"), ({"x": None}, "null"), ({"q": None}, "null"),
                       ({"s": None}, "null"), ({"ldx": 7}, "stride"), ({"ldq": 7}, "stride")):
        refused(quantize(**args), what)
    assert quantize(rows=0, x=None, q=None, s=None) == 0

    def scores(q=ONE, ldq=16, s=ONE, t=ONE, ldt=16, ts=ONE, rows=2, cols=3, k=16, type=0, out=ONE, ldo=3, ws=None, ws_bytes=0):
        return lib().blp_scores8(0, None, q, ldq, s, t, ldt, ts, rows, cols, k, type, out, ldo, ws, ws_bytes)

    for args, what in (({"rows": -1}, "rows"), ({"cols": 0}, "rows"), ({"k": 0}, "k must"), ({"k": 1 << 17, "ldq": 1 << 17, "ldt": 1 << 17}, "k must"),
                       ({"type": 3}, "type"), ({"q": None}, "null"), ({"s": None}, "null"), ({"t": None}, "null"), ({"ts": None}, "null"),
                       ({"out": None}, "null"), ({"ldq": 15}, "stride"), ({"ldt": 15}, "stride"), ({"ldo": 2}, "stride"),
                       ({"ldq": (1 << 22) + 1}, "strides"), ({"k": 15}, "workspace"), ({"q": ONE + 1}, "workspace")):
        refused(scores(**args), what)
    for type, out in ((0, ONE + 2), (1, ONE + 1), (2, ONE + 1)):
        refused(scores(type=type, out=out), "aligned to its elements")
    assert scores(rows=0) == 0


def test_python_refuses_host_tensors():
    torch = pytest.importorskip("torch")
    x, ids = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for bad in (lambda: latent.lookup(x, ids), lambda: latent.lookup_grad(x, ids, 3), lambda: latent.softmax_loss(x, x, ids),
                lambda: latent.softmax_loss_grad(x, x, ids), lambda: latent.quantize_rows(x), lambda: latent.lookup([1.0], ids),
                lambda: latent.int8_scores(x.to(torch.int8), x[:, 0], x.to(torch.int8), x[:, 0]),
                lambda: latent.softmax_loss_backward(x[0], x[0], None, x, x, ids), lambda: latent.softmax_loss(x, None, ids)):
        with pytest.raises(ValueError):
            bad()
    assert blp.version()
