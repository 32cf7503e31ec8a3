"""What the latent-factor entry points launch, on the host (launches.py): the status of every launch, and grids that fit the work."""
import math

import pytest

from launches import run

ONE = 1 << 20  # a stand-in for a device pointer
STAGE = {1: 64, 2: 64, 3: 128}  # elements of k a stage, by the matrix instruction's type


def loss(type, m, n, k, grads=1, mean=1):
    return ("blp_softmax_loss", [0, None, type, ONE, k, ONE, k, ONE, 1, m, n, k, 1.0, ONE, ONE, ONE, mean, grads, ONE, k, ONE, k, ONE,
                                 1 << 50], None)


def backward(type, m, n, k):
    return ("blp_softmax_loss_backward", [0, None, type, ONE, k, ONE, k, ONE, 1, m, n, k, 1.0, ONE, ONE, 1, None, ONE, k, ONE, k, ONE,
                                          1 << 50], None)


@pytest.mark.parametrize("type,m,n,k", [(1, 16384, 87300, 200), (0, 14875, 70587, 104), (0, 15162, 62966, 104), (2, 16000, 20011, 136), (1, 131072, 1100, 136),
                                        (1, 8192, 100000, 1024), (2, 1537, 40961, 384), (0, 9000, 24011, 72)])
def test_every_slice_of_a_product_has_stages(type, m, n, k):
    """The last piece of the catalogue is narrower than the others: its gradient product takes fewer slices."""
    for got in run([loss(type, m, n, k), backward(type, m, n, k)]):
        assert got["rc"] == 0, got["error"]
        products = [(x["grid"], x["product"]) for x in got["launches"] if x["product"]]
        assert len(products) >= 3
        for grid, p in products:
            assert grid[1] == math.ceil(p["segments"] * math.ceil(p["k"] / STAGE[p["type"]]) / p["slice"]), (grid, p)


def lookup_grad(type, n, rows, k):
    return ("blp_lookup_grad", [0, None, type, ONE, k, ONE, 1, n, rows, k, 1.0, ONE, k, 0, ONE, 1 << 50], None)


def scores8(m, n, k, type, out=ONE, ldo=None):
    return ("blp_scores8", [0, None, ONE, k, ONE, ONE, k, ONE, m, n, k, type, out, ldo or n, ONE, 1 << 50], None)


CALLS = {
    "loss_narrow": loss(1, 500, 3000, 64), "loss_narrow_f32": loss(0, 2000, 30011, 50), "loss_wide": loss(1, 600, 3000, 200),
    "loss_pieces": loss(1, 16384, 87300, 200), "loss_pieces_f32": loss(0, 9000, 24011, 72), "loss_forward": loss(2, 3000, 9000, 72, grads=0),
    "loss_no_rows": loss(1, 0, 3000, 64), "backward_narrow": backward(2, 500, 3000, 64), "backward_wide": backward(0, 600, 3000, 200),
    "lookup": ("blp_lookup", [0, None, 1, ONE, 64, 5000, 64, ONE, 1, 3000, 2.0, ONE, 64], None),
    "lookup_grad_short": lookup_grad(0, 3000, 500, 64), "lookup_grad_long": lookup_grad(1, 300000, 50000, 64),
    "quantize": ("blp_quantize_rows", [0, None, 0, ONE, 64, 500, 64, ONE, 64, ONE], None),
    "scores8_narrow": scores8(500, 3000, 64, 0), "scores8_strips": scores8(10000, 99998, 64, 1), "scores8_slices": scores8(10, 1266, 6462, 1),
    "scores8_wide": scores8(4096, 16384, 4096, 1),
}


@pytest.mark.parametrize("name", CALLS)
def test_the_status_of_every_launch_is_returned(name):
    """Each launch of the call in turn fails as the runtime says: the call does, and launches nothing more."""
    fn, args, _ = CALLS[name]
    (whole,) = run([(fn, args, None)])
    assert whole["rc"] == 0, whole["error"]
    n = len(whole["launches"])
    assert n > 0
    at = sorted(set(range(min(n, 24))) | set(range(max(n - 24, 0), n)))
    for i, got in zip(at, run([(fn, args, (i, 2)) for i in at])):
        assert got["rc"] != 0 and got["error"], "launch %d of %d (%s) failed unseen" % (i, n, whole["launches"][i]["name"])
        assert len(got["launches"]) == i + 1


@pytest.mark.parametrize("scale", [2e38, 3.4e38, -3e38])
def test_scales_whose_product_with_log2_e_is_no_float_are_refused(scale):
    fn, args, _ = loss(1, 100, 300, 64)
    args[12] = scale
    (got,) = run([(fn, args, None)])
    assert got["rc"] == -1 and "scale" in got["error"] and not got["launches"]
    args[12] = 2.0 ** 127
    assert run([(fn, args, None)])[0]["rc"] == 0


def quantize(type, rows, k):
    return ("blp_quantize_rows", [0, None, type, ONE, k, rows, k, ONE, k, ONE], None)


HUGE = {
    # 2^26 rows of 64 lanes each: 2^32 threads
    "quantize": [quantize(1, 1 << 26, 513), quantize(0, (1 << 27) + 5, 300), quantize(2, (1 << 31) - 1, 8), quantize(0, (1 << 31) - 1, 1 << 12)],
    "scores8_outer": [scores8(129, 1 << 29, 64, 1), scores8(129, 1 << 28, 64, 0)],
    "scores8_strips": [scores8(1 << 30, 33, 64, 1), scores8((1 << 31) - 1, 35, 128, 2)],
    "loss_forward": [loss(1, 1 << 29, 1000, 8, grads=0), loss(0, (1 << 31) - (1 << 16), 77, 3, grads=0), loss(2, 1 << 30, 5, 200, grads=0)],
    "loss_step": [loss(1, 1 << 29, 1000, 8), loss(0, 1 << 29, 1000, 130), loss(1, 1000, 1 << 30, 64), backward(1, 1 << 30, 300, 8),
                  backward(0, (1 << 31) - (1 << 16), 100000, 1), backward(1, 100000, (1 << 31) - (1 << 16), 8)],
    "lookup": [("blp_lookup", [0, None, 0, ONE, 1 << 20, 5000, 1 << 20, ONE, 1, 1 << 20, 2.0, ONE, 1 << 20], None),
               lookup_grad(1, (1 << 31) - 1, 100, 8), lookup_grad(0, 5, (1 << 31) - 1, 8), lookup_grad(1, 1 << 24, 1000, 1 << 12)],
}


@pytest.mark.parametrize("name", HUGE)
def test_sizes_that_are_accepted_are_launched(name):
    """No launch has 2^32 threads or more, and none is refused by the runtime, at the largest sizes that memory could hold."""
    for got in run(HUGE[name]):
        assert got["rc"] == 0, got["error"]
        for l in got["launches"]:
            assert l["grid"][0] * l["block"][0] < 1 << 32, l


def test_more_scores_than_tiles_can_be_counted_are_refused():
    """Before anything is packed."""
    for k in (64, 300, 15):
        (got,) = run([scores8((1 << 31) - 1, (1 << 31) - 1, k, 1)])
        assert got["rc"] == -1 and "2^45" in got["error"] and not got["launches"]


@pytest.mark.parametrize("m,n,k", [((1 << 31) - (1 << 16), 1000, 1 << 20), (1000, (1 << 31) - (1 << 16), 1 << 11)])
def test_more_elements_than_tiles_can_be_counted_are_refused(m, n, k):
    """Before anything is packed."""
    for got in run([loss(1, m, n, k), backward(0, m, n, k)]):
        assert got["rc"] == -1 and "2^41" in got["error"] and not got["launches"]


def test_grids_fit_31_bits():
    for m, n, k in (((1 << 31) - (1 << 16), 1 << 10, 1 << 10), (1 << 10, (1 << 31) - (1 << 16), 1 << 10), (1 << 21, 1 << 21, 1 << 20)):
        for got in run([loss(t, m, n, k) for t in (0, 1)] if m * n < 1 << 42 else [loss(1, m, n, k, grads=0)]):
            assert got["rc"] == 0, got["error"]
            for l in got["launches"]:
                assert l["grid"][0] * l["block"][0] < 1 << 32
                if l["product"]:
                    assert 0 < l["product"]["tiles_p"] * l["product"]["tiles_q"] < 1 << 31
