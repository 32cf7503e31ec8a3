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


@pytest.mark.parametrize("type,m,n,k", [(1, 16384, 87300, 200), (0, 14875, 70587, 104), (2, 16000, 20011, 136), (1, 131072, 1100, 136),
                                        (1, 8192, 100000, 1024), (2, 1537, 40961, 384), (0, 9000, 24011, 72)])
def test_every_slice_of_a_product_has_stages(type, m, n, k):
    """The last piece of the catalogue is narrower than the others: its gradient product takes fewer slices."""
    for got in run([loss(type, m, n, k), backward(type, m, n, k)]):
        assert got["rc"] == 0, got["error"]
        products = [(x["grid"], x["product"]) for x in got["launches"] if x["product"]]
        assert len(products) >= 3
        for grid, p in products:
            assert grid[1] == math.ceil(p["segments"] * math.ceil(p["k"] / STAGE[p["type"]]) / p["slice"]), (grid, p)
