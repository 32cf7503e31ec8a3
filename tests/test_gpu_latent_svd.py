"""From DeviceSVD's factors to blp.latent and back: 8-bit scores, a training step, lists of the trained factors."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_factors_go_to_latent_and_back(gpu):
    torch = pytest.importorskip("torch")
    from blp import latent
    from blp.factor import DeviceSVD

    rng = np.random.default_rng(3)
    n_users, n_bus, k = 300, 500, 50
    svd = DeviceSVD(rng.standard_normal((n_users, k)) * 3 / k ** 0.5, rng.standard_normal((n_bus, k)), device=gpu)
    users = torch.from_numpy(svd.us).float().cuda()
    businesses = torch.from_numpy(svd.v).float().cuda()
    rows, cols = np.repeat(np.arange(n_users), 7), rng.integers(0, n_bus, 7 * n_users)
    want = svd.score_pairs(rows, cols)

    # 8-bit scores: each factor is off by half a scale at most (and 2^-24 of itself as float32)
    q, s = latent.quantize_rows(users)
    p, t = latent.quantize_rows(businesses)
    scores = latent.int8_scores(q, s, p, t).cpu().numpy().astype(np.float64)
    s, t = s.cpu().numpy().astype(np.float64), t.cpu().numpy().astype(np.float64)
    ax, aw = np.abs(svd.us).sum(1), np.abs(svd.v).sum(1)
    bound = 0.5 * ax[rows] * t[cols] + 0.5 * aw[cols] * s[rows] + 0.25 * k * s[rows] * t[cols]
    assert (np.abs(scores[rows, cols] - want) <= bound * 1.0001).all()

    # a step of training on some links, against the formulas in 64 bits; u = 2^-23, and the factors' own rounding is 2^-24
    ids, target = torch.from_numpy(rows).cuda(), torch.from_numpy(cols).cuda()
    loss, dx, dw = latent.softmax_loss_grad(latent.lookup(users, ids), businesses, target)
    du = latent.lookup_grad(dx, ids, n_users)
    U, W, u, m = svd.us[rows], svd.v, 2.0 ** -23, len(rows)
    z = U @ W.T
    S = (np.abs(U) @ np.abs(W).T).max(1)
    top = z.max(1)
    lse = np.log(np.exp(z - top[:, None]).sum(1)) + top
    p64 = np.exp(z - lse[:, None])
    d = p64.copy()
    d[np.arange(m), cols] -= 1
    dz = (k + 6) * u * S
    assert abs(float(loss) - (lse - z[np.arange(m), cols]).mean()) <= (2 * dz + (64 + n_bus / 64 + 8) * u + 8 * u * (np.abs(lse) + S)).max()
    r = 2 * dz + (64 + n_bus / 64 + 16) * u + 4 * u * (S + np.abs(lse))
    d, e = d / m, (p64 * r[:, None] + 2 * u) / m + u * np.abs(d / m)
    want_x, want_w = d @ W, d.T @ U
    off_x = e @ np.abs(W) + (n_bus + 9) * u * (np.abs(d) @ np.abs(W)) + u * np.abs(want_x)
    off_w = e.T @ np.abs(U) + (m + 9) * u * (np.abs(d).T @ np.abs(U)) + u * np.abs(want_w)
    assert (np.abs(dw.cpu().numpy() - want_w) <= off_w).all()
    want_u, off_u, sum_u = np.zeros_like(svd.us), np.zeros_like(svd.us), np.zeros_like(svd.us)
    for out, x in ((want_u, want_x), (off_u, off_x), (sum_u, np.abs(want_x) + off_x)):
        np.add.at(out, rows, x)
    assert (np.abs(du.cpu().numpy() - want_u) <= off_u + 9 * u * sum_u).all()
    trained = DeviceSVD((users - 0.5 * du).double().cpu().numpy(), (businesses - 0.5 * dw).double().cpu().numpy(), device=gpu)

    # the trained factors' lists are those of their own dense product
    at, _ = trained.topk(np.arange(40), 10)
    dense = trained.us[:40] @ trained.v.T
    np.testing.assert_allclose(np.sort(np.take_along_axis(dense, at, 1), 1), np.sort(dense, 1)[:, -10:], rtol=0, atol=2.0 ** -50 * np.abs(dense).max() * k)
