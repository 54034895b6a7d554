"""rsx.score_logprobs_grad where values lie far apart: item rows and weights of very unequal size, probabilities far below one, masked rows of large
finite values.  Every row of GP and GQ is held to the size of its OWN sum, not to the table's or the batch's largest element.

Tolerance of an element, c_ri the size of the p part of dz_ri (as in test_logprob_grad.py), hot_ri that of its named part: the p part is off by
  e_ri = (3 d + 3) 2^-24 scale sum |P_r||Q_i|  (the score)  +  1.2e-5  (exponent: two half steps of |t| < 128, the exponential)
of itself, times |y|; dz is a pair of halves (fp32 tables: 2^-22 of itself) or one half (bf16 tables: 2^-11), the rows it multiplies are off by 2^-21
(scaled, split; bf16: exact); sums of n terms by 3 n 2^-24; the named part by the same without e_ri (in GP it is added in fp32).  Halves end:
2^-25 of a unit that the largest |dz| |y| of the SAME sum holds at 2^7 or more, rows within a power of two of their scale and, where 32 item
rows share one, within 2^12: 2^-31 n max_j |dz_j| S_j, S_j the row's largest element, or its 32 neighbours' where that is at most 4096 times larger.
The result is rounded once."""
import numpy as np
import pytest

from test_logprob import seen_csr, tables


def within(P, Q, users, items, g, h, mask, scale=1.0, lse=None):
    """the call against the chain rule in 64 bits, every row within its own bound"""
    import torch
    from recsys_pytorch_amd import rsx
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a, t)).cuda()
    f64 = lambda t: t.double().cpu().numpy()
    bf16 = P.dtype == torch.bfloat16
    u, it = dev(users, np.int32), None if items is None else dev(items, np.int32)
    m = None if mask is None else (dev(mask[0], np.int64), dev(mask[1], np.int32))
    f = rsx.score_logprobs(P, Q, u, it, mask=m, scale=scale)
    lse = f.lse if lse is None else dev(lse, np.float32)
    kw = dict(mask=m, scale=scale)
    if h is not None:
        kw.update(entropy=f.entropy, g_entropy=dev(h, np.float32))
    GP, GQ = rsx.score_logprobs_grad(P, Q, u, it, lse, None if g is None else dev(g, np.float32), **kw)
    x, Q64, l64 = f64(P)[users], f64(Q), f64(lse)
    (n, d), I = x.shape, Q64.shape[0]
    keep = np.ones((n, I), bool)
    if mask is not None:
        for r, who in enumerate(users):
            keep[r, mask[1][mask[0][who]:mask[0][who + 1]]] = False
    with np.errstate(invalid="ignore", over="ignore"):
        lp = np.where(keep, scale * (x @ Q64.T) - l64[:, None], -np.inf)
        size = np.where(keep, scale * (np.abs(x) @ np.abs(Q64).T), 0.0)
    p = np.exp(lp)
    lp = np.where(keep, lp, 0.0)
    dz, hot = np.zeros((n, I)), np.zeros((n, I))
    for t in range(0 if items is None else items.shape[1]):
        np.add.at(dz, (np.arange(n), items[:, t]), np.float32(g[:, t]))
        np.add.at(hot, (np.arange(n), items[:, t]), np.abs(np.float32(g[:, t])))
    dz, hot = dz * keep, hot * keep
    sg = dz.sum(1)[:, None]
    hr = np.zeros((n, 1)) if h is None else np.float32(h)[:, None].astype(np.float64)
    H = f64(f.entropy)[:, None] if h is not None else np.zeros((n, 1))
    p = np.where(p > 0, p, 0.0)
    c = scale * p * (np.abs(sg) + np.abs(hr) * (np.abs(lp) + np.abs(H) + 1))
    dz = scale * (dz - p * (sg + hr * (lp + H)))
    hot *= scale
    e = (3 * d + 3) * 2.0 ** -24 * size + 1.2e-5
    step, rows, out = (2.0 ** -11, 0.0, 2.0 ** -8) if bf16 else (2.0 ** -22, 2.0 ** -21, 2.0 ** -24)
    aQ = np.where(keep.any(0)[:, None], np.abs(Q64), 0.0)
    yQ = np.where(keep.any(0)[:, None], Q64, 0.0)
    big = np.abs(Q64).max(1)
    tile = np.repeat(np.maximum.reduceat(big, np.arange(0, I, 32)), 32)[:I]
    S = np.minimum(tile, 4096 * big)
    ax = np.abs(x)
    wantP, wantQ = dz @ yQ, dz.T @ x
    tP = (c * (e + step + rows + 3 * I * 2.0 ** -24)) @ aQ + (2.0 ** -20 + 3 * items.shape[1] * 2.0 ** -24 if items is not None else 0.0) * (hot @ aQ)
    tP += 2.0 ** -31 * I * ((c + hot) * S).max(1)[:, None] + out * np.abs(wantP) + 1e-37
    tQ = (c * (e + step + rows + 3 * n * 2.0 ** -24) + hot * (step + rows + 2.0 ** -22 + 3 * n * 2.0 ** -24)).T @ ax
    tQ += 2.0 ** -31 * n * ((c + hot) * ax.max(1)[:, None]).max(0)[:, None] + out * np.abs(wantQ) + 1e-37
    for got, want, tol, name in ((f64(GP), wantP, tP, "GP"), (f64(GQ), wantQ, tQ, "GQ")):
        err = np.abs(got - want)
        bad = ~(err <= tol)
        assert not bad.any(), (name, int(bad.any(1).sum()), float(np.nanmax(err / tol)), np.argwhere(bad)[0])
    return GP, GQ


@pytest.mark.gpu
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_hip_gradient_of_probabilities_far_below_one(d, entropy):
    """standard normal tables, as a model starts with: most items' probabilities are 2^-30 and less in every row, and their GQ rows are sums of those"""
    import torch
    rng = np.random.default_rng(d)
    n, I = 96, 2500
    P, Q = (torch.from_numpy(rng.standard_normal((r, d)).astype(np.float32)).cuda() for r in (n, I))
    g = rng.standard_normal((n, 1)) / n
    within(P, Q, rng.permutation(n), rng.integers(0, I, (n, 1)), g, 0.1 * rng.standard_normal(n) / n if entropy else None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size,d", [(1e4, 64), (1e6, 64), (1e9, 64), (1e25, 64), (1e9, 32), (1e9, 128), (1e9, 256)])
def test_hip_gradient_beside_masked_rows_of_large_values(size, d, bf16, entropy):
    rng = np.random.default_rng(7)
    n, I = 150, 700
    P, Q = tables(rng, n, I, d, bf16)
    bad = [0, 3, 350, 699]
    Q[bad] *= size
    mask = (np.arange(n + 1, dtype=np.int64) * len(bad), np.tile(np.asarray(bad, np.int32), n))
    items = rng.integers(0, I, (n, 2))
    items[:, 1] = np.where(np.isin(items[:, 1], bad), 5, items[:, 1])
    GP, GQ = within(P, Q, np.arange(n), items, rng.standard_normal((n, 2)) / n, rng.standard_normal(n) / n if entropy else None, mask)
    assert not GQ[bad].any()


@pytest.mark.gpu
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
def test_hip_gradient_beside_an_item_of_probability_zero(bf16, entropy):
    """one unmasked row a million times the others, its score -3 10^6 for everybody"""
    rng = np.random.default_rng(3)
    n, I = 100, 400
    P, Q = tables(rng, n, I, 128, bf16)
    P[:, 0] = 3.0
    Q[70] = 0.0
    Q[70, 0] = -1e6
    items = rng.integers(0, I, (n, 1))
    items[items == 70] = 0
    within(P, Q, np.arange(n), items, rng.standard_normal((n, 1)), rng.standard_normal(n) if entropy else None, None)


@pytest.mark.gpu
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
def test_hip_gradient_of_weights_and_rows_of_many_sizes(d, bf16, entropy):
    """weights from 10^-12 to 1 and user rows from 10^-3 to 1 in one batch, item rows from 10^-6 to 1 side by side"""
    import torch
    rng = np.random.default_rng(5)
    n, I = 130, 600
    P, Q = tables(rng, n, I, d, bf16)
    f = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()
    P = (P.float() * f(np.logspace(-3, 0.3, n))[:, None]).to(P.dtype)
    Q = (Q.float() * f(10.0 ** rng.uniform(-6, 0, (I, 1)))).to(Q.dtype)
    Q[64:96] = 0.0
    w = 10.0 ** rng.uniform(-12, 0, n)
    within(P, Q, rng.permutation(n), rng.integers(0, I, (n, 5)), rng.standard_normal((n, 5)) * w[:, None], rng.standard_normal(n) * w if entropy else None,
           seen_csr(rng, n, I, 20))


@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("n,I,T,masked,entropy", [(6, 300, 1, False, False), (200, 900, 7, True, False), (70, 130, 3, True, True)])
def test_hip_gradient_of_bf16_tables_to_the_results_rounding(n, I, T, masked, entropy, d):
    """dz is not rounded to bf16 on its way: sums that cancel show it"""
    rng = np.random.default_rng(n + d)
    P, Q = tables(rng, n, I, d, True)
    within(P, Q, rng.permutation(n), rng.integers(0, I, (n, T)), rng.standard_normal((n, T)) / n, rng.standard_normal(n) / n if entropy else None,
           seen_csr(rng, n, I, 30) if masked else None)


@pytest.mark.gpu
@pytest.mark.parametrize("weight", [1.0, -3.0])
def test_hip_gradient_of_one_probability(weight):
    """one item, scores of 64 to 127 binades: scale = ln 2, so that the operands (x scale log2 e in 22 bits) are exact to 2^-28 and z log2 e to 2^-21.  p = exp(z - lse) of
    the lse that is handed in: the exponent's half step where it is below 1 is 2^-25, the exponential is off by 2^-23, the half pair by 2^-22, the row by 2^-22,
    z by 2^-21: 1.1e-6; nothing of the normaliser's own size (half a step at 127 is 2.6e-6 of p)"""
    import torch
    from recsys_pytorch_amd import rsx
    n, d, scale = 64, 32, float(np.float32(np.log(2)))
    rng = np.random.default_rng(1)
    P, Q = torch.zeros(n, d), torch.zeros(1, d)
    P[:, 0], Q[0, 0], Q[0, 1] = torch.arange(64, 64 + n) / 8.0, 8.0, 1.0
    z = (P[:, 0] * 8.0).double().numpy() * scale
    lse = np.float32(z + rng.uniform(0.0, 0.01, n))
    p = np.exp(z - lse.astype(np.float64))
    dev = lambda a, t=np.float32: torch.from_numpy(np.ascontiguousarray(a, t)).cuda()
    GP, GQ = rsx.score_logprobs_grad(P.cuda(), Q.cuda(), dev(np.arange(n), np.int32), dev(np.zeros((n, 1)), np.int32), dev(lse), dev(np.full((n, 1), weight)), scale=scale)
    # 1 - p of two numbers near 1: their own roundings (2^-24 each) and the result's beside p's
    want, tol = weight * scale * (1 - p), abs(weight) * scale * (1.1e-6 + 2.0 ** -23)
    assert (np.abs(GP[:, 1].double().cpu().numpy() - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [32, 256])
def test_hip_gradient_of_many_named_items(d, bf16, entropy):
    """70 names a position, one item up to all 70 times: their sum in one cell stays within a half"""
    rng = np.random.default_rng(d)
    n, I, T = 45, 140, 70
    P, Q = tables(rng, n, I, d, bf16)
    items = rng.integers(0, I, (n, T))
    items[:5] = 33
    items[5:9, ::2] = rng.integers(0, 3, (4, 35))
    within(P, Q, rng.permutation(n), items, rng.standard_normal((n, T)) + 0.7, rng.standard_normal(n) if entropy else None, seen_csr(rng, n, I, 6))
