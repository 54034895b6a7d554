"""rsx.score_logprobs_grad and rsx.add_rows against the chain rule in 64 bits.

Tolerances, elementwise.  Write c_ri for the size of the p part of dz: scale p (|sum g| + |h| (|log p| + H + 1)).  p is off by
ep = ez + 1.2e-5 of itself (ez: the scores' (3 d + 3) 2^-24 scale sum |x||y|; the exponent's rounding, as for the forward pass; lse is the
call's own input).  dz is a pair of halves (2^-22 of itself, or 2^-37 of the row's weight w where halves end) or one bf16 (2^-8); the
rows it multiplies are off by 3 2^-24; n terms summed in fp32 are off by 3 n 2^-24 of their absolute sum.  So a gradient by sum c |y| is
off by (ep + 2^-22 + 3 n 2^-24 + 2^-20 [or 2^-8]) sum c |y| + 2^-37 w scale n max |y|, the named items' part by 2^-20 [bf16 item rows:
2^-8] of sum |g| |y| scale, and the result is rounded to its type."""
import math

import numpy as np
import pytest

from test_logprob import reference, seen_csr, tables


def gradient(P, Q, users, items, g, h, lse, ent, mask, scale):
    """(GP, GQ, bounds' sums) in 64 bits from the call's own lse and entropies"""
    n, I, d = len(users), *Q.shape
    GP, GQ = np.zeros((n, d)), np.zeros((I, d))
    cP, cQ, gP, gQ = np.zeros((n, d)), np.zeros((I, d)), np.zeros((n, d)), np.zeros((I, d))
    ez, w, wP = 0.0, np.zeros(n), np.zeros(n)
    Qf = np.where(np.isfinite(Q), Q, 0.0)
    for r, u in enumerate(users):
        if not 0 <= u < P.shape[0] or lse[r] == -np.inf:
            continue
        keep = np.ones(I, bool)
        if mask is not None:
            ids = mask[1][mask[0][u]:mask[0][u + 1]]
            keep[ids[(ids >= 0) & (ids < I)]] = False
        with np.errstate(invalid="ignore"):
            lp = np.where(keep, scale * (Q @ P[u]) - lse[r], -np.inf)
            ez = max(ez, (3 * d + 3) * 2.0 ** -24 * scale * (np.abs(Q[keep]) @ np.abs(P[u])).max(initial=0.0))
        p = np.exp(lp)
        lp = np.where(keep, lp, 0.0)
        dz, sg, hot = np.zeros(I), 0.0, np.zeros(I)
        for t in range(items.shape[1] if items is not None else 0):
            i = items[r, t]
            if 0 <= i < I and keep[i]:
                dz[i] += g[r, t]
                hot[i] += abs(g[r, t])
                sg += g[r, t]
                w[r] += abs(g[r, t])
        hr, H = (h[r], ent[r]) if h is not None else (0.0, 0.0)
        w[r] += abs(hr)
        dz = scale * (dz - p * (sg + hr * (lp + H)))
        c = scale * p * (abs(sg) + abs(hr) * (np.abs(lp) + abs(H) + 1))
        GP[r] = dz @ Qf
        GQ += dz[:, None] * P[u]
        cP[r], gP[r] = c @ np.abs(Qf), scale * (hot @ np.abs(Qf))
        cQ += c[:, None] * np.abs(P[u])
        gQ += scale * hot[:, None] * np.abs(P[u])
        wP[r] = w[r] * np.abs(P[u]).max()
    return GP, GQ, cP, cQ, gP, gQ, ez, w, wP, np.abs(Qf).max()


def check(P, Q, users, items, g, h, mask, scale=1.0):
    import torch
    from recsys_pytorch_amd import rsx
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a, t)).cuda()
    bf16 = P.dtype == torch.bfloat16
    u, it = dev(users, np.int32), None if items is None else dev(items, np.int32)
    m = None if mask is None else (dev(mask[0], np.int64), dev(mask[1], np.int32))
    fwd = rsx.score_logprobs(P, Q, u, it, mask=m, scale=scale)
    kw = dict(mask=m, scale=scale)
    if h is not None:
        kw.update(entropy=fwd.entropy, g_entropy=dev(h, np.float32))
    gt = None if g is None else dev(g, np.float32)
    GP, GQ = rsx.score_logprobs_grad(P, Q, u, it, fwd.lse, gt, **kw)
    assert GP.dtype == P.dtype and GQ.dtype == P.dtype and GP.shape == (len(users), P.shape[1]) and GQ.shape == Q.shape
    f64 = lambda t: t.double().cpu().numpy()
    g64 = None if g is None else np.asarray(g, np.float32).astype(np.float64)
    h64 = None if h is None else np.asarray(h, np.float32).astype(np.float64)
    wP_, wQ_, cP, cQ, gP, gQ, ez, w, wP, topQ = gradient(f64(P), f64(Q), users, items, g64, h64, f64(fwd.lse), f64(fwd.entropy), mask, scale)
    n, I = len(users), Q.shape[0]
    ep, step, out = ez + 1.2e-5, 2.0 ** -8 if bf16 else 2.0 ** -22 + 2.0 ** -20, 2.0 ** -8 if bf16 else 2.0 ** -24
    tP = (ep + step + 3 * I * 2.0 ** -24) * cP + 2.0 ** -20 * gP + 2.0 ** -37 * scale * I * topQ * w[:, None] + out * np.abs(wP_) + 1e-37
    tQ = (ep + step + 3 * n * 2.0 ** -24) * cQ + (step + 3 * n * 2.0 ** -24) * gQ + 2.0 ** -37 * scale * n * wP.max() + out * np.abs(wQ_) + 1e-37
    for got, want, tol, name in ((f64(GP), wP_, tP, "GP"), (f64(GQ), wQ_, tQ, "GQ")):
        err = np.abs(got - want)
        assert (err <= tol).all(), (name, err.max(), float((err / tol).max()), np.abs(want).max())
    again = rsx.score_logprobs_grad(P, Q, u, it, fwd.lse, gt, **kw)
    assert torch.equal(GP, again[0]) and torch.equal(GQ, again[1])
    return GP, GQ


# ---- CPU -------------------------------------------------------------------------------------------------------------------------------
def test_the_chain_rule_against_differences():
    """the oracle of these tests against central differences of the forward's oracle"""
    rng = np.random.default_rng(0)
    U, I, d, n, T = 4, 13, 5, 4, 3
    P, Q = rng.standard_normal((U, d)), rng.standard_normal((I, d))
    users, items = np.array([0, 2, 2, 3]), rng.integers(0, I, (n, T))
    items[1, 1], items[2] = items[1, 0], [-1, 13, 4]                  # the same item twice; ids that name nothing
    g, h = rng.standard_normal((n, T)), rng.standard_normal(n)
    mask = seen_csr(rng, U, I, 6)

    def value(P, Q):
        logp, lse, ent, *_ = reference(P, Q, users, items, 0, mask, 0.7)
        return float((g * np.where(np.isfinite(logp), logp, 0.0)).sum() + (h * ent).sum())
    _, lse, ent, *_ = reference(P, Q, users, items, 0, mask, 0.7)
    GP, GQ, *_ = gradient(P, Q, users, items, g, h, lse, ent, mask, 0.7)
    dP = np.zeros_like(P)
    np.add.at(dP, users, GP)
    for table, grad in ((P, dP), (Q, GQ)):
        for at in np.ndindex(*table.shape):
            old, e = table[at], 1e-5
            table[at] = old + e
            up = value(P, Q)
            table[at] = old - e
            down = value(P, Q)
            table[at] = old
            assert abs((up - down) / (2 * e) - grad[at]) < 1e-7


def test_refusals():
    import torch
    from recsys_pytorch_amd import build, rsx
    build.build()
    P, ids = torch.zeros(4, 32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: rsx.score_logprobs_grad(P, P, ids, None, ids.float(), None), lambda: rsx.score_logprobs_grad_workspace(4, 0, 32),
                 lambda: rsx.score_logprobs_grad_workspace(4, 10, 32, T=-1), lambda: rsx.score_logprobs_grad_workspace(2 ** 31, 10, 32), lambda: rsx.add_rows(P, ids, P[:2]),
                 lambda: rsx.add_rows(P.double(), ids, P[:2])):
        with pytest.raises(rsx.RsxError):
            call()
    L = rsx.lib()
    good = dict(P=16, U=4, ids=16, n=2, Q=16, I=300, d=32, dt=0, mp=None, mi=None, scale=1.0, items=16, T=1, lse=16, g=16, ent=None, h=None, GP=32, GQ=48)

    def call(**kw):
        k = {**good, **kw}
        return L.rsx_score_logprobs_grad(k["P"], k["U"], k["ids"], k["n"], k["Q"], k["I"], k["d"], k["dt"], k["mp"], k["mi"], k["scale"], k["items"], k["T"],
                                         k["lse"], k["g"], k["ent"], k["h"], k["GP"], k["GQ"], None, 0, None)
    for bad in (dict(P=None), dict(GQ=None), dict(GP=8), dict(lse=None), dict(n=0), dict(n=2 ** 31), dict(I=0), dict(d=100), dict(dt=3), dict(mi=16),
                dict(scale=-1.0), dict(GP=48), dict(GP=16), dict(GQ=16), dict(T=0), dict(g=None), dict(items=None), dict(ent=16), dict(h=16)):
        assert call(**bad) == -1, bad
    assert call() == -3 and b"workspace" in L.rsx_last_error() and call(T=0, items=None, g=None, ent=16, h=16) == -3
    assert L.rsx_add_rows(16, 4, 31, 16, 16, 0, 1, None) == -1 and L.rsx_add_rows(16, 0, 32, 16, 16, 0, 1, None) == -1
    assert L.rsx_add_rows(16, 4, 32, 16, 16, 2, 1, None) == -1 and L.rsx_add_rows(16, 4, 32, 16, 16, 0, 0, None) == 0


# ---- GPU -------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("n,I,T,masked,entropy,scale", [(1, 1, 1, False, False, 1.0), (1, 500, 1, True, True, 1.0), (7, 33, 3, True, False, 2.0), (32, 128, 1, False, True, 0.5),
                                                          (33, 1000, 0, True, True, 1.0), (129, 257, 2, True, True, 1.0), (300, 1503, 5, True, False, 1.0), (511, 129, 1, False, False, 1.0)])
def test_hip_logprobs_grad_vs_chain_rule(n, I, T, masked, entropy, scale, d, bf16):
    rng = np.random.default_rng(n * 31 + I + d)
    U = n + 3
    P, Q = tables(rng, U, I, d, bf16)
    items = rng.integers(0, I, (n, T)) if T else None
    g = rng.standard_normal((n, T)) / n if T else None
    check(P, Q, rng.integers(0, U, n), items, g, 0.3 * rng.standard_normal(n) / n if entropy else None, seen_csr(rng, U, I, 30) if masked else None, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
def test_hip_logprobs_grad_empty_rows_padding_and_values_in_masked_places(bf16):
    rng = np.random.default_rng(4)
    U, I, d, n = 9, 700, 64, 150
    P, Q = tables(rng, U, I, d, bf16)
    Q[100, 3], Q[101, :], Q[699, 0], Q[350, 5] = float("nan"), float("inf"), float("-inf"), float("nan")
    bad = [100, 101, 699, 350, -1, 700, 100]
    rows = [np.array(bad), np.arange(I), np.array(bad + list(range(3, 99)))] * 3
    mask = (np.concatenate([[0], np.cumsum([len(r) for r in rows])]), np.concatenate(rows))
    users = rng.integers(0, U, n)
    users[:5] = [-1, 1, 9, 2 ** 31 - 1, 0]
    items = rng.integers(0, I, (n, 4))
    items[:, 1], items[0], items[4] = -1, 700, [2 ** 31 - 1, 699, 100, 0]
    items[:, 3] = items[:, 2]                                            # the same item twice
    g = rng.standard_normal((n, 4))
    g[7] = [1.0, 5.0, -0.5, -0.5]                                        # weights that cancel
    g[8] = 0.0
    items[7, 0], items[7, 2:] = 5, 6
    GP, GQ = check(P, Q, users, items, g, None, mask)
    assert float(GP[:4].abs().max()) == 0.0 and float(GP[8].abs().max()) == 0.0      # nobody's row; everything masked; no weight
    check(P, Q, users, items, g, rng.standard_normal(n), mask, 0.5)


@pytest.mark.gpu
def test_hip_logprobs_grad_magnitudes():
    """weights and tables far from one: the half pairs are scaled to follow"""
    rng = np.random.default_rng(12)
    n, I, d = 70, 900, 128
    for up, weight in ((2.0 ** 30, 1e-12), (2.0 ** -30, 1e12), (1.0, 1e-30)):
        P, Q = tables(rng, n, I, d, False)
        check(P * up, Q / up, np.arange(n), rng.integers(0, I, (n, 2)), weight * rng.standard_normal((n, 2)), None, None)
    P, Q = tables(rng, n, I, d, False)
    Q[320:352] *= 1e-6
    P[3] = 0.0
    check(P, Q, np.arange(n), rng.integers(0, I, (n, 2)), rng.standard_normal((n, 2)) * np.logspace(-6, 0, n)[:, None], rng.standard_normal(n), None)


@pytest.mark.gpu
def test_hip_logprobs_grad_more_positions_than_one_pass():
    """9 000 positions of a million items hold 1.1 GB of seen bits: two passes.  Against the same call in three parts."""
    import torch
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(2)
    gen = torch.Generator(device="cuda").manual_seed(5)
    n, I, d = 9000, 1_000_000, 32
    P, Q = torch.randn(n, d, generator=gen, device="cuda") * 0.5, torch.randn(I, d, generator=gen, device="cuda") * 0.5
    u = torch.arange(n, dtype=torch.int32, device="cuda")
    t = torch.from_numpy(rng.integers(0, I, (n, 1)).astype(np.int32)).cuda()
    mask = tuple(torch.from_numpy(a).cuda() for a in (np.arange(n + 1) * 5, rng.integers(0, I, 5 * n).astype(np.int32)))
    g = torch.full((n, 1), -1.0 / n, device="cuda")
    lse = rsx.score_logprobs(P, Q, u, mask=mask).lse
    GP, GQ = rsx.score_logprobs_grad(P, Q, u, t, lse, g, mask=mask)
    parts = [rsx.score_logprobs_grad(P, Q, u[a:a + 3000], t[a:a + 3000], lse[a:a + 3000], g[a:a + 3000], mask=mask) for a in (0, 3000, 6000)]
    # each side is within 3 n 2^-24 sum c |P| + 2^-19 sum c |P| of the truth, c = p / n: |P| < 4 and sum over positions of p is at most GQ's own
    whole, summed = GQ, sum(p[1].double() for p in parts)
    assert torch.allclose(GP, torch.cat([p[0] for p in parts]), rtol=0, atol=2e-5 * float(GP.abs().max()))
    mass = torch.zeros(I, device="cuda")
    for a in range(0, n, 500):
        mass += torch.exp(P[a:a + 500] @ Q.T - lse[a:a + 500, None]).sum(0)
    mass[t[:, 0].long()] += torch.ones(n, device="cuda")
    tol = 2 * (3 * n * 2.0 ** -24 + 2.0 ** -19) * float(P.abs().max()) * mass / n + 2 * 2.0 ** -37 * float(P.abs().max())
    assert bool(((whole - summed).abs().max(1).values <= tol).all())


@pytest.mark.gpu
def test_hip_logprobs_train_step_captured():
    """forward and backward replayed from a graph over buffers that change, beside eager calls with their own workspaces"""
    import torch
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(9)
    n, I, d = 100, 1500, 64
    P, Q = tables(rng, n, I, d, False)
    u = torch.arange(n, dtype=torch.int32, device="cuda")
    t = torch.from_numpy(rng.integers(0, I, (n, 1)).astype(np.int32)).cuda()
    g = torch.full((n, 1), -1.0 / n, device="cuda")
    mask = tuple(torch.from_numpy(a).cuda() for a in seen_csr(rng, n, I, 30))

    def step(**ws):
        f = rsx.score_logprobs(P, Q, u, t, mask=mask, ws=ws.get("a"))
        return rsx.score_logprobs_grad(P, Q, u, t, f.lse, g, mask=mask, ws=ws.get("b"))
    wsa = torch.empty(rsx.score_logprobs_workspace(n, I, d, masked=True) // 8 + 1, dtype=torch.int64, device="cuda")
    wsb = torch.empty(rsx.score_logprobs_grad_workspace(n, I, d, masked=True) // 8 + 1, dtype=torch.int64, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a=wsa, b=wsb)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            held = step(a=wsa, b=wsb)
    for k in range(4):
        torch.cuda.synchronize()
        Q.mul_(1.1)
        wsb.random_()
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert torch.equal(held[0], eager[0]) and torch.equal(held[1], eager[1]), k


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 63, 1000, 40_000])
def test_hip_add_rows(n):
    """the sums of a row in the order of the positions, to the bit; ids that name nothing are skipped"""
    import torch
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(n)
    for d, bf16 in ((32, False), (128, True), (256, False)):
        rows = 500
        T = rng.standard_normal((rows, d)).astype(np.float32)
        ids = rng.integers(-3, rows + 3, n).astype(np.int32)
        R = torch.from_numpy(rng.standard_normal((n, d)).astype(np.float32))
        R = R.bfloat16() if bf16 else R
        got = rsx.add_rows(torch.from_numpy(T).cuda(), torch.from_numpy(ids).cuda(), R.cuda())
        want, vals = T.copy(), R.float().numpy()
        for r in range(n):
            if 0 <= ids[r] < rows:
                want[ids[r]] += vals[r]
        assert np.array_equal(got.cpu().numpy(), want)
