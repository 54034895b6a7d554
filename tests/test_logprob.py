"""rsx.score_logprobs against the definition in 64 bits.

Tolerances.  A score is a sum of at most 3 d products of 16-bit parts (or d fp32 / bf16 products), each off by at most 3 half steps
2^-24, summed in fp32: |dz| <= (3 d + 3) 2^-24 scale sum |x||y| =: ez (per row, its largest).  2^(t - m): the fused multiply-add and the
factor are off by 3 half steps of |t| <= 60 (what is further below adds nothing), the exponential by 2 steps: 60 * 3 * 2^-24 + 2^-22
< 1.2e-5.  A lane sums at most 512 terms (64 a group of 128 items; the sizes here give a lane at most 8 groups), then joins: 600
half steps, 3.6e-5.  Together: |d lse| <= ez + 5e-5 =: el.  The entropy is sum p |log p| of the same terms, log p <= 45 + rounding:
|dH| <= el (2 + H) + ez.  Log-probabilities of items: 64-bit products minus lse, rounded once: el + 2^-24 |logp|.
The Top-K ids are those of the 64-bit products, exactly."""
import math

import numpy as np
import pytest


def reference(P, Q, users, items, K, mask, scale):
    """(logp, lse, entropy, top_idx, top_logp, ez) in 64 bits; P, Q float64 arrays, mask = (indptr, indices) or None"""
    U, I = P.shape[0], Q.shape[0]
    n = len(users)
    lse, ent, ez = np.full(n, -np.inf), np.zeros(n), np.zeros(n)
    T = 0 if items is None else items.shape[1]
    logp, top, topv = np.zeros((n, T)), np.full((n, K), -1, np.int64), np.full((n, K), -np.inf)
    for r, u in enumerate(users):
        if not 0 <= u < U:
            continue
        keep = np.ones(I, bool)
        if mask is not None:
            ids = mask[1][mask[0][u]:mask[0][u + 1]]
            keep[ids[(ids >= 0) & (ids < I)]] = False
        with np.errstate(invalid="ignore", over="ignore"):
            z = np.where(keep, (Q * P[u]).sum(1) * scale, -np.inf)
            ez[r] = (3 * P.shape[1] + 3) * 2.0 ** -24 * scale * max([0.0, *(np.abs(Q[keep]) * np.abs(P[u])).sum(1)])
        if keep.any():
            m = z.max()
            e = np.exp(z - m)
            lse[r] = m + math.log(e.sum())
            p = e / e.sum()
            ent[r] = -(p[p > 0] * np.log(p[p > 0])).sum()
        for t in range(T):
            i = items[r, t]
            if 0 <= i < I:
                logp[r, t] = z[i] - lse[r] if keep[i] else -np.inf
        order = np.argsort(-z, kind="stable")[:K]
        order = order[keep[order]]
        top[r, :len(order)] = order
        topv[r, :len(order)] = z[order] - lse[r]
    return logp, lse, ent, top, topv, ez


def close(got, want, tol):
    got, want = got.double().cpu().numpy(), np.asarray(want)
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine])
    err = np.abs(got[fine] - want[fine])
    tol = np.broadcast_to(tol, want.shape)[fine]
    assert (err <= tol).all(), (err.max(), tol[err.argmax()])


def tables(rng, users, items, d, bf16, sd=None):
    import torch
    sd = (4.0 / d) ** 0.25 if sd is None else sd
    P = torch.from_numpy((rng.standard_normal((users, d)) * sd).astype(np.float32)).cuda()
    Q = torch.from_numpy((rng.standard_normal((items, d)) * sd * np.exp(0.3 * rng.standard_normal((items, 1)))).astype(np.float32)).cuda()
    return (P.bfloat16(), Q.bfloat16()) if bf16 else (P, Q)


def seen_csr(rng, users, items, most):
    deg = rng.integers(0, min(most, items) + 1, users)
    indptr = np.concatenate([[0], np.cumsum(deg)]).astype(np.int64)
    indices = np.concatenate([rng.choice(items, k, replace=False) for k in deg] + [np.zeros(0)]).astype(np.int32)     # unsorted
    return indptr, indices


def check(P, Q, users, items, K, mask, scale=1.0, ws=None, rows=None):
    """the call against the reference (of the positions `rows`)"""
    import torch
    from recsys_pytorch_amd import rsx
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a, t)).cuda()
    got = rsx.score_logprobs(P, Q, dev(users, np.int32), None if items is None else dev(items, np.int32), K=K,
                             mask=None if mask is None else (dev(mask[0], np.int64), dev(mask[1], np.int32)), scale=scale, ws=ws)
    pick = slice(None) if rows is None else rows
    logp, lse, ent, top, topv, ez = reference(P.double().cpu().numpy(), Q.double().cpu().numpy(), users[pick], None if items is None else items[pick], K, mask, scale)
    el = ez + 5e-5
    close(got.lse[pick], lse, el + 2.0 ** -24 * np.abs(np.where(np.isfinite(lse), lse, 0)))
    close(got.entropy[pick], ent, el * (2 + ent) + ez)
    if items is not None:
        close(got.logp[pick], logp, el[:, None] + 2.0 ** -24 * np.abs(np.where(np.isfinite(logp), logp, 0)))
    else:
        assert got.logp is None
    if K:
        assert np.array_equal(got.top_idx[pick].cpu().numpy(), top)
        close(got.top_logp[pick], topv, el[:, None] + 2.0 ** -24 * np.abs(np.where(np.isfinite(topv), topv, 0)))
    return got


# ---- refusals (no GPU) -----------------------------------------------------------------------------------------------------------
def test_refusals():
    import torch
    from recsys_pytorch_amd import build, rsx
    build.build()
    P, ids = torch.zeros(4, 32), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: rsx.score_logprobs(P, P, ids), lambda: rsx.score_logprobs(P.half(), P.half(), ids),
                 lambda: rsx.score_logprobs_workspace(4, 0, 32), lambda: rsx.score_logprobs_workspace(4, 10, 48), lambda: rsx.score_logprobs_workspace(4, 10, 32, K=129),
                 lambda: rsx.score_logprobs_workspace(4, 10, 32, torch.float16), lambda: rsx.score_logprobs_workspace(-1, 10, 32)):
        with pytest.raises(rsx.RsxError):
            call()
    L = rsx.lib()
    good = dict(P=16, U=4, ids=16, n=2, Q=16, I=300, d=32, dt=0, mp=None, mi=None, scale=1.0, items=None, T=0, K=0, logp=None, idx=None, val=None)

    def call(**kw):
        k = {**good, **kw}
        return L.rsx_score_logprobs(k["P"], k["U"], k["ids"], k["n"], k["Q"], k["I"], k["d"], k["dt"], k["mp"], k["mi"], k["scale"], k["items"], k["T"],
                                    k["K"], k["logp"], None, None, k["idx"], k["val"], None, 0, None)
    for bad in (dict(P=None), dict(Q=24), dict(ids=None), dict(U=0), dict(I=0), dict(I=2 ** 31), dict(d=33), dict(dt=2), dict(mp=16), dict(scale=0.0),
                dict(scale=float("inf")), dict(scale=float("nan")), dict(T=1), dict(T=-1), dict(K=129, idx=16, val=16), dict(K=301, idx=16, val=16), dict(K=5),
                dict(K=5, idx=16), dict(n=-1)):
        assert call(**bad) == -1, bad
    assert call() == -3 and b"workspace" in L.rsx_last_error() and call(n=0) == 0
    assert rsx.score_logprobs_workspace(4096, 100_000, 128, masked=True, K=10) > rsx.score_logprobs_workspace(4096, 100_000, 128, masked=True)


def test_reference_of_a_row_by_hand():
    P, Q = np.array([[1.0, 0.0]]), np.array([[0.0, 0.0], [math.log(2), 5.0], [0.0, 1.0]])
    logp, lse, ent, top, topv, _ = reference(P, Q, [0, 1], np.array([[1, 2], [0, -1]]), 2, (np.array([0, 1]), np.array([2])), 1.0)
    assert np.allclose(lse[0], math.log(3)) and np.allclose(logp[0, 0], math.log(2 / 3)) and logp[0, 1] == -np.inf
    assert np.allclose(ent[0], math.log(3) - 2 / 3 * math.log(2)) and top[0].tolist() == [1, 0]
    assert lse[1] == -np.inf and logp[1].tolist() == [0, 0] and top[1].tolist() == [-1, -1]


# ---- GPU -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("n,I,K,T,masked,scale", [(1, 1, 1, 1, False, 1.0), (1, 1000, 10, 2, True, 1.0), (3, 33, 33, 1, True, 0.5), (16, 128, 5, 0, False, 2.0),
                                                    (17, 5003, 50, 3, True, 1.0), (33, 129, 0, 4, False, 1.0), (64, 2500, 128, 1, True, 1.0), (65, 31, 7, 1, True, 1.0),
                                                    (130, 127, 10, 2, False, 0.25), (300, 5003, 20, 11, True, 1.0), (257, 1537, 100, 1, True, 3.0)])
def test_hip_logprobs_vs_definition(n, I, K, T, masked, scale, d, bf16):
    rng = np.random.default_rng(n * 7919 + I + d)
    U = n + 5
    P, Q = tables(rng, U, I, d, bf16)
    users = rng.integers(0, U, n)                          # users repeat
    items = rng.integers(0, I, (n, T)) if T else None
    mask = seen_csr(rng, U, I, 40) if masked else None
    got = check(P, Q, users, items, K, mask, scale)
    assert got.top_idx is None or got.top_idx.dtype.is_signed


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [5, 140])
def test_hip_logprobs_empty_rows_padding_and_values_in_masked_places(n, bf16):
    """everything masked; ids that name nothing; NaN and infinities in item rows that every row masks"""
    rng = np.random.default_rng(n)
    U, I, d = 9, 700, 64
    P, Q = tables(rng, U, I, d, bf16)
    Q[100, 3], Q[101, :], Q[699, 0], Q[350, 5] = float("nan"), float("inf"), float("-inf"), float("nan")
    bad = [100, 101, 699, 350, -1, 700, 100]                 # (ids outside the catalog and repeats among a row's seen items)
    rows = [np.array(bad), np.arange(I), np.array(bad + list(range(3, 99)))] * 3
    mask = (np.concatenate([[0], np.cumsum([len(r) for r in rows])]), np.concatenate(rows))
    users = rng.integers(0, U, n)
    users[:5] = [-1, 1, 9, 2 ** 31 - 1, 0]
    items = rng.integers(0, I, (n, 4))
    items[:, 1], items[0], items[1, 0], items[4] = -1, 700, 100, [2 ** 31 - 1, 699, 100, 0]
    check(P, Q, users, items, 12, mask)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 100])
def test_hip_logprobs_ties_go_to_the_lowest_id(n):
    """zero users, equal items, items that are equal in groups: thousands of exact ties, some across the K-th place"""
    import torch
    rng = np.random.default_rng(11)
    d, I = 32, 40_000
    Q = np.repeat(rng.integers(-2, 3, (I // 8, d)), 8, axis=0)[rng.permutation(I)]
    P = rng.integers(-2, 3, (n, d))
    P[0] = 0
    P[1, 1:] = 0
    Q[:, 0] = rng.integers(0, 2, I)                          # user 1: half of the items tie at the top
    P[1, 0] = 1
    f = lambda a: torch.from_numpy(a.astype(np.float32)).cuda()
    for K in (1, 20, 128):
        check(f(P), f(Q), np.arange(n), None, K, None, rows=np.arange(min(n, 12)))
    check(f(P).bfloat16(), f(Q).bfloat16(), np.arange(n), None, 20, None, 0.5, rows=np.arange(min(n, 12)))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [4, 100])
def test_hip_logprobs_scores_with_an_offset_and_items_in_order_of_popularity(n):
    """a common component of +-300 under differences of a few units; ids sorted by score, so that the best are neighbours"""
    rng = np.random.default_rng(5)
    d, I = 64, 30_000
    for offset in (300.0, -300.0):
        P, Q = tables(rng, n, I, d, False)
        P[:, 0], Q[:, 0] = 10.0, offset / 10.0
        order = (P[0] @ Q.T).argsort(descending=True)
        check(P, Q[order].contiguous(), np.arange(n), rng.integers(0, I, (n, 2)), 50, None, rows=np.arange(min(n, 8)))


@pytest.mark.gpu
def test_hip_logprobs_magnitudes():
    """tables scaled by powers of two up and down (the split parts follow them), one row a million times the others"""
    rng = np.random.default_rng(6)
    for n in (3, 90):
        for up in (2.0 ** 30, 2.0 ** -30):
            P, Q = tables(rng, n, 900, 128, False)
            check(P * up, Q / up, np.arange(n), rng.integers(0, 900, (n, 2)), 10, None)
        P, Q = tables(rng, n, 900, 128, False)
        Q[777] *= 1e-6
        P[0] *= 1e-6
        P[1] = 0.0
        check(P, Q, np.arange(n), rng.integers(0, 900, (n, 2)), 10, None)


@pytest.mark.gpu
def test_hip_logprobs_more_rows_than_one_pass_and_tables_beyond_32_bits():
    """2 500 rows of a million items take several passes over bits and maxima; a user table of 4.6 GB"""
    import torch
    rng = np.random.default_rng(8)
    gen = torch.Generator(device="cuda").manual_seed(1)
    I, d = 1_000_000, 32
    Q = (torch.randn(I, d, generator=gen, device="cuda") * 0.6).bfloat16()
    U = 72_000_000
    P = torch.zeros(U, d, dtype=torch.bfloat16, device="cuda")
    users = np.concatenate([rng.integers(0, U, 2499), [U - 1]])
    P[torch.from_numpy(users).cuda()] = (torch.randn(2500, d, generator=gen, device="cuda") * 0.6).bfloat16()
    from recsys_pytorch_amd import rsx
    u = torch.from_numpy(users.astype(np.int32)).cuda()
    items = torch.from_numpy(rng.integers(0, I, (2500, 1)).astype(np.int32)).cuda()
    deg = torch.zeros(U + 1, dtype=torch.int64)
    deg[1 + torch.from_numpy(users)] = 3
    indptr = deg.cumsum(0).cuda()
    indices = torch.from_numpy(rng.integers(0, I, int(indptr[-1]))).to(torch.int32).cuda()
    got = rsx.score_logprobs(P, Q, u, items, K=10, mask=(indptr, indices))
    for r in (0, 1023, 1024, 1700, 2498, 2499):
        z = Q.double() @ P[u[r].long()].double()
        lo, hi = int(indptr[u[r].long()]), int(indptr[u[r].long() + 1])
        z[indices[lo:hi].long()] = -math.inf
        lse = torch.logsumexp(z, 0)
        tol = (3 * d + 3) * 2.0 ** -24 * float((Q.abs().float() @ P[u[r].long()].abs().float()).max()) + (64 * 30 + 100) * 2.0 ** -24 + 1.5e-5
        assert abs(float(got.lse[r] - lse)) <= tol and abs(float(got.logp[r, 0] - (z[items[r, 0].long()] - lse))) <= tol
        v, at = z.sort(descending=True, stable=True)
        assert torch.equal(got.top_idx[r].long(), at[:10])


@pytest.mark.gpu
def test_hip_logprobs_captured_on_another_stream_and_reproducible():
    import torch
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(9)
    for n, I, d in ((1, 3000, 128), (200, 3000, 128)):
        P, Q = tables(rng, n, I, d, False)
        u = torch.arange(n, dtype=torch.int32, device="cuda")
        t = torch.from_numpy(rng.integers(0, I, (n, 2)).astype(np.int32)).cuda()
        mask = tuple(torch.from_numpy(a).cuda() for a in seen_csr(rng, n, I, 30))
        want = rsx.score_logprobs(P, Q, u, t, K=10, mask=mask)
        again = rsx.score_logprobs(P, Q, u, t, K=10, mask=mask)
        assert all(torch.equal(a, b) for a, b in zip(want, again))
        ws = torch.empty(rsx.score_logprobs_workspace(n, I, d, masked=True, K=10) // 8 + 1, dtype=torch.int64, device="cuda")
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = rsx.score_logprobs(P, Q, u, t, K=10, mask=mask, ws=ws)
            side.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(want, other))
            with torch.cuda.graph(graph, stream=side):
                held = rsx.score_logprobs(P, Q, u, t, K=10, mask=mask, ws=ws)
        for k in range(4):
            P.copy_(P.flip(0) if k else P)
            ws.random_()
            graph.replay()
            eager = rsx.score_logprobs(P, Q, u, t, K=10, mask=mask)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(eager, held)), k


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("n,tied", [(513, False), (300, True), (513, True)])
def test_hip_logprobs_of_more_rows_than_the_chip_has_room_for_at_once(n, tied, d, bf16):
    """the last kernel's forms for up to two rows a CU and for more; tied: every item four times, so that whole chunks tie at the border"""
    rng = np.random.default_rng(n + d)
    P, Q = tables(rng, 97, 640, d, bf16)
    if tied:
        Q = Q[:160].repeat(4, 1).reshape(640, d).contiguous()
    users = rng.integers(-1, 98, n)
    check(P, Q, users, rng.integers(-1, 641, (n, 2)), 30, seen_csr(rng, 97, 640, 60), 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [7, 300, 600])
@pytest.mark.parametrize("d", [32, 128])
def test_hip_logprobs_of_zero_elements_beside_infinities_in_masked_places(d, n):
    """infinities and NaN in items that everybody has seen, zeros in the users' rows: 0 * inf of a masked item is no neighbour's business"""
    rng = np.random.default_rng(n + d)
    P, Q = tables(rng, n, 1000, d, False)
    P[:, : d // 2] = 0.0
    P[::3] = 0.0
    bad = rng.permutation(1000)[:120]
    Q[bad[:60], : d // 4] = float("inf")
    Q[bad[60:], 1] = float("nan")
    indptr, indices = seen_csr(rng, n, 1000, 20)
    rows = [np.union1d(indices[indptr[u]:indptr[u + 1]], bad) for u in range(n)]
    mask = np.concatenate([[0], np.cumsum([len(r) for r in rows])]).astype(np.int64), np.concatenate(rows).astype(np.int32)
    check(P, Q, np.arange(n), rng.integers(0, 1000, (n, 3)), 40, mask, 1.0)


@pytest.mark.gpu
def test_hip_logprobs_of_more_rows_than_a_grids_second_dimension_takes():
    """nine million positions of a catalog of three"""
    import torch
    from recsys_pytorch_amd import rsx
    P, Q = tables(np.random.default_rng(4), 50, 3, 32, False)
    n = 9_000_000
    users = torch.arange(n, dtype=torch.int32, device="cuda") % 50
    got = rsx.score_logprobs(P, Q, users, (users % 3).view(-1, 1).contiguous(), K=2)
    u = np.arange(150) % 50
    logp, lse, ent, top, topv, ez = reference(P.double().cpu().numpy(), Q.double().cpu().numpy(), u, (u % 3)[:, None], 2, None, 1.0)
    el = ez + 5e-5
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda().view(1, 150, -1)
    whole = lambda t: t.view(n // 150, 150, -1)
    assert (whole(got.top_idx) == dev(top)).all()
    for a, b, tol in ((got.lse, lse, el + 2.0 ** -24 * np.abs(lse)), (got.entropy, ent, el * (2 + ent) + ez), (got.logp, logp, el[:, None] + 2.0 ** -24 * np.abs(logp)),
                      (got.top_logp, topv, el[:, None] + 2.0 ** -24 * np.abs(topv))):
        assert ((whole(a).double() - dev(b)).abs() <= dev(tol)).all()
