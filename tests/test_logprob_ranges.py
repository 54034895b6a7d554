"""rsx.score_logprobs where values lie far apart: scores thousands of units below a row's best, item rows of very unequal length, masked
rows of large finite values, long sums of equal terms.

Tolerances: test_logprob.py's (its `check`), whose score error counts the unmasked items only; what a test allows instead is derived at it."""
import numpy as np
import pytest

from test_logprob import check, reference, seen_csr, tables


def _mask_all(users, ids):
    return np.arange(users + 1, dtype=np.int64) * len(ids), np.tile(np.asarray(ids, np.int32), users)


# ---- the K best ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [4, 140, 300, 600])
def test_hip_top_items_of_scores_far_apart(n, bf16):
    """scores over hundreds of thousands of units: far below a row's reference is not the same as masked"""
    import torch
    rng = np.random.default_rng(n)
    for I, K, near in ((100, 100, 1), (3000, 128, 30)):
        P, Q = (rng.standard_normal((r, 32)).astype(np.float32) for r in (n, I))
        P[:, 0] = rng.choice([1.0, 2.0, -1.0], n)
        P[:2, 0] = 1.0, -1.0
        Q[:, 0] = 0.0
        far = rng.permutation(I)[near:]
        Q[far, 0] = -np.linspace(1e5, 3e5, I - near)
        P, Q = torch.from_numpy(P).cuda(), torch.from_numpy(Q).cuda()
        P, Q = (P.bfloat16(), Q.bfloat16()) if bf16 else (P, Q)
        mask = _mask_all(n, far[:40]) if I == 3000 else None
        check(P, Q, np.arange(n), rng.integers(0, I, (n, 2)), K, mask, rows=np.r_[0:4, n - 4:n])


@pytest.mark.gpu
@pytest.mark.parametrize("n,bf16", [(4, False), (4, True), (140, True), (600, True)])
def test_hip_top_items_beside_masked_rows_of_large_values(n, bf16):
    """finite products of 10^20 in masked places, where a row's reference may look too"""
    rng = np.random.default_rng(n)
    for I, bad in ((2, [1]), (33, [0, 16]), (900, [0, 450, 899]), (900, [450, 899])):
        P, Q = tables(rng, n, I, 64, bf16)
        P[:, 5] = P[:, 5].abs() + 1.0
        Q[bad, 5] = 1e20 if I != 33 else -1e20
        check(P, Q, np.arange(n), rng.integers(0, I, (n, 2)), min(I, 20), _mask_all(n, bad), rows=np.r_[0:4, n - 4:n])


# ---- item rows of unequal length (fp32 rows share scales) ------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("size", [1e5, 1e6, 1e9, 1e12, 1e30])
def test_hip_logprobs_beside_masked_rows_of_large_values(size, d):
    """what a masked cell's product would have been does not matter: finite values too, however large"""
    rng = np.random.default_rng(d)
    n, I = 140, 500
    P, Q = tables(rng, n, I, d, False)
    bad = [0, 37, 250, 251, 499]
    Q[bad] *= size
    check(P, Q, np.arange(n), rng.integers(0, I, (n, 3)), 30, _mask_all(n, bad))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 140])
def test_hip_logprobs_beside_an_item_of_probability_zero(n):
    """an unmasked row a million times the others whose score is -3 10^6 for everybody: the others' log-probabilities are those without it"""
    import torch
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(n)
    I, out = 400, 70
    P, Q = tables(rng, n, I, 64, False)
    P[:, 0] = 3.0
    Q[out] = 0.0
    Q[out, 0] = -1e6
    items = rng.integers(0, I, (n, 3))
    items[items == out] = 0
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    got = rsx.score_logprobs(P, Q, dev(np.arange(n)), dev(items), K=20)
    logp, lse, ent, top, topv, ez = reference(P.double().cpu().numpy(), Q.double().cpu().numpy(), np.arange(n), items, 20, _mask_all(n, [out]), 1.0)
    el = ez + 5e-5
    err = lambda a, b: np.abs(a.double().cpu().numpy() - b)
    assert (err(got.lse, lse) <= el + 2.0 ** -24 * np.abs(lse)).all()
    assert (err(got.entropy, ent) <= el * (2 + ent) + ez).all()
    assert (err(got.logp, logp) <= el[:, None] + 2.0 ** -24 * np.abs(logp)).all()
    assert np.array_equal(got.top_idx.cpu().numpy(), top) and (err(got.top_logp, topv) <= el[:, None] + 2.0 ** -24 * np.abs(topv)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 90])
@pytest.mark.parametrize("power", [60, 80, 100])
def test_hip_logprobs_of_tables_of_opposite_size(n, power):
    rng = np.random.default_rng(power)
    for up in (2.0 ** power, 2.0 ** -power):
        P, Q = tables(rng, n, 300, 64, False)
        check(P * up, Q / up, np.arange(n), rng.integers(0, 300, (n, 2)), 10, None)


# ---- the normaliser's last bits --------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", [2, 200])
def test_hip_normaliser_of_one_item_is_its_score(n, bf16):
    """one item: lse = z, exact products.  2^(t - m) is 2^r with r what the reference's rounding left (the fused multiply-add is exact to 2^-24 of
    it): 2^-22 for exponential and logarithm, half a step of the result below 16 (2^-24 16): together 7.2e-7 on scores up to 16.  Many fp32 rows: the operand is x scale log2 e as two halves (2^-24 of it), two products are
    added up in fp32 (2^-24 of the score each): 3 2^-24 16 = 2.9e-6 more"""
    import torch
    from recsys_pytorch_amd import rsx
    two = np.log2(np.e)
    scales = np.arange(1, 4000, dtype=np.float32) / np.float32(2500)
    scale = float(scales[np.argmax(np.abs((scales * np.float32(two)).astype(np.float64) / (scales.astype(np.float64) * two) - 1))])       # rounds worst
    x = np.arange(1, 1 + n) % 128 + 128.0                          # eight bits
    y = np.float32(15.9 / 255 / scale)
    y = float(torch.tensor(y).bfloat16())
    P, Q = torch.zeros(n, 32), torch.zeros(1, 32)
    P[:, 3], Q[:, 3] = torch.from_numpy(x.astype(np.float32)), y
    P, Q = (P.bfloat16().cuda(), Q.bfloat16().cuda()) if bf16 else (P.cuda(), Q.cuda())
    got = rsx.score_logprobs(P, Q, torch.arange(n, dtype=torch.int32, device="cuda"), scale=scale)
    want = x * y * float(np.float32(scale))
    assert want.max() < 16.0
    assert np.abs(got.lse.double().cpu().numpy() - want).max() <= 7.2e-7 + (2.9e-6 if n > 64 and not bf16 else 0.0)


def _sum_in_fp32(e, groups):
    """a lane's sum of 64 equal terms a group, groups added one to the next, all in fp32; relative to the exact one"""
    e = np.float32(e)
    tile = np.float32(0)
    for _ in range(16):
        tile = np.float32(tile + e)
    group = np.float32(0)
    for _ in range(4):
        group = np.float32(group + tile)
    total = np.float32(0)
    for _ in range(groups):
        total = np.float32(total + group)
    return float(total) / (64.0 * groups * float(e)) - 1


@pytest.mark.gpu
@pytest.mark.parametrize("bf16", [False, True])
def test_hip_normaliser_of_a_long_sum_of_equal_terms(bf16):
    """30 000 equal scores under one that is larger, in one piece of the catalog: the groups' sums must not pile up fp32 roundings (equal terms round
    the same way).  Exponential 2^-22, 20 additions of a group 20 2^-24, half a step of a result below 16: 1.9e-6"""
    import torch
    from recsys_pytorch_amd import rsx
    n, I = 70_000, 30_000
    steps = np.arange(1, 128) / 128.0
    off = [abs(_sum_in_fp32(np.exp2(np.float32(np.log2(np.e)) * -s), I // 128)) for s in steps]
    gap = float(steps[int(np.argmax(off))])
    assert max(off) > 3e-6
    P, Q = torch.zeros(n, 32), torch.zeros(I, 32)
    P[:, 0], Q[:, 0], Q[7, 0] = 1.0, -gap, 0.0
    P, Q = (P.bfloat16().cuda(), Q.bfloat16().cuda()) if bf16 else (P.cuda(), Q.cuda())
    got = rsx.score_logprobs(P, Q, torch.arange(n, dtype=torch.int32, device="cuda"))
    p = (I - 1) * np.exp(-gap)
    want = np.log1p(p)
    assert np.abs(got.lse.double().cpu().numpy() - want).max() <= 1.9e-6
    # H = lse - E z, E z = -gap p / (1 + p): twice the terms' roundings, and half a step of the result
    assert np.abs(got.entropy.double().cpu().numpy() - (want + gap * p / (1 + p))).max() <= 4e-6


# ---- a mask of nothing -----------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 140])
def test_hip_a_mask_without_entries_masks_nothing(n):
    import scipy.sparse as sp
    import torch
    import recsys_pytorch_amd as pkg
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(n)
    P, Q = tables(rng, n, 300, 64, False)
    dev = lambda a, t=np.int32: torch.from_numpy(np.ascontiguousarray(a, t)).cuda()
    u, it = dev(np.arange(n)), dev(rng.integers(0, 300, (n, 2)))
    empty = torch.zeros(n + 1, dtype=torch.int64, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")
    want, got = rsx.score_logprobs(P, Q, u, it, K=7), rsx.score_logprobs(P, Q, u, it, K=7, mask=empty)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    g = dev(rng.standard_normal((n, 2)), np.float32)
    for a, b in zip(rsx.score_logprobs_grad(P, Q, u, it, want.lse, g), rsx.score_logprobs_grad(P, Q, u, it, want.lse, g, mask=empty)):
        assert torch.equal(a, b)
    assert torch.equal(rsx.score(P, Q, u), rsx.score(P, Q, u, mask=empty)) and torch.equal(rsx.score_topk(P, Q, u, 7), rsx.score_topk(P, Q, u, 7, mask=empty))
    with pytest.raises(rsx.RsxError, match="indptr"):                # (its shape is still looked at)
        rsx.score_logprobs(P, Q, u, it, mask=(empty[0][:-1], empty[1]))
    ds = pkg.InteractionData(sp.random(n, 300, 0.1, random_state=1, data_rvs=np.ones).tocsr())
    m = pkg.MF(ds, {"hidden_dim": 64, "pointwise": False, "loss_func": "ce", "optimizer": "sgd"}, "cuda")
    nothing = sp.csr_matrix((n, 300))
    for a, b in zip(m.predict_logprobs(np.arange(n), np.arange(n), K=5), m.predict_logprobs(np.arange(n), np.arange(n), eval_pos=nothing, K=5)):
        assert np.array_equal(a, b)


# ---- scores closer than the fast products' rounding ---------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 140, 600])
@pytest.mark.parametrize("I", [700, 1900, 9000])
def test_hip_top_items_among_items_that_are_nearly_equal(I, n):
    """item rows that differ in their last bits: the order of the scores is that of their products in 64 bits all the same"""
    import torch
    rng = np.random.default_rng(I + n)
    P = torch.from_numpy(rng.standard_normal((n, 64)).astype(np.float32)).cuda()
    base = rng.standard_normal(64)
    Q = torch.from_numpy((base + 3e-7 * rng.standard_normal((I, 64))).astype(np.float32)).cuda()
    check(P, Q, np.arange(n), rng.integers(0, I, (n, 2)), 20, None, rows=np.r_[0:3, n - 3:n])
    Q[::5] += 0.5                                             # ... and half a unit above the others a fifth of them
    check(P, Q, np.arange(n), rng.integers(0, I, (n, 2)), 20, _mask_all(n, [5, 10, 200]), rows=np.r_[0:3, n - 3:n])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 140])
@pytest.mark.parametrize("size", [1e-4, 1.0, 100.0])
def test_hip_top_items_of_scores_whose_terms_cancel(size, n):
    """products of size^2 whose sums are thousands of times smaller, and tables whose scores differ by 10^-8 of one"""
    import torch
    rng = np.random.default_rng(n)
    half = rng.standard_normal((n, 32))
    P = torch.from_numpy((np.concatenate([half, -half], 1) * size).astype(np.float32)).cuda()
    twin = rng.standard_normal((3000, 32))
    Q = torch.from_numpy((np.concatenate([twin, twin + 1e-4 * rng.standard_normal(twin.shape)], 1) * size).astype(np.float32)).cuda()
    check(P, Q, np.arange(n), rng.integers(0, 3000, (n, 2)), 20, None, rows=np.r_[0:3, n - 3:n])
