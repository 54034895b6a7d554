"""Measured cases of the full-catalog log-probability, its gradient, and the orthogonalised update.

    logprobs   rsx.score_logprobs       log-softmax of a user's scores over the whole catalog at given items, its normaliser and entropy,
                                        and the K most probable items with their log-probabilities
    grad       rsx.score_logprobs_grad  gradient of a weighted sum of those log-probabilities and entropies, by user row and by item row
    orth       rsx.orthogonalize        Newton-Schulz iteration of a [rows x d] matrix towards its nearest orthonormal columns
    muon       rsx.muon_apply           one optimizer step: momentum, orthogonalised update, decoupled weight decay

Where `own` is false, `run` is the same arithmetic in elementary torch operations; where it is true, the calls of a user's program.
"""
import math

import numpy as np
import torch

own = False

COEFFS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one user's request against a 100 000-item catalog: latency of a serving call
        {"name": "serve one user", "op": "logprobs", "n": 1, "items": 100_000, "d": 128, "dtype": "fp32", "T": 1, "K": 10, "mask": True, "scale": 1.0},
        # a handful of concurrent requests against a catalog of a million in bf16
        {"name": "serve 16, 1M items, bf16", "op": "logprobs", "n": 16, "items": 1_000_000, "d": 128, "dtype": "bf16", "T": 1, "K": 20, "mask": True, "scale": 1.0},
        # the evaluation of a small catalog (ml-100k: 943 users, 1 682 items; hidden_dim 50 is stored as 64 columns)
        {"name": "evaluate ml-100k", "op": "logprobs", "n": 943, "items": 1682, "d": 64, "dtype": "fp32", "T": 5, "K": 50, "mask": True, "scale": 1.0},
        # one evaluation batch against 100 000 items with ten held-out items per user
        {"name": "evaluate 1024 of 100K", "op": "logprobs", "n": 1024, "items": 100_000, "d": 128, "dtype": "fp32", "T": 10, "K": 50, "mask": True, "scale": 1.0},
        # a whole pass of a large evaluation in bf16
        {"name": "evaluate 8192 of 100K bf16", "op": "logprobs", "n": 8192, "items": 100_000, "d": 128, "dtype": "bf16", "T": 1, "K": 10, "mask": True, "scale": 1.0},
        # training with the softmax loss at the reference's batch of 256 on ml-100k
        {"name": "train ml-100k, 256", "op": "grad", "n": 256, "items": 1682, "d": 64, "dtype": "fp32", "T": 1, "mask": False, "entropy": False, "scale": 1.0},
        # a large training batch over 100 000 items
        {"name": "train 4096 of 100K", "op": "grad", "n": 4096, "items": 100_000, "d": 128, "dtype": "fp32", "T": 1, "mask": False, "entropy": False, "scale": 1.0},
        # several positives per user, an entropy bonus, a temperature, seen items left out, wide rows in bf16
        {"name": "train 1000 of 50021 bf16", "op": "grad", "n": 1000, "items": 50_021, "d": 256, "dtype": "bf16", "T": 4, "mask": True, "entropy": True, "scale": 2.0},
        # the optimizer step of a small item table
        {"name": "muon 1682 x 64", "op": "muon", "rows": 1682, "d": 64, "dtype": "fp32", "steps": 5},
        # ... of the 100 000-item table, and of a million user rows
        {"name": "muon 100K x 128", "op": "muon", "rows": 100_000, "d": 128, "dtype": "fp32", "steps": 5},
        {"name": "muon 1M x 128", "op": "muon", "rows": 1_000_000, "d": 128, "dtype": "fp32", "steps": 5},
        # the bare iteration on a wide bf16 gradient with an odd number of rows
        {"name": "orthogonalize 20011 x 256 bf16", "op": "orth", "rows": 20_011, "d": 256, "dtype": "bf16", "steps": 5},
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "grad", "grad", "orth", "muon"])
    d = rng.choice([32, 64, 128, 256])
    dtype = rng.choice(["fp32", "bf16"])
    if op in ("orth", "muon"):
        return {"op": op, "rows": _spread(rng, 33, 128_000_000 // d), "d": d, "dtype": dtype, "steps": rng.choice([4, 5, 5, 6])}
    items = _spread(rng, 600, 1_000_000)
    room = (8192 if op == "logprobs" else 4096) * 100_000 * min(1.0, 128 / d)
    n = _spread(rng, 1 if op == "logprobs" else 8, max(16, min(8192, int(room / items))))
    c = {"op": op, "n": n, "items": items, "d": d, "dtype": dtype, "T": rng.choice([1, 1, 2, 5, 10]), "mask": rng.random() < 0.6,
         "scale": rng.choice([1.0, 0.5, 2.0])}
    if op == "logprobs":
        return {**c, "K": rng.choice([0, 1, 5, 10, 20, 50, 100])}
    return {**c, "entropy": rng.random() < 0.3}


def _seen(gen, users, items, dev):
    """CSR of seen items, up to 40 a user, popular ones more often"""
    deg = torch.randint(0, min(41, items // 8), (users,), generator=gen, device=dev)
    who = torch.repeat_interleave(torch.arange(users, device=dev), deg)
    what = (torch.rand(who.numel(), generator=gen, device=dev).square() * items).long().clamp_(max=items - 1)
    key = torch.unique(who * items + what)
    indptr = torch.zeros(users + 1, dtype=torch.int64, device=dev)
    indptr[1:] = torch.bincount(key // items, minlength=users).cumsum(0)
    return indptr, (key % items).to(torch.int32)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed))
    normal = lambda *s: torch.randn(*s, generator=gen, device=dev)
    dt, d = DTYPES[case["dtype"]], case["d"]
    s = dict(case)
    if case["op"] in ("orth", "muon"):
        # a gradient whose columns are correlated and of unequal size, as a trained table's are
        mix = normal(d, d) / math.sqrt(d) * torch.logspace(0, -2, d, device=dev)
        g = (normal(case["rows"], d) @ mix * 1e-3).to(dt)
        if case["op"] == "orth":
            s["X"] = g
        else:
            s["grad"], s["G"] = g, torch.zeros_like(g)
            s["W"], s["M"] = normal(case["rows"], d) * 0.1, normal(case["rows"], d) * 1e-3
        return s
    n, items = case["n"], case["items"]
    users = n + n // 3 + 7
    sd = (4.0 / d) ** 0.25                                   # scores of standard deviation about 2
    popular = torch.exp(0.3 * normal(items, 1))              # item rows of unequal length
    s["P"], s["Q"] = (normal(users, d) * sd).to(dt), (normal(items, d) * sd * popular).to(dt)
    s["users"] = torch.randperm(users, generator=gen, device=dev)[:n].to(torch.int32)
    s["targets"] = torch.randint(0, items, (n, case["T"]), generator=gen, device=dev, dtype=torch.int32)
    s["mask_csr"] = _seen(gen, users, items, dev) if case["mask"] else None
    if case["op"] == "grad":
        s["g_logp"] = -(0.5 + torch.rand(n, case["T"], generator=gen, device=dev)) / (n * case["T"])
        s["g_entropy"] = -0.1 * torch.rand(n, generator=gen, device=dev) / n if case["entropy"] else None
        S = _scores(s)
        s["lse"] = torch.logsumexp(S, 1)
        s["entropy"] = _entropy(S, s["lse"]) if case["entropy"] else None
    return s


def _masked_cells(s):
    """(row of the call, item) of every seen item of the call's users"""
    indptr, indices = s["mask_csr"]
    u = s["users"].long()
    deg = indptr[u + 1] - indptr[u]
    row = torch.repeat_interleave(torch.arange(u.numel(), device=u.device), deg)
    start = torch.repeat_interleave(indptr[u] - (deg.cumsum(0) - deg), deg)
    return row, indices[start + torch.arange(row.numel(), device=u.device)].long()


def _scores(s, dt=torch.float32):
    S = s["P"][s["users"].long()].to(dt) @ s["Q"].to(dt).T
    if s["scale"] != 1.0:
        S = S * s["scale"]
    if s["mask_csr"] is not None:
        S[_masked_cells(s)] = -math.inf
    return S


def _entropy(S, lse):
    L = S - lse[:, None]
    return -(torch.exp(L) * L.masked_fill(L == -math.inf, 0.0)).sum(1)


def _top(s, S, lse, K):
    """the K best by (score in 64 bits, lowest id): candidates by the 32-bit scores, ordered by their 64-bit products"""
    value, at = torch.topk(S, min(K + 16, S.shape[1]), dim=1)
    at, order = at.sort(1)
    value = value.gather(1, order)
    p = s["P"][s["users"].long()].double()
    exact = (s["Q"][at].double() * p[:, None, :]).sum(2) * s["scale"]
    exact = torch.where(value == -math.inf, -math.inf, exact)
    exact, order = exact.sort(dim=1, descending=True, stable=True)
    exact, at = exact[:, :K], at.gather(1, order)[:, :K]
    return torch.where(exact == -math.inf, -1, at).to(torch.int32), (exact - lse[:, None].double()).float()


def _polynomial(X, a, b, c):
    A = X.T @ X
    return a * X + X @ (b * A + c * (A @ A))


def _newton_schulz(X, steps):
    X = X.float()
    X = X / (X.square().sum().sqrt() + EPS)
    X = _polynomial(_polynomial(_polynomial(_polynomial(X, *COEFFS), *COEFFS), *COEFFS), *COEFFS)
    X = _polynomial(X, *COEFFS) if steps >= 5 else X
    return _polynomial(X, *COEFFS) if steps >= 6 else X


LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def _run_logprobs(s):
    if own:
        from recsys_pytorch_amd import rsx
        r = rsx.score_logprobs(s["P"], s["Q"], s["users"], s["targets"], K=s["K"], mask=s["mask_csr"], scale=s["scale"])
        out = {"logp": r.logp, "lse": r.lse, "entropy": r.entropy}
        return {**out, "top_idx": r.top_idx, "top_logp": r.top_logp} if s["K"] else out
    S = _scores(s)
    lse = torch.logsumexp(S, 1)
    out = {"logp": S.gather(1, s["targets"].long()) - lse[:, None], "lse": lse, "entropy": _entropy(S, lse)}
    if s["K"]:
        out["top_idx"], out["top_logp"] = _top(s, S, lse, s["K"])
    return out


def _run_grad(s):
    if own:
        from recsys_pytorch_amd import rsx
        GP, GQ = rsx.score_logprobs_grad(s["P"], s["Q"], s["users"], s["targets"], s["lse"], s["g_logp"], entropy=s["entropy"],
                                         g_entropy=s["g_entropy"], mask=s["mask_csr"], scale=s["scale"])
        return {"GP": GP, "GQ": GQ}
    L = _scores(s) - s["lse"][:, None]
    p = torch.exp(L)
    t = s["targets"].long()
    g = torch.where(L.gather(1, t) == -math.inf, 0.0, s["g_logp"])           # a masked item's log-probability is a constant
    D = p * -g.sum(1, keepdim=True)
    if s["g_entropy"] is not None:
        D = D - s["g_entropy"][:, None] * p * (L.masked_fill(L == -math.inf, 0.0) + s["entropy"][:, None])
    D.scatter_add_(1, t, g)
    D = D * s["scale"]
    dt = s["P"].dtype
    return {"GP": (D @ s["Q"].float()).to(dt), "GQ": (D.T @ s["P"][s["users"].long()].float()).to(dt)}


def _run_orth(s):
    if own:
        from recsys_pytorch_amd import rsx
        return rsx.orthogonalize(s["X"], steps=s["steps"], coeffs=COEFFS, eps=EPS)
    return _newton_schulz(s["X"], s["steps"]).to(s["X"].dtype)


def _run_muon(s):
    s["G"].copy_(s["grad"])                                  # the backward pass of a training step fills it anew
    W, M, G = s["W"], s["M"], s["G"]
    if own:
        from recsys_pytorch_amd import rsx
        rsx.muon_apply(W, M, G, LR, momentum=MOMENTUM, nesterov=True, steps=s["steps"], coeffs=COEFFS, eps=EPS, weight_decay=DECAY)
    else:
        M.mul_(MOMENTUM).add_(G.float())
        O = _newton_schulz(G.float() + MOMENTUM * M, s["steps"])
        W.mul_(1.0 - LR * DECAY).sub_(O * (LR * math.sqrt(max(1.0, W.shape[0] / W.shape[1]))))
        G.zero_()
    return {"W": W, "M": M}


def run(state):
    return {"logprobs": _run_logprobs, "grad": _run_grad, "orth": _run_orth, "muon": _run_muon}[state["op"]](state)


def work(case):
    d, es = case["d"], 2 if case["dtype"] == "bf16" else 4
    if case["op"] in ("orth", "muon"):
        N = case["rows"]
        flops = 3.0 * N * d * d                              # the symmetric Gram matrix and one product with a [d x d] matrix
        return {"bytes": 2.0 * N * d * es if case["op"] == "orth" else N * d * (2.0 * es + 16.0), "flops": flops}
    n, items, T = case["n"], case["items"], case["T"]
    tables = (n + items) * d * es
    if case["op"] == "logprobs":
        return {"bytes": tables + n * (8.0 * T + 8 + 8.0 * case["K"]), "flops": 2.0 * n * items * d}
    return {"bytes": 2.0 * tables + n * (8.0 * T + 4), "flops": 6.0 * n * items * d}


def _exact_logprobs(s):
    """row by block, in 64 bits; the K best by a full stable sort where it is small, else among a wider choice"""
    K, outs = s["K"], []
    Q, P, ids = s["Q"].double(), s["P"].double(), s["users"].long()
    step = max(1, int(2e8 / Q.shape[0]))
    for lo in range(0, ids.numel(), step):
        u, t = ids[lo:lo + step], s["targets"][lo:lo + step].long()
        z = torch.mm(P[u], Q.t()).mul_(s["scale"])
        if s["mask_csr"] is not None:
            ptr, idx = s["mask_csr"]
            for r, who in enumerate(u.tolist()) if u.numel() <= 64 else ():
                z[r, idx[ptr[who]:ptr[who + 1]].long()] = -math.inf
            if u.numel() > 64:
                hit = torch.zeros_like(z, dtype=torch.bool)
                owner = torch.searchsorted(ptr, torch.arange(idx.numel(), device=ptr.device), right=True) - 1
                place = torch.full((P.shape[0],), -1, dtype=torch.int64, device=ptr.device)
                place[u] = torch.arange(u.numel(), device=ptr.device)
                keep = place[owner] >= 0
                hit[place[owner][keep], idx[keep].long()] = True
                z.masked_fill_(hit, -math.inf)
                del hit
        top = z.max(1).values
        e = torch.exp(z - top[:, None])
        total = e.sum(1)
        lse = top + total.log()
        entropy = lse - (e * z.masked_fill(z == -math.inf, 0.0)).sum(1) / total
        o = {"logp": z.gather(1, t) - lse[:, None], "lse": lse, "entropy": entropy}
        del e
        if K:
            v, at = z.topk(min(K + 4, z.shape[1]), dim=1)
            at, o1 = at.sort(1)
            v, o2 = v.gather(1, o1).sort(dim=1, descending=True, stable=True)
            at = at.gather(1, o2)[:, :K]
            o["top_idx"] = torch.where(v[:, :K] == -math.inf, -1, at).to(torch.int32)
            o["top_logp"] = v[:, :K] - lse[:, None]
        outs.append(o)
    return {k: torch.cat([o[k] for o in outs]) for k in outs[0]}


def _exact_grad(s):
    """the chain rule through the scores, a block of rows at a time, in 64 bits (lse and entropy are inputs of the operator)"""
    Q, P, ids = s["Q"].double(), s["P"].double(), s["users"].long()
    GP, GQ = torch.zeros(ids.numel(), Q.shape[1], dtype=torch.float64, device=Q.device), torch.zeros_like(Q)
    step = max(1, int(2e8 / Q.shape[0]))
    for lo in range(0, ids.numel(), step):
        b = slice(lo, lo + step)
        x = P[ids[b]]
        logp = torch.mm(x, Q.t()).mul_(s["scale"]).sub_(s["lse"][b, None].double())
        allowed = torch.ones_like(logp, dtype=torch.bool)
        if s["mask_csr"] is not None:
            r, i = _masked_cells({**s, "users": s["users"][b]})
            allowed[r, i] = False
        prob = logp.exp() * allowed
        weight = torch.zeros_like(prob)
        t = s["targets"][b].long()
        weight.scatter_add_(1, t, s["g_logp"][b].double())
        weight *= allowed
        dz = weight - prob * weight.sum(1, keepdim=True)
        if s["g_entropy"] is not None:
            dz -= prob * s["g_entropy"][b, None].double() * (torch.where(allowed, logp, 0.0) + s["entropy"][b, None].double())
        dz *= s["scale"]
        GP[b] = torch.mm(dz, Q)
        GQ += torch.mm(dz.t().contiguous(), x)
        del logp, allowed, prob, weight, dz
    return {"GP": GP, "GQ": GQ}


def _exact_orth(X, steps):
    X = X.double()
    X = X / (torch.linalg.vector_norm(X) + EPS)
    a, b, c = COEFFS
    for _ in range(steps):
        gram = torch.mm(X.t().contiguous(), X)
        X = a * X + b * torch.mm(X, gram) + c * torch.mm(X, torch.mm(gram, gram))
    return X


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        return _exact_logprobs(s)
    if case["op"] == "grad":
        return _exact_grad(s)
    if case["op"] == "orth":
        return _exact_orth(s["X"], case["steps"])
    g = s["grad"].double()
    M = MOMENTUM * s["M"].double() + g
    O = _exact_orth(g + MOMENTUM * M, case["steps"])
    return {"W": (1.0 - LR * DECAY) * s["W"].double() - LR * math.sqrt(max(1.0, case["rows"] / case["d"])) * O, "M": M}
