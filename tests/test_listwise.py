"""The softmax over the catalog and the orthogonalised step as the models use them: BPREngine.listwise_step, optimizer 'muon',
MF / LightGCN.predict_logprobs, the fit loops.

Tolerance of a listwise SGD step: the gradients' of test_logprob_grad.py, with lse now the forward call's (off by el = ez + 5e-5,
test_logprob.py, which is that much of every p on top), the k rows of a user summed in fp32 (k half steps of their absolute sum), the
sweep's product and sum (one half step of lr |g|, one of the result)."""
import types

import numpy as np
import pytest
import scipy.sparse as sp
import torch

import cpu_kernels
from test_logprob import reference
from test_logprob_grad import gradient
from test_ortho import newton_schulz

HP = {"hidden_dim": 32, "pointwise": False, "loss_func": "ce"}


# ---- plain kernels on the CPU: the engine's and the models' logic without a GPU ------------------------------------------------------
def _plain_kernels():
    from recsys_pytorch_amd import rsx
    k = types.SimpleNamespace(**{n: getattr(cpu_kernels, n) for n in dir(cpu_kernels) if not n.startswith("_")})
    k.calls = []

    def score_logprobs(P, Q, u, items=None, K=0, mask=None, scale=1.0, ws=None):
        m = None if mask is None else tuple(t.numpy() for t in mask)
        r = reference(P.double().numpy(), Q.double().numpy(), u.numpy(), None if items is None else items.numpy(), K, m, scale)
        f = lambda a: torch.from_numpy(np.asarray(a, np.float32))
        return rsx.LogProbs(None if items is None else f(r[0]), f(r[1]), f(r[2]), torch.from_numpy(r[3].astype(np.int32)) if K else None, f(r[4]) if K else None)

    def score_logprobs_grad(P, Q, u, items, lse, g, out=None, ws=None):
        k.calls.append((u.clone(), items.clone(), g.clone()))
        GP, GQ = gradient(P.double().numpy(), Q.double().numpy(), u.numpy(), items.numpy(), g.double().numpy(), None, lse.double().numpy(), None, None, 1.0)[:2]
        out[0].copy_(torch.from_numpy(GP))
        out[1].copy_(torch.from_numpy(GQ))
        return out

    def muon_apply(W, M, G, lr, momentum=0.95, nesterov=True, steps=5, weight_decay=0.0, update_scale=None, ws=None):
        M.mul_(momentum).add_(G)
        U = G + momentum * M if nesterov else M
        W.mul_(1 - lr * weight_decay).sub_(torch.from_numpy(lr * update_scale * newton_schulz(U.double().numpy(), steps)).float())
        G.zero_()
    k.score_logprobs, k.score_logprobs_grad, k.muon_apply = score_logprobs, score_logprobs_grad, muon_apply
    k.score_logprobs_workspace = k.score_logprobs_grad_workspace = lambda n, I, d: 16
    k.orthogonalize_workspace = lambda rows, d: 16
    k.add_rows = lambda T, ids, R: T.index_add_(0, ids.long(), R)
    return k


def _matrix(U=40, I=60, seed=1):
    rng = np.random.default_rng(seed)
    m = sp.random(U, I, 0.1, random_state=rng, data_rvs=lambda n: np.ones(n)).tocsr()
    m[3] = 0                                           # a user without interactions
    m.eliminate_zeros()
    return m


def _dataset(mat):
    import recsys_pytorch_amd as pkg
    return pkg.InteractionData(mat)


def _conf(batch, epochs):
    return types.SimpleNamespace(batch_size=batch, num_epochs=epochs, verbose=0, test_from=1, test_step=1)


def test_refusals(monkeypatch):
    import recsys_pytorch_amd as pkg
    from recsys_pytorch_amd.sharded import BPREngine, dist
    ds, k = _dataset(_matrix()), _plain_kernels()
    with pytest.raises(ValueError, match="two losses"):
        pkg.MF(ds, dict(HP, pointwise=True, listwise=True), "cpu", kernels=k)
    with pytest.raises(ValueError, match="optimizer"):
        pkg.MF(ds, dict(HP, optimizer="lion"), "cpu", kernels=k)
    m = pkg.MF(ds, dict(HP, optimizer="muon"), "cpu", kernels=k)
    with pytest.raises(ValueError, match="SGD"):
        m._engine.native_trainer(torch.zeros(41, dtype=torch.int64), torch.zeros(0, dtype=torch.int32), 4)
    for items in (np.zeros(3), np.zeros((2, 2, 2)), np.int32(4)):
        with pytest.raises(ValueError, match="items must be"):
            m.predict_logprobs([0, 1], items)
    monkeypatch.setattr(dist, "is_initialized", lambda: True)
    monkeypatch.setattr(dist, "get_world_size", lambda group=None: 2)
    monkeypatch.setattr(dist, "get_backend", lambda group=None: "gloo")
    P, Q = torch.zeros(4, 32), torch.zeros(5, 32)
    with pytest.raises(ValueError, match="one GPU"):
        BPREngine(P, Q, 0.1, kernels=k, optimizer="muon")
    with pytest.raises(ValueError, match="one GPU"):
        BPREngine(P, Q, 0.1, kernels=k).listwise_step(torch.zeros(1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("optimizer", ["sgd", "adam", "muon"])
def test_listwise_step_on_plain_kernels_is_the_softmax_losss_step(optimizer):
    """two steps against torch's own differentiation of the mean loss in 64 bits; users and items twice, an item that is none"""
    import recsys_pytorch_amd as pkg
    ds = types.SimpleNamespace(num_users=12, num_items=20)
    torch.manual_seed(3)
    m = pkg.MF(ds, dict(HP, hidden_dim=24, optimizer=optimizer, listwise=True, lr=0.05), "cpu", kernels=_plain_kernels())
    ref = [t[:, :24].double().clone() for t in (m._P, m._Q)]
    state = [[torch.zeros_like(t), torch.zeros_like(t)] for t in ref]
    u, i = torch.tensor([0, 3, 3, 11, 5]), torch.tensor([7, 7, 2, 19, -1])
    for t in (1, 2):
        for w in ref:
            w.requires_grad_(True)
        nll = torch.logsumexp(ref[0][u] @ ref[1].T, 1) - (ref[0][u] * ref[1][i]).sum(1)
        loss = nll[:4].sum() / 5
        g = torch.autograd.grad(loss, ref)
        assert abs(float(m.process_one_batch(u, i, None)) - float(loss)) < 1e-5 * float(loss)
        assert abs(float(m.train_step(u, i, None)) - float(loss)) < 1e-5 * float(loss)
        with torch.no_grad():
            for w, gr, (a, b) in zip(ref, g, state):
                w.requires_grad_(False)
                if optimizer == "sgd":
                    w -= 0.05 * gr
                elif optimizer == "adam":
                    a += 0.1 * (gr - a)
                    b.mul_(0.999).addcmul_(gr, gr, value=1e-3)
                    w -= 0.05 / (1 - 0.9 ** t) * a / (b.sqrt() / (1 - 0.999 ** t) ** 0.5 + 1e-8)
                else:
                    a.mul_(0.95).add_(gr)
                    w -= 0.05 * max(1.0, w.shape[0] / 24) ** 0.5 * torch.from_numpy(newton_schulz((gr + 0.95 * a).numpy(), 5))
        if optimizer == "sgd":                         # (the others divide by what the fp32 gradients' rounding reaches)
            for got, want in ((m._P, ref[0]), (m._Q, ref[1])):
                assert (got[:, :24].double() - want).abs().max() < 1e-6
        assert (m._P[:, 24:] == 0).all() and (m._Q[:, 24:] == 0).all()
    assert not m._engine.G.any() and not m._engine.GP.any()
    assert m._engine.step_count == 2


@pytest.mark.parametrize("optimizer", ["sgd", "muon"])
def test_listwise_fit_on_plain_kernels_takes_the_samplers_positives(optimizer):
    import recsys_pytorch_amd as pkg
    mat = _matrix()
    ds, k = _dataset(mat), _plain_kernels()
    m = pkg.MF(ds, dict(HP, optimizer=optimizer, listwise=True), "cpu", kernels=k)
    logged = []
    m.fit(ds, _conf(16, 2), loggers=[types.SimpleNamespace(log_metrics=lambda d, epoch: logged.append(d["loss"]))])
    assert [len(c[0]) for c in k.calls] == [16, 16, 8] * 2 and len(logged) == 2 and np.isfinite(logged).all()
    dense = mat.toarray() > 0
    for u, i, g in k.calls:
        assert i.shape == (len(u), 1) and torch.allclose(g, torch.full_like(g, -1.0 / len(u)))
        for a, b in zip(u.tolist(), i[:, 0].tolist()):
            assert dense[a, b] if a != 3 else b == -1
    assert m._engine.step_count == 6


def test_predict_logprobs_on_plain_kernels():
    import recsys_pytorch_amd as pkg
    mat = _matrix()
    m = pkg.MF(_dataset(mat), dict(HP, optimizer="sgd"), "cpu", kernels=_plain_kernels())
    users = np.array([5, 0, 39, 5])
    r = m.predict_logprobs(users, np.array([1, 2, 3, 4]), eval_pos=mat, K=7, test_batch_size=3)
    one = m.predict_logprobs(users, np.array([[1, 1], [2, 0], [3, 5], [4, 1]]), eval_pos=mat, K=7)
    assert r.logp.shape == (4,) and one.logp.shape == (4, 2) and r.top_idx.shape == (4, 7)
    assert np.array_equal(r.logp, one.logp[:, 0]) and all(np.array_equal(a, b) for a, b in zip(r[1:], one[1:]))
    assert m.predict_logprobs(users).logp is None and m.predict_logprobs(users).top_idx is None
    assert m.predict_logprobs([], np.zeros((0, 3)), K=2).logp.shape == (0, 3)


def test_predict_logprobs_of_ids_beyond_32_bits():
    """an id that names nothing names nothing, whatever its lower half is"""
    import recsys_pytorch_amd as pkg
    mat = _matrix()
    m = pkg.MF(_dataset(mat), dict(HP, optimizer="sgd"), "cpu", kernels=_plain_kernels())
    far = 2 ** 32
    r = m.predict_logprobs([5, far + 5, -far], np.array([[1, far + 1], [1, 2], [3, 4]]), K=3)
    want = m.predict_logprobs([5, -1, -1], np.array([[1, -1], [1, 2], [3, 4]]), K=3)
    assert all(np.array_equal(a, b) for a, b in zip(r, want))
    assert r.logp[0, 1] == 0.0 and r.lse[1] == -np.inf and (r.top_idx[1:] == -1).all()


@pytest.mark.parametrize("argv", [["--listwise"], ["--optimizer", "muon"]])
def test_command_line_refuses_what_a_model_lacks(argv, capsys):
    from recsys_pytorch_amd import main
    with pytest.raises(SystemExit) as stop:
        main.main(["--data", "nowhere.npz", "--model", "LightGCN", *argv])
    assert stop.value.code == 2 and "LightGCN" in capsys.readouterr().err


# ---- on the GPU ------------------------------------------------------------------------------------------------------------------
def _engine(U, I, d, optimizer="sgd", lr=0.5, seed=5):
    from recsys_pytorch_amd.sharded import BPREngine
    rng = np.random.default_rng(seed)
    P, Q = ((rng.standard_normal((n, d)) * (4.0 / d) ** 0.25).astype(np.float32) for n in (U, I))
    return BPREngine(torch.from_numpy(P).cuda(), torch.from_numpy(Q).cuda(), lr, optimizer=optimizer), P.astype(np.float64), Q.astype(np.float64)


@pytest.mark.gpu
@pytest.mark.parametrize("U,I,n,d", [(7, 1, 1, 32), (50, 333, 1, 64), (50, 333, 77, 64), (300, 1682, 256, 128), (40, 901, 33, 256)])
def test_hip_listwise_step_vs_formula(U, I, n, d):
    lr = 0.5
    eng, P, Q = _engine(U, I, d)
    rng = np.random.default_rng(n)
    u, i = rng.integers(0, U, n), rng.integers(0, I, n)
    i[n // 2:n // 2 + 1] = -1 if n > 1 else i[0]
    loss = eng.listwise_step(torch.from_numpy(u.astype(np.int32)).cuda(), torch.from_numpy(i.astype(np.int32)).cuda())
    logp, lse, ent, _, _, ez = reference(P, Q, u, i[:, None], 0, None, 1.0)
    el = ez + 5e-5
    assert abs(float(loss.sum()) + logp.sum()) <= (el + 2.0 ** -24 * np.abs(logp[:, 0])).sum() + n * 2.0 ** -24 * np.abs(logp).sum()
    g = np.full((n, 1), np.float64(np.float32(-1.0 / n)))
    GP, GQ, cP, cQ, gP, gQ, ezm, w, wP, topQ = gradient(P, Q, u, i[:, None], g, None, lse, ent, None, 1.0)
    rel = ezm + 1.2e-5 + el.max() + 2.0 ** -22 + 2.0 ** -20
    tP = (rel + 3 * I * 2.0 ** -24) * cP + 2.0 ** -20 * gP + 2.0 ** -37 * I * topQ * w[:, None] + 2.0 ** -24 * np.abs(GP) + 1e-37
    tQ = (rel + 3 * n * 2.0 ** -24) * cQ + (2.0 ** -20 + 3 * n * 2.0 ** -24) * gQ + 2.0 ** -37 * n * wP.max() + 2.0 ** -24 * np.abs(GQ) + 1e-37
    sP, stP, saP = np.zeros_like(P), np.zeros_like(P), np.zeros_like(P)
    np.add.at(sP, u, GP)
    np.add.at(stP, u, tP)
    np.add.at(saP, u, np.abs(GP) + tP)
    count = np.bincount(u, minlength=U)[:, None]
    for got, old, grad, tol in ((eng.P, P, sP, stP + count * 2.0 ** -24 * saP), (eng.Q, Q, GQ, tQ)):
        want = old - lr * grad
        tol = lr * (tol + 2.0 ** -24 * (np.abs(grad) + tol)) * 1.001 + 2.0 ** -24 * (np.abs(want) + lr * tol)
        assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    assert not eng.G.any() and not eng.GP.any()


@pytest.mark.gpu
@pytest.mark.parametrize("branch", ["listwise", "bpr", "pointwise"])
def test_hip_muon_steps_are_the_calls_they_are_made_of(branch):
    """three steps of the engine, users and items of a step distinct where the branch sums by atomics: the same bits as the calls"""
    from recsys_pytorch_amd import rsx
    U, I, d, n, lr = 211, 500, 64, 90, 0.02
    eng, P, Q = _engine(U, I, d, "muon", lr)
    eng.muon_width = 50
    P, Q = eng.P.clone(), eng.Q.clone()
    mP, mQ = torch.zeros_like(P), torch.zeros_like(Q)
    rng = np.random.default_rng(0)
    dev = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
    for _ in range(3):
        perm = rng.permutation(I)
        u, i, j = dev(rng.permutation(U)[:n]), dev(perm[:n]), dev(perm[n:2 * n])
        GP, GQ = torch.zeros_like(P), torch.zeros_like(Q)
        if branch == "listwise":
            u[:20] = u[20:40]                           # (this branch has no atomics: users and items twice)
            i[:30] = i[30:60]
            eng.listwise_step(u, i)
            lp = rsx.score_logprobs(P, Q, u, i.view(-1, 1))
            R, GQ = rsx.score_logprobs_grad(P, Q, u, i.view(-1, 1), lp.lse, torch.full((n, 1), -1.0 / n, device="cuda"))
            rsx.add_rows(GP, u, R)
        elif branch == "bpr":
            eng.step(u, i, j)
            rsx.bpr_grad(P, Q, GP, GQ, u, i, j, 1.0 / n)
        else:
            y = torch.from_numpy(rng.random(n).astype(np.float32)).cuda()
            eng.pointwise_step(u, i, y)
            rsx.pointwise_grad(P, Q, GP, GQ, u, i, y, 1.0 / n)
        rsx.muon_apply(Q, mQ, GQ, lr, update_scale=(I / 50) ** 0.5)
        rsx.muon_apply(P, mP, GP, lr, update_scale=(U / 50) ** 0.5)
        assert torch.equal(eng.P, P) and torch.equal(eng.Q, Q) and not eng.G.any() and not eng.GP.any()


def _fit(mat, steps=2, **hp):
    import recsys_pytorch_amd as pkg
    ds = _dataset(mat)
    torch.manual_seed(11)
    m = pkg.MF(ds, dict(HP, hidden_dim=50, **hp), "cuda")
    start = m._P.clone(), m._Q.clone()
    m.fit(ds, _conf(64, steps))
    return m, start


@pytest.mark.gpu
@pytest.mark.parametrize("hp", [{"listwise": True, "optimizer": "sgd"}, {"listwise": True, "optimizer": "adam"}, {"listwise": True, "optimizer": "muon"},
                                {"optimizer": "muon"}, {"pointwise": True, "optimizer": "muon"}], ids=lambda h: "-".join(map(str, h.values())))
def test_hip_fit_runs(hp):
    """padded columns stay zero, a batch with a user who has no interactions is one; the listwise branch repeats itself bit by bit"""
    mat = _matrix(150, 333)
    m, start = _fit(mat, **hp)
    for now, was in zip((m._P, m._Q), start):
        assert torch.isfinite(now).all() and not torch.equal(now, was) and not now[:, 50:].any()
    if hp.get("listwise"):
        again, _ = _fit(mat, **hp)
        assert torch.equal(m._P, again._P) and torch.equal(m._Q, again._Q)


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["MF", "LightGCN"])
def test_hip_predict_logprobs_of_the_models(name):
    import recsys_pytorch_amd as pkg
    mat = _matrix(150, 333)
    ds = _dataset(mat)
    torch.manual_seed(11)
    if name == "MF":
        m = pkg.MF(ds, dict(HP, hidden_dim=50, optimizer="sgd"), "cuda")
        P, Q = m._P, m._Q
    else:
        m = pkg.LightGCN(ds, {"emb_dim": 50, "num_layers": 2, "node_dropout": 0.0, "split": False, "num_folds": 100, "reg": 1e-4, "graph_dir": "graph"}, "cuda")
        m.getSparseGraph(mat)
        m.update_lightgcn_embedding()
        P, Q = m.user_embeddings, m.item_embeddings
    rng = np.random.default_rng(2)
    users, items = rng.permutation(150)[:101], rng.integers(0, 333, (101, 3))
    csr = sp.csr_matrix(mat)
    csr.sort_indices()
    for pos in (None, mat):
        r = m.predict_logprobs(users, items, eval_pos=pos, K=9, test_batch_size=40)
        want = reference(P.double().cpu().numpy(), Q.double().cpu().numpy(), users, items, 9, None if pos is None else (csr.indptr, csr.indices), 1.0)
        el = want[5] + 5e-5
        fine = np.isfinite(want[0])
        assert np.array_equal(r.logp[~fine], want[0][~fine]) and np.array_equal(r.top_idx, want[3])
        assert (np.abs(r.logp[fine] - want[0][fine]) <= (el[:, None] + 2.0 ** -24 * np.abs(want[0]))[fine]).all()
        assert (np.abs(r.lse - want[1]) <= el + 2.0 ** -24 * np.abs(want[1])).all()
        assert (np.abs(r.entropy - want[2]) <= el * (2 + want[2]) + want[5]).all()
        assert (np.abs(r.top_logp - want[4]) <= el[:, None] + 2.0 ** -24 * np.abs(want[4])).all()


@pytest.mark.gpu
def test_hip_command_line_takes_them(tmp_path):
    from recsys_pytorch_amd import main
    path = tmp_path / "ratings.txt"
    path.write_text("".join(f"{u}\t{u + n}\t5\t{12 * u + n}\n" for u in range(30) for n in range(12)))
    ret = main.main(["--data", str(path), "--hidden-dim", "32", "--optimizer", "muon", "--listwise", "--batch-size", "8", "--num-epochs", "2"])
    assert all(np.isfinite(v) for v in ret["scores"].values())


@pytest.mark.gpu
def test_hip_calls_at_once_on_two_streams():
    """the calls of two training steps side by side, workspaces their own: the same bits as one after the other"""
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(9)
    f = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()
    jobs = []
    for U, I, d, n in ((300, 5000, 64, 200), (500, 3001, 128, 129)):
        jobs.append((f(U, d), f(I, d), torch.from_numpy(rng.integers(0, U, n).astype(np.int32)).cuda(), torch.from_numpy(rng.integers(0, I, (n, 2)).astype(np.int32)).cuda(), f(n, 2)))

    def step(P, Q, u, it, g):
        P, Q, M = P.clone(), Q.clone(), torch.zeros_like(Q)
        lp = rsx.score_logprobs(P, Q, u, it, K=10)
        GP, GQ = rsx.score_logprobs_grad(P, Q, u, it, lp.lse, g)
        rsx.add_rows(P, u, GP)
        rsx.muon_apply(Q, M, GQ, 0.02)
        return (*lp, GP, P, Q, M, rsx.orthogonalize(P))
    want = [step(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(*jobs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for run in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[k]))


@pytest.mark.gpu
@pytest.mark.parametrize("optimizer", ["sgd", "muon"])
def test_hip_captured_listwise_step_outlives_larger_eager_ones(optimizer):
    """a step of 60 pairs replayed from its graph after an eager step of 700 and other work in the memory between: the same bits as eager steps"""
    rng = np.random.default_rng(4)
    dev = lambda n, top: torch.from_numpy(rng.integers(0, top, n).astype(np.int32)).cuda()
    (eng, *_), (twin, *_) = _engine(200, 900, 64, optimizer), _engine(200, 900, 64, optimizer)
    u, i, many_u, many_i = dev(60, 200), dev(60, 900), dev(700, 200), dev(700, 900)
    for e in (eng, twin):
        e.listwise_step(u, i)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        eng.listwise_step(u, i)
    torch.cuda.synchronize()
    for _ in range(3):
        for e in (eng, twin):
            e.listwise_step(many_u, many_i)
        others = [torch.full((1 << 18,), 7.0, device="cuda") for _ in range(40)]
        torch.cuda.synchronize()
        graph.replay()
        twin.listwise_step(u, i)
        torch.cuda.synchronize()
        assert torch.equal(eng.P, twin.P) and torch.equal(eng.Q, twin.Q) and all(bool((o == 7.0).all()) for o in others)
