"""rsx.orthogonalize / rsx.muon_apply against the iteration written out in 64 bits (X_k itself, no Gram shortcut).

Tolerance of the product X M (M the [d x d] polynomial, rounded once to fp32; d products summed in fp32):
|O - O*| <= (d + 3) 2^-24 |X| |M|, elementwise -- the standard bound of a dot product -- plus 2^-8 |O*| where the result is
rounded to bf16.  The [d x d] part is in 64 bits: its noise (2^-53 amplified by a^2 a step) is 1e-9 of |X| |M| at most for the six
steps used here, and is allowed for as such."""
import math
import os

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COEFFS = (3.4445, -4.7750, 2.0315)


def newton_schulz(X, steps, coeffs=COEFFS, eps=1e-7):
    a, b, c = coeffs
    X = X / (np.sqrt((X * X).sum()) + eps)
    for _ in range(steps):
        A = X.T @ X
        X = a * X + X @ (b * A + c * (A @ A))
    return X


def polynomial(X, steps, coeffs=COEFFS, eps=1e-7):
    """M with newton_schulz(X) == X @ M"""
    a, b, c = coeffs
    s = 1.0 / (np.sqrt((X * X).sum()) + eps)
    A, M = s * s * (X.T @ X), s * np.eye(X.shape[1])
    for _ in range(steps):
        T = a * np.eye(X.shape[1]) + b * A + c * (A @ A)
        M, A = M @ T, T @ A @ T
    return M


def bound(X, steps, want, bf16=False, **kw):
    d = X.shape[1]
    terms = np.abs(X) @ np.abs(polynomial(X, steps, **kw))
    return ((d + 3) * 2.0 ** -24 + 1e-9) * terms + (2.0 ** -8 * np.abs(want) if bf16 else 0.0) + 1e-30


def matrix(rng, rows, d, spread=2.0):
    mix = rng.standard_normal((d, d)) / math.sqrt(d) * np.logspace(0, -spread, d)
    return (rng.standard_normal((rows, d)) @ mix).astype(np.float32)


# ---- refusals (no GPU) ---------------------------------------------------------------------------------------------------------
def test_refusals():
    import torch
    from recsys_pytorch_amd import build, rsx
    build.build()
    X = torch.zeros(4, 32)
    for call in (lambda: rsx.orthogonalize(X), lambda: rsx.orthogonalize(X.half()), lambda: rsx.orthogonalize(X[0]),
                 lambda: rsx.muon_apply(X, X.clone(), X.clone(), 0.1), lambda: rsx.orthogonalize_workspace(4, 48), lambda: rsx.orthogonalize_workspace(-1, 32)):
        with pytest.raises(rsx.RsxError):
            call()
    L = rsx.lib()
    good = dict(rows=4, d=32, dtype=0, steps=5, a=1.0, b=0.0, c=0.0, eps=0.0)

    def orth(X=16, out=16, ws=0, ws_bytes=0, **kw):
        k = {**good, **kw}
        return L.rsx_orthogonalize(X, out, k["rows"], k["d"], k["dtype"], k["steps"], k["a"], k["b"], k["c"], k["eps"], ws, ws_bytes, None)
    assert orth(d=48) == -1 and orth(rows=-1) == -1 and orth(dtype=2) == -1 and orth(steps=33) == -1 and orth(steps=-1) == -1
    assert orth(a=float("nan")) == -1 and orth(eps=-1.0) == -1 and orth(X=0) == -1 and orth(X=8) == -1 and orth(out=24) == -1
    assert orth() == -3 and b"workspace" in L.rsx_last_error() and orth(rows=0) == 0

    def muon(momentum=0.9, lr=0.1, ws=0, ws_bytes=0, rows=4, g=16):
        return L.rsx_muon_apply(16, 16, g, rows, 32, 0, lr, momentum, 1, 5, 1.0, 0.0, 0.0, 0.0, 0.0, 1.0, ws, ws_bytes, None)
    assert muon(momentum=1.0) == -1 and muon(momentum=-0.1) == -1 and muon(lr=float("inf")) == -1 and muon(g=20) == -1
    assert muon() == -3 and muon(rows=0) == 0


def test_a_workspace_between_16_byte_lines_is_refused():
    """the kernels read it 16 bytes at a time"""
    from recsys_pytorch_amd import build, rsx
    build.build()
    L = rsx.lib()
    for ws in (8, 4104):
        assert L.rsx_orthogonalize(16, 16, 4, 32, 0, 5, 1.0, 0.0, 0.0, 0.0, ws, 1 << 30, None) == -3 and b"16-byte" in L.rsx_last_error()
        assert L.rsx_muon_apply(16, 32, 48, 4, 32, 0, 0.1, 0.9, 1, 5, 1.0, 0.0, 0.0, 0.0, 0.0, 1.0, ws, 1 << 30, None) == -3 and b"16-byte" in L.rsx_last_error()


def test_the_polynomial_is_the_iteration():
    """the bound's M against the iteration itself, and the Gram-space form against it (64 bits, CPU)"""
    rng = np.random.default_rng(0)
    for rows, d in ((50, 32), (7, 32), (300, 64)):
        X = matrix(rng, rows, d).astype(np.float64)
        O = newton_schulz(X, 5)
        assert np.abs(X @ polynomial(X, 5) - O).max() < 1e-9
        if rows > d:
            s = np.linalg.svd(O, compute_uv=False)
            assert s[:d // 4].min() > 0.6 and s.max() < 1.3          # the large directions are near one


# ---- GPU ---------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("d", [32, 64, 128, 256])
@pytest.mark.parametrize("rows", [1, 5, 31, 64, 257, 1000, 6007])
@pytest.mark.parametrize("bf16", [False, True])
def test_hip_orthogonalize_vs_iteration(rows, d, bf16):
    import torch
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(rows * 1000 + d)
    X = torch.from_numpy(matrix(rng, rows, d)).cuda()
    X = X.bfloat16() if bf16 else X
    X64 = X.double().cpu().numpy()
    for steps in (5,) if rows not in (64, 257) else (0, 1, 2, 5, 6):
        got = rsx.orthogonalize(X, steps=steps)
        assert got.dtype == X.dtype
        want = newton_schulz(X64, steps)
        err = np.abs(got.double().cpu().numpy() - want)
        assert (err <= bound(X64, steps, want, bf16)).all(), (steps, err.max(), np.abs(want).max())
        assert torch.equal(got, rsx.orthogonalize(X, steps=steps))                    # the same bits again


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
def test_hip_orthogonalize_in_place_zero_columns_and_other_coefficients(d):
    import torch
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(d)
    X0 = matrix(rng, 777, d)
    X0[:, d - 14:] = 0.0                                    # padded columns stay zero
    X64 = X0.astype(np.float64)
    X = torch.from_numpy(X0).cuda()
    kw = dict(coeffs=(1.5, -0.5, 0.0), eps=1e-3)            # the cubic iteration
    out = rsx.orthogonalize(X, steps=6, out=X, **kw)
    assert out is X and float(X[:, d - 14:].abs().max()) == 0.0
    want = newton_schulz(X64, 6, **kw)
    assert (np.abs(X.double().cpu().numpy() - want) <= bound(X64, 6, want, **kw)).all()
    Z = torch.zeros(100, d, device="cuda")
    assert float(rsx.orthogonalize(Z).abs().max()) == 0.0
    Z[3, 5] = float("nan")
    assert bool(rsx.orthogonalize(Z).isnan().all())
    assert rsx.orthogonalize(torch.zeros(0, d, device="cuda")).shape == (0, d)


def _muon_reference(W, M, G, lr, mu, nesterov, steps, wd, scale):
    """M as the kernel rounds it (one rounding per fused multiply-add), the rest in 64 bits"""
    mu = np.float64(np.float32(mu))
    M1 = (mu * M + G).astype(np.float32).astype(np.float64)
    U = (mu * M1 + G).astype(np.float32).astype(np.float64) if nesterov else M1
    O = newton_schulz(U, steps)
    return M1, O, (1 - lr * wd) * W - lr * scale * O, U


@pytest.mark.gpu
@pytest.mark.parametrize("rows,d", [(40, 32), (333, 64), (5000, 128), (1234, 256), (20_001, 32)])
@pytest.mark.parametrize("bf16", [False, True])
def test_hip_muon_apply(rows, d, bf16):
    import torch
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(d + rows)
    W = torch.from_numpy((rng.standard_normal((rows, d)) * 0.1).astype(np.float32)).cuda()
    M = torch.from_numpy(matrix(rng, rows, d)).cuda()
    ws = torch.empty(rsx.orthogonalize_workspace(rows, d) // 8 + 1, dtype=torch.int64, device="cuda")
    for nesterov, wd, scale in ((True, 0.01, None), (False, 0.0, 0.25)):
        G = torch.from_numpy(matrix(rng, rows, d)).cuda()
        G = G.bfloat16() if bf16 else G
        W64, M64, G64 = (t.double().cpu().numpy() for t in (W, M, G))
        s = max(1.0, rows / d) ** 0.5 if scale is None else scale
        M1, O, W1, U = _muon_reference(W64, M64, G64, 0.02, 0.9, nesterov, 5, wd, s)
        rsx.muon_apply(W, M, G, 0.02, momentum=0.9, nesterov=nesterov, weight_decay=wd, update_scale=scale, ws=ws)
        assert float(G.float().abs().max()) == 0.0
        assert (np.abs(M.double().cpu().numpy() - M1) <= 2.0 ** -23 * np.abs(M1)).all()
        tol = 0.02 * s * bound(U, 5, O) + 4 * 2.0 ** -24 * (np.abs(W64) + np.abs(0.02 * s * O))
        assert (np.abs(W.double().cpu().numpy() - W1) <= tol).all()


@pytest.mark.gpu
def test_hip_muon_apply_captured_and_on_a_side_stream():
    """the step replayed from a graph equals the eager one, with eager work between the replays; and on a stream of its own"""
    import torch
    from recsys_pytorch_amd import rsx
    rng = np.random.default_rng(3)
    rows, d = 3001, 128
    W0, M0, G0 = (torch.from_numpy(matrix(rng, rows, d)).cuda() for _ in range(3))
    eager = [t.clone() for t in (W0, M0)]
    ws = [torch.empty(rsx.orthogonalize_workspace(rows, d) // 8 + 1, dtype=torch.int64, device="cuda") for _ in range(2)]
    W, M, G = W0.clone(), M0.clone(), torch.zeros_like(G0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        rsx.muon_apply(W.clone(), M.clone(), G0.clone(), 0.01, ws=ws[0])
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            G.copy_(G0)
            rsx.muon_apply(W, M, G, 0.01, ws=ws[0])
    torch.cuda.synchronize()
    for _ in range(4):
        graph.replay()
        g = G0.clone()
        rsx.muon_apply(eager[0], eager[1], g, 0.01, ws=ws[1])
        torch.cuda.synchronize()
        assert torch.equal(W, eager[0]) and torch.equal(M, eager[1])
