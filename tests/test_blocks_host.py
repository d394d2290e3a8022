"""The gated delta rule, the norms around a block and gradient clipping without a GPU: the plain restatement that the GPU tests compare with is held to
autograd and to differences, its bounds to a computation in float32, and calls that cannot be right are refused before anything reaches a device."""
import ctypes

import numpy as np
import pytest
import torch

from tests import blocks_ref as ref
from tests.test_rows_host import _refused

R4 = np.array([[12, 40], [0, 5], [7, 7], [5, 12]])


def _maps(rng, N=43, H=4, G=2, Kd=5, Vd=3):
    f = lambda *s: rng.standard_normal(s)  # noqa: E731
    unit = lambda t: (t / np.sqrt((t ** 2).sum(2, keepdims=True))).reshape(N, -1)  # noqa: E731
    return dict(Q=unit(f(N, G, Kd)), K=unit(f(N, G, Kd)), V=f(N, H * Vd), beta=1 / (1 + np.exp(-f(N, H))), decay=-np.exp(f(N, H) - 2)), f(N, H * Vd)


def _torch_delta(v, R, G, scale):
    N, H = v["beta"].shape
    of = torch.arange(H) // (H // G)
    q, k, x = v["Q"].view(N, G, -1)[:, of], v["K"].view(N, G, -1)[:, of], v["V"].view(N, H, -1)
    rows = torch.zeros_like(x)
    for s, e in R.tolist():
        S = torch.zeros(H, k.shape[2], x.shape[2], dtype=torch.float64)
        for t in range(s, e):
            if v["decay"] is not None:
                S = torch.exp(v["decay"][t])[:, None, None] * S
            u = v["beta"][t][:, None] * (x[t] - (S * k[t][:, :, None]).sum(1))
            S = S + k[t][:, :, None] * u[:, None]
            rows = rows.index_put((torch.tensor(t),), scale * (S * q[t][:, :, None]).sum(1))
    return rows.view(N, -1)


@pytest.mark.parametrize("decays", [True, False])
def test_restated_delta_rule_agrees_with_autograd_and_differences(decays):
    rng = np.random.default_rng(5)
    v, dO = _maps(rng)
    if not decays:
        v["decay"] = None
    call = lambda d=None: ref.delta(v["Q"], v["K"], v["V"], v["beta"], v["decay"], R4, 2, 0.7, dO=d)  # noqa: E731
    got = call(dO)
    t = {k: None if a is None else torch.from_numpy(a).requires_grad_() for k, a in v.items()}
    O = _torch_delta(t, R4, 2, 0.7)
    inside = ~np.isnan(got[0][:, 0])
    assert inside.sum() == 40
    np.testing.assert_allclose(got[0][inside], O.detach().numpy()[inside], rtol=1e-11, atol=1e-13)
    O.backward(torch.from_numpy(dO))
    names = ("Q", "K", "V", "beta", "decay")
    for name, grad in zip(names, got[2:]):
        if t[name] is not None:
            np.testing.assert_allclose(grad[inside], t[name].grad.numpy()[inside], rtol=1e-9, atol=1e-11, err_msg=name)
    f = lambda: np.nansum(call()[0] * dO)  # noqa: E731
    for name, grad in zip(names, got[2:]):
        if v[name] is None:
            continue
        for i in ((1, 2), (13, 0), (30, 3)):
            old, step = v[name][i], 1e-5
            v[name][i] = old + step
            up = f()
            v[name][i] = old - step
            down = f()
            v[name][i] = old
            assert abs((up - down) / (2 * step) - grad[i]) < 1e-7 * (1 + abs(grad[i])), name


def _chunked_in_float32(v, R, G, scale, dO):
    """The chunked form in float32, forward and the values' gradient, for one region: what the bounds have to hold for."""
    N, H = v["beta"].shape
    f = np.float32
    O, dV = np.full((N, H, v["V"].shape[1] // H), np.nan), np.full((N, H, v["V"].shape[1] // H), np.nan)
    for h in range(H):
        q, k, x = (v[n].reshape(N, m, -1)[:, h // (H // G) if m == G else h].astype(f) for n, m in (("Q", G), ("K", G), ("V", H)))
        b, g = v["beta"][:, h].astype(f), v["decay"][:, h].astype(f)
        for s, e in R.tolist():
            S, held = np.zeros((k.shape[1], x.shape[1]), f), []
            for c in range(s, e, 16):
                at = slice(c, min(c + 16, e))
                n = at.stop - c
                D = np.array([[np.exp(g[c:][j + 1:i + 1].sum()) if j <= i else 0 for j in range(n)] for i in range(n)], f)
                first = np.exp(np.cumsum(g[at]))
                T = np.linalg.inv((np.eye(n) + b[at][:, None] * D * np.tril(k[at] @ k[at].T, -1)).astype(f)).astype(f)
                Pm = D * (q[at] @ k[at].T)
                u = T @ (b[at][:, None] * (x[at] - first[:, None] * (k[at] @ S)))
                O[at, h] = f(scale) * (first[:, None] * (q[at] @ S) + Pm @ u)
                held.append((at, D, first, T, Pm))
                S = first[-1] * S + k[at].T @ (D[-1][:, None] * u)
            dS = np.zeros_like(S)
            for at, D, first, T, Pm in reversed(held):
                d = f(scale) * dO[at].reshape(at.stop - at.start, H, -1)[:, h].astype(f)
                dy = T.T @ (Pm.T @ d + D[-1][:, None] * (k[at] @ dS))
                dV[at, h] = b[at][:, None] * dy
                dS = first[-1] * dS - k[at].T @ (first[:, None] * b[at][:, None] * dy) + q[at].T @ (first[:, None] * d)
    return O.reshape(N, -1), dV.reshape(N, -1)


def test_bounds_of_the_delta_rule_hold_in_float32_and_are_not_empty():
    rng = np.random.default_rng(6)
    v, dO = _maps(rng, N=203, H=2, G=1, Kd=24, Vd=6)
    v = {k: a.astype(np.float32).astype(np.float64) for k, a in v.items()}
    dO = dO.astype(np.float32).astype(np.float64)
    R = np.array([[150, 203], [0, 150]])
    want = ref.delta(v["Q"], v["K"], v["V"], v["beta"], v["decay"], R, 1, 0.2, dO=dO)
    bounds = ref.delta_bounds(v["Q"], v["K"], v["V"], v["beta"], v["decay"], R, 1, 0.2, dO=dO)
    O, dV = _chunked_in_float32(v, R, 1, 0.2, dO)
    u = 2.0 ** -24
    assert (np.abs(O - want[0]) <= u * bounds[0]).all() and (np.abs(dV - want[4]) <= u * bounds[4]).all()
    # worst cases of all roundings at once, they lie far above what happens, but still far below the values
    for b, w in zip(bounds, want):
        assert np.nanmedian(u * b) < 2.0 ** -5 * np.sqrt(np.nanmean(w ** 2))
    # roundings that do not conspire: the bound by norms that the GPU tests add holds here as well
    for got, w in ((O, want[0]), (dV, want[4])):
        assert np.linalg.norm(got - w) <= 32 * u * np.linalg.norm(w)


@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("norm,nxt", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("gated", [True, False])
def test_restated_block_norms_agree_with_autograd(rms, norm, nxt, gated):
    rng = np.random.default_rng(7)
    n, nchunk, w = 5, 3, 7
    m = nchunk * w
    f = lambda *s: rng.standard_normal(s)  # noqa: E731
    a = dict(Y=f(n, m), R=f(n, m), gate=f(n, m) if gated else None, gamma=f(1, m) if norm else np.ones((1, m)), beta=f(1, m) if norm else np.zeros((1, m)), scale=f(1, m),
             ngamma=f(1, m), nbeta=f(1, m))
    dR, dZ = f(n, m), f(n, m)
    eps = 1e-2
    t = {k: None if x is None else torch.from_numpy(x).requires_grad_() for k, x in a.items()}

    def normed(x):
        v = x.view(n, nchunk, w)
        c = v if rms else v - v.mean(2, keepdim=True)
        return (c / torch.sqrt((c * c).mean(2, keepdim=True) + eps)).reshape(n, m)

    p = (normed(t["Y"]) if norm else t["Y"]) * t["gamma"] + t["beta"]
    O = t["R"] + t["scale"] * p * (torch.nn.functional.silu(t["gate"]) if gated else 1)
    loss = (O * torch.from_numpy(dR)).sum()
    (Or, Zr, _), _ = ref.blocknorm(*(a[k] for k in a), nchunk, rms, norm, nxt, eps)
    np.testing.assert_allclose(Or, O.detach().numpy(), rtol=1e-12, atol=1e-13)
    if nxt:
        Z = normed(O) * t["ngamma"] + t["nbeta"]
        np.testing.assert_allclose(Zr, Z.detach().numpy(), rtol=1e-11, atol=1e-12)
        loss = loss + (Z * torch.from_numpy(dZ)).sum()
    loss.backward()
    grads, sizes = ref.blocknorm_bprop(*(a[k] for k in a), nchunk, rms, norm, nxt, eps, dR, dZ, Or)
    for k, got, size in zip(("Y", "R", "gate", "gamma", "beta", "scale", "ngamma", "nbeta"), grads, sizes):
        if t[k] is None or t[k].grad is None:
            continue
        np.testing.assert_allclose(got, t[k].grad.numpy(), rtol=1e-9, atol=1e-11, err_msg=k)
        assert (np.abs(got) <= size * (1 + 1e-9) + 1e-12).all(), k


def test_restated_clipping_agrees_with_torch():
    rng = np.random.default_rng(8)
    grads = [rng.standard_normal(s) for s in ((4, 6), (1, 9), (7, 2))]
    params = [torch.nn.Parameter(torch.zeros(g.shape, dtype=torch.float64)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = torch.from_numpy(g.copy())
    total = torch.nn.utils.clip_grad_norm_(params, 1.5)
    norms, out = ref.clip(grads, 1.5, 1, [False] * 3)
    assert abs(norms[0] - float(total)) < 1e-12
    for p, o in zip(params, out):
        np.testing.assert_allclose(o, p.grad.numpy(), rtol=1e-5)             # (torch adds 1e-6 to the norm)
    norms, out = ref.clip([grads[0], grads[2].T], 0.5, 2, [False, True])
    assert abs(norms[1] - np.sqrt((grads[0][:, 3:] ** 2).sum() + (grads[2].T[1:] ** 2).sum())) < 1e-12
    np.testing.assert_allclose(out[1][1:], grads[2].T[1:] * 0.5 / norms[1])


def test_delta_rule_refusals():
    from deepbind_amd import kangaroo_smat as ks
    Q, V, b, R = torch.zeros(9, 10), torch.zeros(9, 12), torch.zeros(9, 4), torch.zeros(2, 2, dtype=torch.int32)
    keep = torch.zeros(1, 60)
    call = lambda *a, **k: ks.deltarule(*a, **dict(dict(groups=2), **k))  # noqa: E731
    _refused("divisible by the number of key heads", call, Q, Q, V, b, R, groups=3)
    _refused("K must be (rows x key heads", call, Q, torch.zeros(9, 11), V, b, R)
    _refused("V must be (rows x heads", call, Q, Q, torch.zeros(9, 13), b, R)
    _refused("1 to 128 columns, got 129", call, torch.zeros(9, 258), torch.zeros(9, 258), V, b, R)
    _refused("Q must be a (9, 10) matrix", call, Q[:, :8], Q, V, b, R)
    _refused("Q must be torch.bfloat16", call, Q, Q.bfloat16(), V.bfloat16(), b, R)
    _refused("beta must be torch.float32", call, Q.bfloat16(), Q.bfloat16(), V.bfloat16(), b.bfloat16(), R)
    _refused("decay must be a (9, 4) matrix", call, Q, Q, V, b, R, decay=b[:, :2])
    _refused("rows, got torch.float16", call, Q.half(), Q.half(), V.half(), b, R)
    _refused("regions must be uint32", call, Q, Q, V, b, R.long())
    _refused("state must be (2, 5, 12)", call, Q, Q, V, b, R, state=torch.zeros(2, 4, 12))
    _refused("state must be torch.float32", call, Q, Q, V, b, R, state=torch.zeros(2, 5, 12).bfloat16())
    _refused("keep must be (1, 60)", call, Q, Q, V, b, R, keep=torch.zeros(1, 5, 12))
    _refused("no initial state", call, Q, Q, V, b, R, keep=keep, state=torch.zeros(2, 5, 12))
    _refused("out must be a (9, 12) matrix", call, Q, Q, V, b, R, out=torch.zeros(9, 11))
    _refused("expected a device tensor", call, Q, Q, V, b, R)
    _refused("kept are needed", ks.deltarule_bprop, Q, Q, V, b, R, None, V, groups=2)
    _refused("no decay, no gradient", ks.deltarule_bprop, Q, Q, V, b, R, keep, V, groups=2, out=(None,) * 4 + (b,))
    _refused("dO must be a (9, 12) matrix", ks.deltarule_bprop, Q, Q, V, b, R, keep, V[:8], groups=2)
    _refused("out must be (dQ", ks.deltarule_bprop, Q, Q, V, b, R, keep, V, groups=2, out=(None,) * 4)
    _refused("dbeta must be a (9, 4) matrix", ks.deltarule_bprop, Q, Q, V, b, R, keep, V, groups=2, out=(None, None, None, V, None))
    _refused("state is needed", ks.deltarule_step, Q, Q, V, b, None, groups=2)
    _refused("state must be (9, 5, 12)", ks.deltarule_step, Q, Q, V, b, torch.zeros(2, 5, 12), groups=2)
    assert ks.kept_delta(Q, V, b, groups=2).shape == (1, 60)


def test_block_norm_refusals():
    from deepbind_amd import smat as sm
    X, g = torch.zeros(4, 12), torch.ones(1, 12)
    _refused("rows, got torch.float16", sm.blocknorm, X.half())
    _refused("divisible by nchunk", sm.blocknorm, X, nchunk=5)
    _refused("must be a matrix", sm.blocknorm, X[0])
    _refused("gamma must be (1, 12)", sm.blocknorm, X, gamma=g[:, :4])
    _refused("scale must be torch.float32", sm.blocknorm, X, scale=g.double())
    _refused("R must be a (4, 12) matrix", sm.blocknorm, X, X[:3])
    _refused("gate must be torch.bfloat16", sm.blocknorm, X.bfloat16(), gate=X)
    _refused("without norm there is no gamma", sm.blocknorm, X, gamma=g, norm=False)
    _refused("without next_norm there is no next_gamma", sm.blocknorm, X, next_gamma=g, next_norm=False)
    _refused("without next_norm there is no Z", sm.blocknorm, X, next_norm=False, out=(None, X))
    _refused("expected a device tensor", sm.blocknorm, X)
    st = torch.zeros(4, 4)
    _refused("dZ is given exactly", sm.blocknorm_bprop, X, X, st, X, None)
    _refused("neither dR nor dZ", sm.blocknorm_bprop, X, X, st, None, None, next_norm=False)
    _refused("statistics of the forward call", sm.blocknorm_bprop, X, X, None, X, X)
    _refused("O of the forward call", sm.blocknorm_bprop, X, None, st, X, X)
    _refused("stats must be (4, 4)", sm.blocknorm_bprop, X, X, st[:3], X, X)
    _refused("no gamma, no gradient", sm.blocknorm_bprop, X, X, st, X, X, out=(None, None, None, g, None, None, None, None))
    _refused("out must be (dY", sm.blocknorm_bprop, X, X, st, X, X, out=(None,) * 7)


def test_clip_refusals():
    from deepbind_amd import deepity_smat as ds
    X = torch.zeros(4, 12)
    _refused("nblock must be at least 1", ds.clip_gradients, [X], 1.0, nblock=0)
    _refused("largest norm must be positive", ds.clip_gradients, [X], 0.0)
    _refused("largest norm must be positive", ds.clip_gradients, [X], float("nan"))
    _refused("no tensors", ds.clip_gradients, [], 1.0)
    _refused("as many tensors", ds.clip_gradients, [X], 1.0, out=[])
    _refused("an entry for every tensor", ds.clip_gradients, [X], 1.0, by_rows=[])
    _refused("lists of tensors", ds.clip_gradients, [None], 1.0)
    _refused("rows, got torch.float16", ds.clip_gradients, [X.half()], 1.0)
    _refused("equal blocks", ds.clip_gradients, [X], 1.0, nblock=5)
    _refused("equal blocks", ds.clip_gradients, [X], 1.0, nblock=3, by_rows=[True])
    _refused("blocks of matrices", ds.clip_gradients, [X[0]], 1.0, nblock=2)
    _refused("next to each other", ds.clip_gradients, [X.t()], 1.0)
    _refused("must be contiguous", ds.clip_gradients, [torch.zeros(3, 4, 5).transpose(0, 1)], 1.0)
    _refused("out[0] must be torch.float32", ds.clip_gradients, [X], 1.0, out=[X.double()])
    _refused("expected a device tensor", ds.clip_gradients, [X, X.double()], 1.0)
    # nor where there is nothing in them: the norms would lie on the host
    _refused("expected a device tensor", ds.clip_gradients, [torch.zeros(0)], 1.0)


def test_library_refusals_of_blocks_reach_no_device():
    from deepbind_amd import _lib
    lib = _lib.dll()
    err = lambda: lib.dbk_last_error().decode()  # noqa: E731
    one = ctypes.c_void_p(16)
    assert lib.dbk_deltarule_args_size() == ctypes.sizeof(_lib.DeltaRuleArgs)
    assert lib.dbk_deltarule(None, None, None, 0) and "null argument" in err()
    a = _lib.DeltaRuleArgs()
    at = ctypes.addressof(a)
    a.dtype, a.N, a.H, a.G, a.K, a.V, a.nregion = 3, 70, 4, 3, 129, 6, 1
    assert lib.dbk_deltarule(None, at, None, 0) and "DBK_BF16, got 3" in err()
    a.dtype = 0
    assert lib.dbk_deltarule(None, at, None, 0) and "divisible by the number of key heads" in err()
    a.G = 2
    assert lib.dbk_deltarule(None, at, None, 0) and "1 to 128 columns, got 129" in err()
    a.K = 5
    assert lib.dbk_deltarule(None, at, None, 0) and "null matrix" in err()
    a.Q = a.Kk = a.Vv = a.beta = a.decay = 16
    a.ldq = a.ldk = 10
    a.ldv, a.ldbeta = 24, 4
    assert lib.dbk_deltarule(None, at, None, 0) and "row strides" in err()
    a.lddecay = 4
    assert lib.dbk_deltarule(None, at, None, 0) and "null regions" in err()
    a.regions = 16
    assert lib.dbk_deltarule(None, at, None, 0) and "null matrix" in err()
    a.O, a.ldo, a.keep, a.state = 16, 24, 16, 16
    assert lib.dbk_deltarule(None, at, None, 0) and "no initial state" in err()
    a.state = None
    assert lib.dbk_deltarule(None, at, None, 0) and "workspace has 0 bytes" in err()
    assert lib.dbk_deltarule_bprop(None, at, None, 0) and "null matrix" in err()
    a.dO = a.dQ = a.dK = a.dV = a.dbeta = a.ddecay = 16
    assert lib.dbk_deltarule_bprop(None, at, None, 0) and "row strides" in err()
    a.lddo = a.lddv = 24
    a.lddq = a.lddk = 10
    a.lddbeta = a.ldddecay = 4
    assert lib.dbk_deltarule_bprop(None, at, None, 0) and "workspace has 0 bytes" in err()
    a.keep = None
    assert lib.dbk_deltarule_bprop(None, at, None, 0) and "kept are needed" in err()
    a.decay = None
    assert lib.dbk_deltarule_bprop(None, at, None, 0) and "no decay" in err()
    assert lib.dbk_deltarule_step(None, at) and "null matrix or state" in err()
    a.N, a.nregion, a.last, a.state = 1 << 24, 1 << 24, 16, 16
    assert lib.dbk_deltarule(None, at, one, 1 << 60) and "too many regions" in err()
    a.nregion = 1
    assert lib.dbk_deltarule_step(None, at) and "too many sequences" in err()
    a.H, a.K, a.V = 60000, 128, 16
    assert lib.dbk_deltarule(None, at, one, 1 << 60) and "too many heads" in err()
    a.H, a.K, a.V = 4, 5, 6
    # what is kept goes by the sizes alone, whatever the regions
    need = ctypes.c_size_t(0)
    kept = []
    for a.N, a.nregion in ((100000, 0), (100000, 9), (100000, 5000)):
        assert lib.dbk_deltarule_kept(at, ctypes.addressof(need)) == 0
        kept.append(need.value)
    assert kept[0] == kept[1] == kept[2] >= (100000 + 63) // 64 * 5 * 24
    a.V = 0
    assert lib.dbk_deltarule_kept(at, ctypes.addressof(need)) == 0 and need.value == 0
    a.V, a.nregion = 6, 1
    a.N = 0
    assert lib.dbk_deltarule_step(None, at) == 0 and err() == ""

    assert lib.dbk_blocknorm_args_size() == ctypes.sizeof(_lib.BlockNormArgs)
    assert lib.dbk_blocknorm(None, None) and "null argument" in err()
    b = _lib.BlockNormArgs()
    at = ctypes.addressof(b)
    b.norm = b.next = 1
    b.n, b.m, b.group = 4, 12, 5
    assert lib.dbk_blocknorm(None, at) and "divisible" in err()
    b.group = 4
    assert lib.dbk_blocknorm(None, at) and "null matrix" in err()
    b.Y, b.ldy = 16, 11
    assert lib.dbk_blocknorm(None, at) and "null matrix" in err()
    b.O = b.Z = 16
    b.ldo = b.ldz = 12
    assert lib.dbk_blocknorm(None, at) and "row strides" in err()
    b.ldy = 12
    b.next, b.next_gamma = 0, 16
    assert lib.dbk_blocknorm(None, at) and "left out" in err()
    b.next = 1
    assert lib.dbk_blocknorm_bprop(None, at, None, 0) and "null matrix" in err()
    b.dY = b.dZ = b.stats = b.dgamma = 16
    b.lddy = b.lddz = 12
    assert lib.dbk_blocknorm_bprop(None, at, None, 0) and "workspace has 0 bytes" in err()
    b.n = 0
    assert lib.dbk_blocknorm(None, at) == 0 and err() == ""

    t = (_lib.ClipTensor * 2)((16, 16, 4, 6, 6, 6, 0, 0), (16, 16, 1, 70000, 70000, 70000, 2, 0))
    where = ctypes.addressof(t)
    assert lib.dbk_clip_gradients(None, 2, where, 0, 1.0, one, None, 0) and "65535 blocks" in err()
    assert lib.dbk_clip_gradients(None, 2, where, 4, 1.0, one, None, 0) and "does not divide" in err()
    assert lib.dbk_clip_gradients(None, 2, where, 2, 1.0, None, None, 0) and "null norms" in err()
    assert lib.dbk_clip_gradients(None, 2, where, 2, -1.0, one, None, 0) and "must be positive" in err()
    assert lib.dbk_clip_gradients(None, 2, where, 2, 1.0, one, None, 0) and "workspace has 0 bytes" in err()
    t[0].ld_out = 5
    assert lib.dbk_clip_gradients(None, 2, where, 2, 1.0, one, None, 0) and "row strides" in err()
    t[0].dtype = 7
    assert lib.dbk_clip_gradients(None, 2, where, 2, 1.0, one, None, 0) and "got 7" in err()
    need = ctypes.c_size_t(5)
    assert lib.dbk_clip_gradients_workspace(0, None, 3, ctypes.addressof(need)) == 0 and need.value == 0 and err() == ""


def test_long_lists_of_tensors_that_share_memory_are_told_apart():
    from deepbind_amd._lib import Arguments, DeepbindError, check_many

    def shared(outs, ins, at=0):
        a = Arguments()
        for out, tensors in ((False, ins), (True, outs)):
            for t in tensors:
                a.rows("t", t, t.shape, t.dtype, out=out)
        for group in (a.ins, a.outs):            # (as if they lay on the current device: there is none here)
            group[:] = [(lo, hi, at, t) for lo, hi, _, t in group]
        try:
            check_many(a)
        except DeepbindError as e:
            assert ("lies on device 1" if at else "shares memory") in str(e)
            return True
        return False

    base = torch.zeros(8, 12)
    before = torch.cuda.current_device
    torch.cuda.current_device = lambda: 0
    try:
        assert not shared((base[:, :6], base[:, 6:]), ())
        assert not shared((base[4:],), (base[:4], base[:4], base[:0]))
        assert shared((base, base), ()) and shared((base[:5],), (base[4:],)) and shared((base[:, :7],), (base[:, 6:],))
        assert shared((base,), (), at=1)
    finally:
        torch.cuda.current_device = before


def test_no_error_text_is_left_to_other_tests():
    from deepbind_amd import _lib
    lib = _lib.dll()
    need = ctypes.c_size_t(0)
    assert lib.dbk_clip_gradients_workspace(0, None, 1, ctypes.addressof(need)) == 0 and lib.dbk_last_error() == b""
