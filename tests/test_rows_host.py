"""The row operators without a GPU: the plain restatement that the GPU tests compare with is held to autograd and to differences,
and calls that cannot be right are refused before anything reaches a device."""
import ctypes

import numpy as np
import pytest
import torch

from tests import rows_ref as ref


def _case(rng, N=23, D=6, G=2, S=3, gate=True):
    R = np.array([[12, 20], [0, 5], [7, 7], [5, 12]])
    f = lambda *s: rng.standard_normal(s)  # noqa: E731
    return dict(X=f(N, D), dt=f(N, D), A=-np.exp(f(S, D)), B=f(N, G * S), C=f(N, G * S), D=f(1, D), gate=f(N, D) if gate else None, bias=f(1, D)), R, f(N, D)


def _torch_scan(v, R, G, S):
    """The scan by its definition in torch, differentiable."""
    rows = torch.zeros_like(v["X"])
    out = []
    n = v["X"].shape[1]
    of = torch.arange(n) // (n // G)
    for s, e in R.tolist():
        h = torch.zeros(S, n, dtype=torch.float64)
        for t in range(s, e):
            d = torch.nn.functional.softplus(v["dt"][t] + v["bias"][0])
            h = torch.exp(d * v["A"]) * h + d * v["X"][t] * v["B"][t].view(G, S)[of].t()
            y = (v["C"][t].view(G, S)[of].t() * h).sum(0) + v["D"][0] * v["X"][t]
            if v["gate"] is not None:
                y = y * torch.nn.functional.silu(v["gate"][t])
            out.append((t, y))
    for t, y in out:
        rows = rows.index_put((torch.tensor(t),), y)
    return rows


@pytest.mark.parametrize("gate", [True, False])
def test_restated_scan_agrees_with_autograd_and_differences(gate):
    rng = np.random.default_rng(3)
    v, R, dY = _case(rng, gate=gate)
    G, S = 2, 3
    got, _ = ref.statescan(v["X"], v["dt"], v["A"], v["B"], v["C"], R, v["D"], v["gate"], v["bias"], dY=dY)
    t = {k: None if a is None else torch.from_numpy(a).requires_grad_() for k, a in v.items()}
    Y = _torch_scan(t, R, G, S)
    inside = ~np.isnan(got[0][:, 0])
    assert inside.sum() == 20
    np.testing.assert_allclose(got[0][inside], Y.detach().numpy()[inside], rtol=1e-12, atol=1e-13)
    Y.backward(torch.from_numpy(dY))
    names = ("X", "dt", "A", "B", "C", "D", "gate", "bias")
    for name, grad in zip(names, got[2:]):
        if t[name] is None:
            continue
        want = t[name].grad.numpy()
        if want.shape[0] == 23:
            assert not want[~inside].any()
            grad, want = grad[inside], want[inside]
        np.testing.assert_allclose(grad, want, rtol=1e-10, atol=1e-11, err_msg=name)
    # central differences: truncation of order step^2, rounding of order 1e-16 / step
    f = lambda: np.nansum(ref.statescan(v["X"], v["dt"], v["A"], v["B"], v["C"], R, v["D"], v["gate"], v["bias"])[0][0] * dY)  # noqa: E731
    for name, grad in zip(names, got[2:]):
        if v[name] is None:
            continue
        for i in ((1, 2), (10, 5)) if v[name].shape[0] == 23 else ((0, 1),):
            old, step = v[name][i], 1e-5
            v[name][i] = old + step
            up = f()
            v[name][i] = old - step
            down = f()
            v[name][i] = old
            assert abs((up - down) / (2 * step) - grad[i]) < 1e-7 * (1 + abs(grad[i])), name


def test_restated_norm_and_convolution_agree_with_autograd():
    rng = np.random.default_rng(4)
    X, gamma, beta, dZ = rng.standard_normal((5, 12)), rng.standard_normal((1, 12)), rng.standard_normal((1, 12)), rng.standard_normal((5, 12))
    t = [torch.from_numpy(a).requires_grad_() for a in (X, gamma, beta)]
    Z = torch.nn.functional.layer_norm(t[0].view(5, 3, 4), (4,), eps=1e-3).reshape(5, 12) * t[1] + t[2]
    Z.backward(torch.from_numpy(dZ))
    np.testing.assert_allclose(ref.layernorm(X, gamma, beta, 3, 1e-3)[0][0], Z.detach().numpy(), rtol=1e-12, atol=1e-13)
    for got, v in zip(ref.layernorm_bprop(X, gamma, 3, 1e-3, dZ)[0], t):
        np.testing.assert_allclose(got, v.grad.numpy(), rtol=1e-10, atol=1e-12)
    R = np.array([[9, 14], [0, 1], [3, 9], [14, 14]])
    for K in (1, 2, 3, 4):
        for silu in (True, False):
            X, W, b, dZ = (rng.standard_normal(s) for s in ((15, 5), (K, 5), (1, 5), (15, 5)))
            t = [torch.from_numpy(a).requires_grad_() for a in (X, W, b)]
            Z = torch.zeros(15, 5, dtype=torch.float64)
            for s, e in R.tolist():
                if e > s:
                    x = torch.nn.functional.pad(t[0][s:e].t()[None], (K - 1, 0))
                    p = torch.nn.functional.conv1d(x, t[1].t()[:, None, :], t[2][0], groups=5)[0].t()
                    Z = torch.cat([Z[:s], torch.nn.functional.silu(p) if silu else p, Z[e:]])
            Z.backward(torch.from_numpy(dZ))
            inside = np.r_[0:1, 3:14]
            (Zr, last), _ = ref.causalconv(X, W, b, R, silu)
            np.testing.assert_allclose(Zr[inside], Z.detach().numpy()[inside], rtol=1e-12, atol=1e-13)
            grads, _ = ref.causalconv_bprop(X, W, b, R, dZ, silu)
            for got, v in zip(grads, t):
                want = v.grad.numpy()
                if got.shape[0] == 15:
                    got, want = got[inside], want[inside]
                np.testing.assert_allclose(got, want, rtol=1e-10, atol=1e-12)


def _refused(text, f, *args, **kw):
    from deepbind_amd._lib import DeepbindError
    with pytest.raises(DeepbindError) as e:
        f(*args, **kw)
    assert text in str(e.value), str(e.value)


def test_layernorm_refusals():
    from deepbind_amd import smat as sm
    X, g = torch.zeros(4, 12), torch.ones(1, 12)
    _refused("rows, got torch.float16", sm.layernorm, X.half(), g, g)
    _refused("divisible by nchunk", sm.layernorm, X, g, g, nchunk=5)
    _refused("gamma must be (1, 12)", sm.layernorm, X, g[:, :4], g)
    _refused("gamma must be torch.float32", sm.layernorm, X, g.double(), g)
    _refused("beta must be torch.float64", sm.layernorm, X.double(), g.double(), g)
    _refused("next to each other", sm.layernorm, torch.zeros(12, 4).t(), g, g)
    _refused("must not overlap", sm.layernorm, torch.zeros(1, 12).expand(4, 12), g, g)
    _refused("out must be a (4, 12) matrix", sm.layernorm, X, g, g, out=torch.zeros(4, 11))
    _refused("must be a matrix", sm.layernorm, torch.zeros(12), g, g)
    _refused("expected a device tensor", sm.layernorm, X, g, g)
    _refused("statistics of the forward call", sm.layernorm_bprop, X, g, None, X)
    _refused("stats must be (2, 4)", sm.layernorm_bprop, X, g, torch.zeros(2, 3), X)
    _refused("dZ must be a (4, 12) matrix", sm.layernorm_bprop, X, g, torch.zeros(2, 4), X[:3])


def test_causalconv_refusals():
    from deepbind_amd import kangaroo_smat as ks
    X, W, b, R = torch.zeros(9, 6), torch.zeros(4, 6), torch.zeros(1, 6), torch.zeros(2, 2, dtype=torch.int32)
    _refused("1 to 4 taps, got 5", ks.causalconv, X, torch.zeros(5, 6), b, R)
    _refused("taps x channels", ks.causalconv, X, torch.zeros(4, 5), b, R)
    _refused("b must be (1, 6)", ks.causalconv, X, W, torch.zeros(6), R)
    _refused("regions must be uint32", ks.causalconv, X, W, b, R.long())
    _refused("contiguous (P x 2)", ks.causalconv, X, W, b, torch.zeros(2, 3, dtype=torch.int32))
    _refused("state must be (2, 3, 6)", ks.causalconv, X, W, b, R, state=torch.zeros(2, 4, 6))
    _refused("state must be torch.bfloat16", ks.causalconv, X.bfloat16(), W, b, R, state=torch.zeros(2, 3, 6))
    _refused("expected a device tensor", ks.causalconv, X, W, b, R)
    _refused("no gradient of it", ks.causalconv_bprop, X, W, None, R, X, out=(None, None, b))
    _refused("dZ must be torch.float32", ks.causalconv_bprop, X, W, b, R, X.double())
    _refused("state is needed", ks.causalconv_step, X, W, b, None)
    _refused("state must be (9, 3, 6)", ks.causalconv_step, X, W, b, torch.zeros(2, 3, 6))


def test_statescan_refusals():
    from deepbind_amd import kangaroo_smat as ks
    X, A, B, R = torch.zeros(9, 6), torch.zeros(4, 6), torch.zeros(9, 8), torch.zeros(2, 2, dtype=torch.int32)
    keep = torch.zeros(2, 4, 6)
    _refused("1 to 64 states per channel, got 65", ks.statescan, X, X, torch.zeros(65, 6), torch.zeros(9, 65), torch.zeros(9, 65), R)
    _refused("B must be (rows x groups", ks.statescan, X, X, A, torch.zeros(9, 7), B, R)
    _refused("divisible by the number of groups", ks.statescan, X, X, A, torch.zeros(9, 16), torch.zeros(9, 16), R)
    _refused("C must be a (9, 8) matrix", ks.statescan, X, X, A, B, torch.zeros(9, 4), R)
    _refused("dt must be a (9, 6) matrix", ks.statescan, X, X[:8], A, B, B, R)
    _refused("B must be torch.float32", ks.statescan, X.bfloat16(), X.bfloat16(), A, B.bfloat16(), B, R)
    _refused("gate must be torch.bfloat16", ks.statescan, X.bfloat16(), X.bfloat16(), A, B, B, R, gate=X)
    _refused("D must be (1, 6)", ks.statescan, X, X, A, B, B, R, D=torch.zeros(6))
    _refused("state must be (2, 4, 6)", ks.statescan, X, X, A, B, B, R, state=torch.zeros(4, 6))
    _refused("no initial state", ks.statescan, X, X, A, B, B, R, state=torch.zeros(2, 4, 6), keep=keep)
    _refused("keep must be (2, 4, 6)", ks.statescan, X, X, A, B, B, R, keep=torch.zeros(1, 4, 6))
    _refused("expected a device tensor", ks.statescan, X, X, A, B, B, R)
    _refused("kept are needed", ks.statescan_bprop, X, X, A, B, B, R, None, X)
    _refused("no gate, no gradient", ks.statescan_bprop, X, X, A, B, B, R, keep, X, out=(None,) * 6 + (X, None))
    _refused("state is needed", ks.statescan_step, X, X, A, B, B, None)


def test_library_refusals_reach_no_device():
    from deepbind_amd import _lib
    lib = _lib.dll()
    one = ctypes.c_void_p(16)
    err = lambda: lib.dbk_last_error().decode()  # noqa: E731
    assert lib.dbk_layernorm(None, 3, one, 8, None, None, 4, 8, 8, 1e-5, one, 8, None) and "DBK_BF16, got 3" in err()
    assert lib.dbk_layernorm(None, 0, one, 8, None, None, 4, 8, 3, 1e-5, one, 8, None) and "divisible" in err()
    assert lib.dbk_layernorm(None, 0, one, 7, None, None, 4, 8, 8, 1e-5, one, 8, None) and "row strides" in err()
    assert lib.dbk_layernorm(None, 0, None, 8, None, None, 4, 8, 8, 1e-5, one, 8, None) and "null" in err()
    assert lib.dbk_layernorm_bprop(None, 0, one, 8, one, one, one, 8, 4, 8, 8, one, 8, one, one, None, 0) and "workspace has 0 bytes" in err()
    assert lib.dbk_layernorm(None, 0, None, 8, None, None, 0, 8, 8, 1e-5, None, 8, None) == 0 and err() == ""
    assert lib.dbk_causalconv(None, 0, one, 8, one, None, 5, 4, 8, one, 1, 1, None, one, 8, None, None, 0) and "1 to 4 taps" in err()
    assert lib.dbk_causalconv(None, 0, one, 8, one, None, 4, 100000, 8, one, 1, 1, None, one, 8, None, None, 0) and "workspace has 0 bytes" in err()
    assert lib.dbk_causalconv(None, 0, one, 8, one, None, 4, 4, 8, None, 1, 1, None, one, 8, None, None, 0) and "null regions" in err()
    assert lib.dbk_causalconv_bprop(None, 0, one, 8, one, None, 4, 4, 8, one, 1, 1, one, 8, one, 8, one, None, one, 8) and "workspace has 8 bytes" in err()
    assert lib.dbk_causalconv_step(None, 0, one, 8, one, None, 4, 4, 8, 1, None, one, one, 8) and "null state" in err()
    assert lib.dbk_statescan_args_size() == ctypes.sizeof(_lib.StateScanArgs)
    a = _lib.StateScanArgs()
    at = ctypes.addressof(a)
    assert lib.dbk_statescan(None, None, None, 0) and "null argument block" in err()
    a.N, a.D, a.S, a.G, a.nregion = 10, 8, 65, 1, 1
    assert lib.dbk_statescan(None, at, None, 0) and "1 to 64 states" in err()
    a.S, a.G = 4, 3
    assert lib.dbk_statescan(None, at, None, 0) and "divisible by the number of groups" in err()
    a.G = 2
    assert lib.dbk_statescan(None, at, None, 0) and "null weights" in err()
    a.A = a.X = a.dt = a.B = a.C = 16
    a.ldx = a.lddt = a.ldb = 8
    assert lib.dbk_statescan(None, at, None, 0) and "row strides" in err()
    a.ldc = 8
    assert lib.dbk_statescan(None, at, None, 0) and "null regions" in err()
    a.regions, a.Y, a.ldy, a.keep, a.state = 16, 16, 8, 16, 16
    assert lib.dbk_statescan(None, at, None, 0) and "no initial state" in err()
    a.state = None
    assert lib.dbk_statescan_bprop(None, at, None, 0) and "null gradient" in err()
    a.dA = a.dY = a.dX = a.ddt = a.dB = a.dC = 16
    a.lddy = a.lddx = a.ldddt = a.lddb = a.lddc = 8
    assert lib.dbk_statescan_bprop(None, at, None, 0) and "workspace has 0 bytes" in err()
    assert lib.dbk_statescan_step(None, at) and "null matrix or state" in err()
    a.N = 0
    assert lib.dbk_statescan_step(None, at) == 0 and err() == ""


def test_outputs_that_share_memory_are_told_apart():
    from deepbind_amd._lib import Arguments, DeepbindError

    def shared(outs, ins):
        a = Arguments()
        for out, tensors in ((False, ins), (True, outs)):
            for t in tensors:
                a.rows("t", t, t.shape, t.dtype, out=out)
        for group in (a.ins, a.outs):            # (as if they lay on the current device: there is none here)
            group[:] = [(lo, hi, 0, t) for lo, hi, _, t in group]
        try:
            a.check()
        except DeepbindError as e:
            assert "shares memory" in str(e)
            return True
        return False

    base = torch.zeros(8, 12)
    before = torch.cuda.current_device
    torch.cuda.current_device = lambda: 0
    try:
        assert not shared((base[:, :6],), (base[:, 6:],))
        assert not shared((base[:, 6:],), (base[:, :6], base[:, 2:4]))
        assert not shared((base[4:],), (base[:4],))
        assert not shared((), (base, base))
        assert not shared((base,), (base[:0],))
        for outs, ins in (((base,), (base,)), ((base[:, :7],), (base[:, 6:],)), ((base[1:],), (base[:4],)), ((base[:, :3], base[:, 2:5]), ()),
                          ((base[2:4, :3],), (base[:, 1:2],))):
            assert shared(outs, ins)
    finally:
        torch.cuda.current_device = before


def test_calls_beyond_one_launch_are_refused():
    """A launch holds fewer than 2^32 threads: 2^24 workgroups of 256 are one too many, and would run none of them without a word."""
    from deepbind_amd import _lib
    lib = _lib.dll()
    one = ctypes.c_void_p(16)
    err = lambda: lib.dbk_last_error().decode()  # noqa: E731
    n = 1 << 24
    assert lib.dbk_causalconv(None, 0, one, 1, one, None, 2, n, 1, one, n, 1, None, one, 1, None, one, 1 << 40) and "map too large" in err()
    assert lib.dbk_causalconv_bprop(None, 0, one, 1, one, None, 2, n, 1, one, n, 1, one, 1, one, 1, one, None, one, 1 << 40) and "map too large" in err()
    assert lib.dbk_causalconv(None, 0, one, 1, one, None, 2, (1 << 32) - 3, 1, one, 1, 1, None, one, 1, None, one, 1 << 40) and "map too large" in err()
    assert lib.dbk_causalconv_step(None, 0, one, 1 << 12, one, None, 2, 1 << 22, 1 << 12, 1, one, one, one, 1 << 12) and "too many sequences" in err()
    a = _lib.StateScanArgs()
    at = ctypes.addressof(a)
    a.N, a.D, a.S, a.G, a.nregion = n, 1, 1, 1, n
    a.A = a.X = a.dt = a.B = a.C = a.regions = a.Y = a.dA = a.dY = a.dX = a.ddt = a.dB = a.dC = a.keep = 16
    a.ldx = a.lddt = a.ldb = a.ldc = a.ldy = a.lddy = a.lddx = a.ldddt = a.lddb = a.lddc = 1
    assert lib.dbk_statescan(None, at, one, 1 << 40) and "map too large" in err()
    assert lib.dbk_statescan_bprop(None, at, one, 1 << 40) and "map too large" in err()
    a.keep, a.state, a.last = None, 16, 16
    assert lib.dbk_statescan_step(None, at) and "too many sequences" in err()
    assert lib.dbk_layernorm_bprop(None, 0, one, 1 << 27, one, one, one, 1 << 27, 1, 1 << 27, 1 << 27, one, 1 << 27, one, one, one, 1 << 40) and "too wide" in err()


def test_backward_scans_of_many_wide_groups_are_taken():
    """A call within the limits named for regions and channels is not refused for what its groups' gradients come to: it gets as far as its workspace."""
    from deepbind_amd import _lib
    lib = _lib.dll()
    a = _lib.StateScanArgs()
    at = ctypes.addressof(a)
    a.A = a.X = a.dt = a.B = a.C = a.regions = a.Y = a.dA = a.dY = a.dX = a.ddt = a.dB = a.dC = a.keep = 16
    for dtype, N, D, S, G in ((_lib.DBK_BF16, 10 ** 6, 8192, 16, 64), (_lib.DBK_BF16, 10 ** 6, 2080, 64, 32), (_lib.DBK_F32, 520, 66560, 64, 1024)):
        a.dtype, a.N, a.D, a.S, a.G, a.nregion = dtype, N, D, S, G, 5
        a.ldx = a.lddt = a.ldy = a.lddy = a.lddx = a.ldddt = D
        a.ldb = a.ldc = a.lddb = a.lddc = G * S
        assert lib.dbk_statescan_bprop(None, at, None, 0)
        assert "workspace has 0 bytes" in lib.dbk_last_error().decode()


def test_one_row_without_a_row_stride_shares_memory_with_itself():
    """A matrix of one row is taken with any row stride, none among them."""
    from deepbind_amd._lib import Arguments, DeepbindError
    base = torch.zeros(12)
    for a, b, same in ((base.as_strided((1, 6), (0, 1)), base.as_strided((1, 6), (0, 1)), True), (base.as_strided((1, 6), (0, 1)), base.as_strided((1, 6), (0, 1), 4), True),
                       (base.as_strided((1, 6), (2, 1)), base.as_strided((1, 6), (2, 1), 2), True), (base.as_strided((1, 6), (0, 1)), base.as_strided((1, 6), (0, 1), 6), False)):
        args = Arguments()
        args.rows("a", a, a.shape, a.dtype)
        args.rows("b", b, b.shape, b.dtype, out=True)
        for group in (args.ins, args.outs):      # (as if they lay on the current device: there is none here)
            group[:] = [(lo, hi, 0, t) for lo, hi, _, t in group]
        before = torch.cuda.current_device
        torch.cuda.current_device = lambda: 0
        try:
            if same:
                with pytest.raises(DeepbindError, match="shares memory"):
                    args.check()
            else:
                args.check()
        finally:
            torch.cuda.current_device = before


def test_refusals_of_other_tests_leave_no_error_text():
    from deepbind_amd import _lib
    assert _lib.dll().dbk_last_error() == b""
    with pytest.raises(_lib.DeepbindError):
        _lib.call("dbk_layernorm", None, 3, None, 0, None, None, 0, 8, 8, 1e-5, None, 8, None)


def test_nor_does_the_one_before():
    from deepbind_amd import _lib
    assert _lib.dll().dbk_last_error() == b""
