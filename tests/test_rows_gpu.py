"""Layer norm, causal convolution and state scan on the GPU against their plain restatement in 64 bits.

Tolerances: a result is allowed k u size + r |value| + tiny, with u the unit roundoff of the arithmetic (float32 2^-24, float64 2^-53), r that of
the stored type where it is narrower (bfloat16 2^-8), `size` the sum of its terms' absolute values (rows_ref) and k the most
roundings that a term can go through: the number of terms it is summed with, plus those of its own formation."""
import numpy as np
import pytest
import torch

from tests import rows_ref as ref
from tests.gpu_util import host

pytestmark = pytest.mark.gpu

TYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16}
U = {"float32": 2.0 ** -24, "float64": 2.0 ** -53, "bfloat16": 2.0 ** -24}
STORED = {"float32": 2.0 ** -24, "float64": 2.0 ** -53, "bfloat16": 2.0 ** -8}
SENTINEL = 7.0


def wide(kind):
    return torch.float64 if kind == "float64" else torch.float32


def put(a, dtype):
    """On the device in that type, and what it then holds, in 64 bits."""
    t = torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()
    return t, t.double().cpu().numpy()


def check(got, want, size, k, kind, what, rows=None, stored=True):
    got = host(got.double())
    if rows is not None:
        out = np.ones(got.shape[0], bool)
        out[rows] = False
        assert (got[out] == SENTINEL).all(), "%s: rows in no region were written" % what
        got, want, size = got[rows], want[rows], size[rows]
    assert got.shape == want.shape, what
    bound = k * U[kind] * size + (STORED[kind] if stored else U[kind]) * np.abs(want) + 1e-35
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), "%s: %d of %d values off, worst %.3g of the bound" % (what, bad.sum(), bad.size, np.nanmax(np.abs(got - want) / bound))


def inside(R, N):
    return np.concatenate([np.arange(s, e) for s, e in ref.rows_of(R, N)] or [[]]).astype(int)


def regions(t):
    return torch.from_numpy(np.asarray(t, dtype=np.int64).astype(np.uint32)).cuda()


def sliced(a, dtype, pad):
    """The matrix as a block of columns of a wider one."""
    t, v = put(a, dtype)
    if not pad:
        return t, v
    big = torch.full((a.shape[0], a.shape[1] + 2 * pad + 1), float("nan"), dtype=dtype, device="cuda")
    big[:, pad:pad + a.shape[1]] = t
    return big[:, pad:pad + a.shape[1]], v


# ------------------------------------------------------------------------------------------------ layer norm
NORM = [(1, 1, 1, 0), (3, 1, 7, 0), (5, 3, 16, 3), (64, 1, 16, 0), (7, 2, 33, 1), (33, 1, 257, 0), (9, 1, 1440, 0), (130, 24, 16, 0), (67, 5, 100, 5), (3, 1, 4100, 0),
        (2, 2, 20001, 3), (5000, 1, 5, 0), (700, 90, 3, 0), (600, 1, 1024, 0)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,nchunk,w,pad", NORM)
def test_layernorm_and_its_gradient(kind, n, nchunk, w, pad):
    from deepbind_amd import smat as sm
    rng = np.random.default_rng([n, nchunk, w])
    m = n and nchunk * w
    X, x = sliced(rng.standard_normal((n, m)) * 2 + rng.standard_normal((n, 1)), TYPES[kind], pad)
    dZ, dz = sliced(rng.standard_normal((n, m)), TYPES[kind], pad and pad + 1)
    g, gv = put(1 + 0.3 * rng.standard_normal((1, m)), wide(kind))
    b, bv = put(0.3 * rng.standard_normal((1, m)), wide(kind))
    eps = 1e-3
    (Zr, mean, r), (Zs, ms, rs) = ref.layernorm(x, gv, bv, nchunk, eps)
    Z, stats = sm.layernorm(X, g, b, nchunk=nchunk, eps=eps, want_stats=True)
    k = 16 + w / 16                              # the sums over a chunk, and the dozen roundings of one value
    check(Z, Zr, Zs, k, kind, "Z")
    check(stats[0], mean, ms, k, kind, "mean", stored=False)
    check(stats[1], r, rs, 2 * k, kind, "deviation", stored=False)
    (dXr, dgr, dbr), (dXs, dgs, dbs) = ref.layernorm_bprop(x, gv, nchunk, eps, dz)
    dX, dg, db = sm.layernorm_bprop(X, g, stats, dZ, nchunk=nchunk)
    check(dX, dXr, dXs, 4 * k, kind, "dX")
    check(dg, dgr, dgs, k + n, kind, "dgamma", stored=False)
    check(db, dbr, dbs, n, kind, "dbeta", stored=False)
    # into given tensors, and without weights
    out = torch.full((n, m + 2), SENTINEL, dtype=TYPES[kind], device="cuda")
    Z2, none = sm.layernorm(X, g, b, nchunk=nchunk, eps=eps, out=out[:, 1:-1])
    assert none is None and torch.equal(Z2, Z) and bool((out[:, 0] == SENTINEL).all()) and bool((out[:, -1] == SENTINEL).all())
    again = sm.layernorm_bprop(X, g, stats, dZ, nchunk=nchunk, out=(torch.empty_like(dX), torch.empty_like(dg), None))
    assert all(torch.equal(p, q) for p, q in zip(again, (dX, dg, db)))
    Z3, _ = sm.layernorm(X, nchunk=nchunk, eps=eps)
    one, zero = np.ones((1, m)), np.zeros((1, m))
    (Zr, _, _), (Zs, _, _) = ref.layernorm(x, one, zero, nchunk, eps)
    check(Z3, Zr, Zs, k, kind, "Z without weights")
    dX3, n1, n2 = sm.layernorm_bprop(X, None, stats, dZ, nchunk=nchunk)
    (dXr, _, _), (dXs, _, _) = ref.layernorm_bprop(x, one, nchunk, eps, dz)
    check(dX3, dXr, dXs, 4 * k, kind, "dX without weights")
    assert n1 is None and n2 is None


def test_layernorm_of_no_rows():
    from deepbind_amd import smat as sm
    X, g = torch.zeros(0, 12, device="cuda"), torch.ones(1, 12, device="cuda")
    Z, stats = sm.layernorm(X, g, g, nchunk=3, want_stats=True)
    dX, dg, db = sm.layernorm_bprop(X, g, stats, X, nchunk=3, out=(None, g * 5, g * 5))
    assert Z.shape == (0, 12) and dX.shape == (0, 12) and not dg.any() and not db.any()


def test_layernorm_keeps_a_bad_row_to_itself():
    from deepbind_amd import smat as sm
    X = torch.randn(50, 48, device="cuda")
    want, _ = sm.layernorm(X, nchunk=3)
    X[7, 20], X[30, 0] = float("nan"), float("inf")
    got, _ = sm.layernorm(X, nchunk=3)
    bad = torch.zeros(50, 48, dtype=torch.bool, device="cuda")
    bad[7, 16:32] = bad[30, :16] = True
    assert torch.equal(got[~bad], want[~bad]) and bool(got[bad].isnan().any())


# ------------------------------------------------------------------------------------------------ causal convolution
TABLES = {
    "one": ([[0, 9]], 9),
    "ragged": ([[30, 61], [0, 1], [1, 3], [70, 70], [3, 30], [61, 64]], 75),
    "outside": ([[5, 9], [9, 4], [20, 90], [200, 300], [12, 20]], 40),             # a range that ends early, one cut at the map's end, one behind it
    "reads": ([[i * 37, i * 37 + 37 - i % 5] for i in range(300)], 300 * 37 + 5),
    "long": ([[2000, 9001], [3, 1300], [1300, 1301]], 9010),
    "none": ([], 6),
}


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("table,D,K,silu,pad", [("one", 1, 4, True, 0), ("ragged", 5, 4, True, 0), ("ragged", 16, 1, True, 2), ("outside", 33, 3, False, 0), ("reads", 24, 4, True, 0),
                                                ("reads", 257, 2, True, 1), ("long", 12, 4, True, 0), ("long", 300, 4, False, 0), ("none", 8, 4, True, 0), ("long", 2, 3, True, 0)])
def test_causalconv_and_its_gradient(kind, table, D, K, silu, pad):
    from deepbind_amd import kangaroo_smat as ks
    R, N = TABLES[table]
    rng = np.random.default_rng([N, D, K])
    X, x = sliced(rng.standard_normal((N, D)), TYPES[kind], pad)
    dZ, dz = sliced(rng.standard_normal((N, D)), TYPES[kind], pad)
    W, w = put(rng.standard_normal((K, D)), wide(kind))
    b, bv = put(rng.standard_normal((1, D)), wide(kind))
    state, s = put(rng.standard_normal((len(R), K - 1, D)), TYPES[kind])
    T, rows = regions(np.asarray(R).reshape(-1, 2)), inside(R, N)
    hidden = torch.ones(N, dtype=torch.bool, device="cuda")
    hidden[rows] = False
    X[hidden], dZ[hidden] = float("nan"), float("nan")            # what lies in no region is not looked at
    x[hidden.cpu().numpy()] = 0
    dz[hidden.cpu().numpy()] = 0
    k = K + 12                                   # the taps, the bias, and the roundings of the sigmoid's exponential, reciprocal and product
    new = lambda *shape, dtype=TYPES[kind]: torch.full(shape, SENTINEL, dtype=dtype, device="cuda")  # noqa: E731
    for start in (None, state):
        Z, last = ks.causalconv(X, W, b, T, silu=silu, state=start, want_state=True, out=new(N, D))
        (Zr, lr), (Zs, _) = ref.causalconv(x, w, bv, R, silu, None if start is None else s)
        check(Z, Zr, Zs, k, kind, "Z", rows)
        assert np.array_equal(host(last.double()), lr), "last"
    Z0, none = ks.causalconv(X, W, b, T, silu=silu, state=state)
    assert none is None and not Z0[hidden].any() and torch.equal(Z0[rows], Z[rows])
    out = (new(N, D), new(K, D, dtype=wide(kind)), new(1, D, dtype=wide(kind)))
    got = ks.causalconv_bprop(X, W, b, T, dZ, silu=silu, out=out)
    assert all(p is q for p, q in zip(got, out))
    (dXr, dWr, dbr), (dXs, dWs, dbs) = ref.causalconv_bprop(x, w, bv, R, dz, silu)
    check(got[0], dXr, dXs, 2 * k, kind, "dX", rows)
    check(got[1], dWr, dWs, k + len(rows), kind, "dW", stored=False)
    check(got[2], dbr, dbs, k + len(rows), kind, "db", stored=False)
    again = ks.causalconv_bprop(X, W, b, T, dZ, silu=silu)
    assert torch.equal(again[0][rows], got[0][rows]) and not again[0][hidden].any() and torch.equal(again[1], got[1]) and torch.equal(again[2], got[2])
    # without a bias
    Z1, _ = ks.causalconv(X, W, None, T, silu=silu, out=new(N, D))
    (Zr, _), (Zs, _) = ref.causalconv(x, w, 0 * bv, R, silu)
    check(Z1, Zr, Zs, k, kind, "Z without bias", rows)
    assert ks.causalconv_bprop(X, W, None, T, dZ, silu=silu)[2] is None


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("K", [1, 2, 3, 4])
def test_causalconv_steps_are_the_convolution_row_by_row(kind, K):
    from deepbind_amd import kangaroo_smat as ks
    n, L, D = 5, 11, 19
    rng = np.random.default_rng(K)
    X, _ = put(rng.standard_normal((n * L, D)), TYPES[kind])
    W, b = put(rng.standard_normal((K, D)), wide(kind))[0], put(rng.standard_normal((1, D)), wide(kind))[0]
    T = regions([[i * L, (i + 1) * L] for i in range(n)])
    Z, last = ks.causalconv(X, W, b, T, want_state=True)
    state = torch.zeros(n, K - 1, D, dtype=TYPES[kind], device="cuda")
    for t in range(L):
        kept = state.clone()
        moved = torch.empty_like(state)
        rows = X.view(n, L, D)[:, t]             # (every L-th row of the map: a row stride of L * D)
        z = ks.causalconv_step(rows, W, b, state, into=moved)
        assert torch.equal(state, kept)
        assert torch.equal(ks.causalconv_step(rows, W, b, state), z) and torch.equal(state, moved)
        assert torch.equal(z, Z.view(n, L, D)[:, t])         # the same operations on the same numbers
    assert torch.equal(state, last)


# ------------------------------------------------------------------------------------------------ state scan
SCAN = [("one", 1, 1, 1, 0), ("ragged", 6, 2, 3, 0), ("ragged", 70, 1, 16, 3), ("outside", 48, 3, 16, 0), ("outside", 40, 2, 5, 1), ("reads", 64, 1, 4, 0),
        ("ragged", 130, 2, 17, 0), ("long", 40, 2, 16, 0), ("long", 65, 1, 7, 2), ("none", 8, 1, 4, 0), ("ragged", 8, 8, 2, 0), ("outside", 300, 1, 64, 0)]


def scan_inputs(kind, table, D, G, S, pad, seed=0):
    R, N = TABLES[table]
    rng = np.random.default_rng([N, D, G, S, seed])
    f = lambda *s: rng.standard_normal(s)  # noqa: E731
    rows = inside(R, N)
    out = np.ones(N, bool)
    out[rows] = False
    t, v = {}, {}
    for name, shape, dtype in (("X", (N, D), TYPES[kind]), ("dt", (N, D), TYPES[kind]), ("gate", (N, D), TYPES[kind]), ("dY", (N, D), TYPES[kind]),
                               ("B", (N, G * S), wide(kind)), ("C", (N, G * S), wide(kind))):
        t[name], v[name] = sliced(f(*shape), dtype, pad)
        t[name][torch.from_numpy(out).cuda()] = float("nan")
        v[name][out] = 0
    t["A"], v["A"] = put(-np.exp(1.5 * f(S, D)), wide(kind))
    t["D"], v["D"] = put(f(1, D), wide(kind))
    t["bias"], v["bias"] = put(f(1, D) - 2, wide(kind))
    t["state"], v["state"] = put(f(len(R), S, D), wide(kind))
    return t, v, R, N, rows


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("table,D,G,S,pad", SCAN)
def test_statescan_and_its_gradient(kind, table, D, G, S, pad):
    from deepbind_amd import kangaroo_smat as ks
    t, v, R, N, rows = scan_inputs(kind, table, D, G, S, pad)
    T = regions(np.asarray(R).reshape(-1, 2))
    longest = max([e - s for s, e in ref.rows_of(R, N)] + [0])
    k = 16 * (longest + 8) + S                   # at most 16 roundings per row on the way of a term (step, decay, input, sum), the sum over states
    new = lambda *shape, dtype=TYPES[kind]: torch.full(shape, SENTINEL, dtype=dtype, device="cuda")  # noqa: E731
    base = [t[n] for n in ("X", "dt", "A", "B", "C")]
    val = [v[n] for n in ("X", "dt", "A", "B", "C")]
    for gate, soft, start in ((True, True, True), (False, True, False)) + (((True, False, False),) if table == "ragged" else ()):
        if not soft:                             # steps as they are: positive ones, or states grow without bound
            t["dt"].abs_()
            np.abs(v["dt"], out=v["dt"])         # (in place, as on the device: both lists of arguments hold these)
        bias = "bias" if soft else None
        kw = dict(D=t["D"], gate=t["gate"] if gate else None, dt_bias=t["bias"] if soft else None, softplus=soft)
        rv = (R, v["D"], v["gate"] if gate else None, v["bias"] if soft else np.zeros((1, D)), soft)
        Y, last = ks.statescan(*base, T, state=t["state"] if start else None, want_state=True, out=new(N, D), **kw)
        (Yr, lr), (Ys, ls) = ref.statescan(*val, *rv, state=v["state"] if start else None)
        check(Y, Yr, Ys, k, kind, "Y", rows)
        check(last, lr, ls, k, kind, "last", stored=False)
        keep = ks.kept_states(t["X"], t["A"])
        Y0, none = ks.statescan(*base, T, keep=keep, **kw)
        (Yr, _, *grads), (Ys, _, *sizes) = ref.statescan(*val, *rv, dY=v["dY"])
        out = np.ones(N, bool)
        out[rows] = False
        assert none is None and not Y0[torch.from_numpy(out).cuda()].any()
        check(Y0[rows], Yr[rows], Ys[rows], k, kind, "Y from zeros")
        made = lambda name, like: None if like is None else new(*like.shape, dtype=like.dtype)  # noqa: E731
        outs = tuple(made(n, x) for n, x in zip("xtABCDgb", (t["X"], t["dt"], t["A"], t["B"], t["C"], t["D"], kw["gate"], kw["dt_bias"])))
        got = ks.statescan_bprop(*base, T, keep, t["dY"], out=outs, **kw)
        assert all(p is q for p, q in zip(got, outs))
        for name, g, want, size in zip(("dX", "ddt", "dA", "dB", "dC", "dD", "dgate", "ddt_bias"), got, grads, sizes):
            if g is None:
                continue
            per_row = name in ("dX", "ddt", "dB", "dC", "dgate")
            # both ways along the rows, the sum over states, over a group's channels, over all rows
            check(g, want, size, 2 * k + D // G + (0 if per_row else len(rows)), kind, name, rows if per_row else None, stored=name in ("dX", "ddt", "dgate"))
        again = ks.statescan_bprop(*base, T, keep, t["dY"], **kw)
        for name, g, a in zip(("dX", "ddt", "dA", "dB", "dC", "dD", "dgate", "ddt_bias"), got, again):
            if g is not None:
                assert torch.equal(g[rows], a[rows]) if g.shape[0] == N and name not in ("dA", "dD", "ddt_bias") else torch.equal(g, a), name
        assert bias is None or got[7] is not None


@pytest.mark.parametrize("kind", list(TYPES))
def test_statescan_goes_on_from_its_state(kind):
    """Pieces of sequences, then single rows, against the whole: the states carry everything over."""
    from deepbind_amd import kangaroo_smat as ks
    n, L, D, G, S = 3, 700, 24, 2, 9
    rng = np.random.default_rng(5)
    f = lambda *s, dtype: put(rng.standard_normal(s), dtype)[0]  # noqa: E731
    X, dt, gate = (f(n * L, D, dtype=TYPES[kind]) for _ in range(3))
    B, C = (f(n * L, G * S, dtype=wide(kind)) for _ in range(2))
    A = -torch.exp(f(S, D, dtype=wide(kind)))
    kw = dict(D=f(1, D, dtype=wide(kind)), dt_bias=f(1, D, dtype=wide(kind)))
    whole, last = ks.statescan(X, dt, A, B, C, regions([[i * L, (i + 1) * L] for i in range(n)]), gate=gate, want_state=True, **kw)
    state, Y = None, torch.zeros_like(whole)
    for a, b in ((0, 1), (1, 340), (340, 340), (340, 690)):
        _, state = ks.statescan(X, dt, A, B, C, regions([[i * L + a, i * L + b] for i in range(n)]), gate=gate, state=state, want_state=True, out=Y, **kw)
    for t in range(690, L):
        at = lambda m: m.view(n, L, -1)[:, t]  # noqa: E731
        kept, moved = state.clone(), torch.empty_like(state)
        y = ks.statescan_step(at(X), at(dt), A, at(B), at(C), state, gate=at(gate), into=moved, **kw)
        assert torch.equal(kept, state)
        Y.view(n, L, D)[:, t] = ks.statescan_step(at(X), at(dt), A, at(B), at(C), state, gate=at(gate), **kw)
        assert torch.equal(moved, state) and torch.equal(Y.view(n, L, D)[:, t], y)
    # both ways round 16 times per row at most; the states' size is a few units here, the decays forget in a few rows
    scale = 64 * 16 * U[kind]
    assert float((state - last).abs().max()) <= scale * float(last.abs().max())
    tol = (2 * STORED[kind] + scale) * float(whole.double().abs().max())
    assert float((Y.double() - whole.double()).abs().max()) <= tol


def test_statescan_with_infinite_and_undefined_values_stays_in_its_region():
    from deepbind_amd import kangaroo_smat as ks
    t, v, R, N, rows = scan_inputs("float32", "ragged", 70, 1, 16, 0)
    T = regions(R)
    base = [t[n] for n in ("X", "dt", "A", "B", "C")]
    keep = ks.kept_states(t["X"], t["A"])
    Y, _ = ks.statescan(*base, T, keep=keep)
    g = ks.statescan_bprop(*base, T, keep, t["dY"])
    t["X"][10, 3], t["dt"][12, 66] = float("inf"), float("nan")               # rows of region 4: rows 3 to 29
    Y2, _ = ks.statescan(*base, T, keep=keep)
    g2 = ks.statescan_bprop(*base, T, keep, t["dY"])
    other = [i for i in rows if not 3 <= i < 30]
    assert torch.equal(Y[other], Y2[other])
    for name in (0, 1, 3, 4):
        assert torch.equal(g[name][other], g2[name][other])
    assert torch.equal(Y[3:10], Y2[3:10]) and not bool(torch.isfinite(Y2[10:30, 3]).all()) and torch.equal(Y[3:30, 4:66], Y2[3:30, 4:66])


# ------------------------------------------------------------------------------------------------ together, as they are used
def test_layers_between_the_motif_scan_and_the_pooling():
    """Motif scan -> layer norm -> convolution -> state scan -> pooling per sequence, and the gradient all the way back, in double
    precision against autograd of the same chain in plain torch."""
    from deepbind_amd import data, kangaroo_smat as ks, smat as sm
    rng = np.random.default_rng(9)
    seqs = ["".join("ACGTN"[i] for i in rng.integers(0, 5, size=n)) for n in (1, 40, 17, 133, 64)]
    m, F, S, K = 5, 12, 4, 3
    Xc, R = data.pack_sequences(seqs, m - 1)
    codes, T = torch.from_numpy(Xc.ravel()).cuda(), torch.from_numpy(R.astype(np.int64).astype(np.int32)).cuda().view(torch.uint32)
    N = codes.numel()
    p = {n: torch.from_numpy(rng.standard_normal(s) * 0.5) for n, s in (("W", (4 * m, F)), ("gamma", (1, F)), ("beta", (1, F)), ("K", (K, F)), ("b", (1, F)), ("A", (S, F)),
                                                                       ("D", (1, F)), ("bias", (1, F)), ("B", (N, 2 * S)), ("C", (N, 2 * S)), ("gate", (N, F)), ("dt", (N, F)))}
    p["A"] = -p["A"].abs()
    d = {n: v.cuda() for n, v in p.items()}
    # the package
    Z = torch.zeros(N, F, dtype=torch.float64, device="cuda")
    ks.corr1ord(d["W"], codes, Z, 4)
    H, stats = sm.layernorm(Z, d["gamma"], d["beta"], nchunk=3, want_stats=True)
    V, _ = ks.causalconv(H, d["K"], d["b"], T)
    keep = ks.kept_states(V, d["A"])
    kw = dict(D=d["D"], gate=d["gate"], dt_bias=d["bias"])
    Y, _ = ks.statescan(V, d["dt"], d["A"], d["B"], d["C"], T, keep=keep, **kw)
    pooled, _ = ks.poolrgn(Y, T, "avg")
    up = torch.from_numpy(rng.standard_normal(tuple(pooled.shape))).cuda()
    dY = torch.zeros_like(Y)
    ks.poolrgn_bprop(dY, T, up, None, "avg")
    dV, ddt, dA, dB, dC, dD, dgate, dbias = ks.statescan_bprop(V, d["dt"], d["A"], d["B"], d["C"], T, keep, dY, **kw)
    dH, dK, db = ks.causalconv_bprop(H, d["K"], d["b"], T, dV)
    dZ, dgamma, dbeta = sm.layernorm_bprop(Z, d["gamma"], stats, dH, nchunk=3)
    dW = torch.zeros_like(d["W"])
    ks.corr1ord_bprop_W(dW, codes, dZ, 4)
    # plain torch
    q = {n: v.clone().requires_grad_() for n, v in p.items()}
    c = Xc.ravel()
    onehot = torch.zeros(N + m, 4, dtype=torch.float64)
    for i, k in enumerate(c):
        onehot[i] = torch.eye(4, dtype=torch.float64)[k] if k < 4 else 0.25
    z = sum(onehot[j:j + N] @ q["W"][4 * j:4 * j + 4] for j in range(m))
    z = torch.cat([z[:N - m + 1], torch.zeros(m - 1, F, dtype=torch.float64)])
    h = torch.nn.functional.layer_norm(z.view(N, 3, 4), (4,), eps=1e-5).reshape(N, F) * q["gamma"] + q["beta"]
    pool = []
    of = torch.arange(F) // (F // 2)
    for s, e in R.astype(int).tolist():
        x = torch.nn.functional.pad(h[s:e].t()[None], (K - 1, 0))
        x = torch.nn.functional.silu(torch.nn.functional.conv1d(x, q["K"].t()[:, None, :], q["b"][0], groups=F)[0].t())
        st, ys = torch.zeros(S, F, dtype=torch.float64), []
        for t in range(s, e):
            dd = torch.nn.functional.softplus(q["dt"][t] + q["bias"][0])
            st = torch.exp(dd * q["A"]) * st + dd * x[t - s] * q["B"][t].view(2, S)[of].t()
            ys.append(((q["C"][t].view(2, S)[of].t() * st).sum(0) + q["D"][0] * x[t - s]) * torch.nn.functional.silu(q["gate"][t]))
        pool.append(torch.stack(ys).mean(0))
    pool = torch.stack(pool)
    pool.backward(up.cpu())
    # (double precision end to end, a few hundred terms per value: 1e-10 of the largest leaves four digits above rounding)
    for name, got, want in [("pooled", pooled, pool.detach())] + [(n, g, q[n].grad) for n, g in (
            ("W", dW), ("gamma", dgamma), ("beta", dbeta), ("K", dK), ("b", db), ("A", dA), ("D", dD), ("bias", dbias), ("B", dB), ("C", dC), ("gate", dgate), ("dt", ddt))]:
        got = got.cpu()
        assert float((got - want).abs().max()) <= 1e-10 * float(want.abs().max()), name


def test_captured_passes_replay_like_eager_ones():
    """Forward and backward of all three captured into one graph on a stream that never ran them; replays with new inputs and the
    program's own eager work between them give the eager results' bits."""
    from deepbind_amd import kangaroo_smat as ks, smat as sm
    t, v, R, N, rows = scan_inputs("float32", "long", 40, 1, 16, 0)
    T = regions(R)
    D = 40
    for n in ("X", "dt", "gate", "dY", "B", "C"):
        t[n] = torch.nan_to_num(t[n])
    W, b, g = torch.randn(4, D, device="cuda"), torch.randn(1, D, device="cuda"), torch.randn(1, D, device="cuda")

    def work():
        H, stats = sm.layernorm(t["X"], g, b, nchunk=2, want_stats=True)
        V, _ = ks.causalconv(H, W, b, T)
        keep = ks.kept_states(V, t["A"])
        keep.zero_()
        Y, last = ks.statescan(V, t["dt"], t["A"], t["B"], t["C"], T, D=t["D"], gate=t["gate"], dt_bias=t["bias"], keep=keep, want_state=True)
        grads = ks.statescan_bprop(V, t["dt"], t["A"], t["B"], t["C"], T, keep, t["dY"], D=t["D"], gate=t["gate"], dt_bias=t["bias"])
        dH, dW, db = ks.causalconv_bprop(H, W, b, T, grads[0])
        return (Y, last) + tuple(grads) + (dH, dW, db) + tuple(sm.layernorm_bprop(t["X"], g, stats, dH, nchunk=2))

    work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = work()
    for i in range(4):
        t["X"].normal_()
        t["dY"].normal_()
        eager = [x.clone() for x in work()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for j, (x, y) in enumerate(zip(captured, eager)):
            assert torch.equal(x, y), (i, j)
        work()
        torch.cuda.synchronize()


def test_calls_on_two_streams_do_not_meet():
    from deepbind_amd import kangaroo_smat as ks
    t, v, R, N, rows = scan_inputs("float32", "long", 40, 1, 16, 0)
    T = regions(R)
    base = [t[n] for n in ("X", "dt", "A", "B", "C")]
    keeps = [ks.kept_states(t["X"], t["A"]) for _ in range(2)]
    want, _ = ks.statescan(*base, T, keep=keeps[0])
    grads = ks.statescan_bprop(*base, T, keeps[0], t["dY"])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(3):
        for s, keep in zip(streams, keeps):
            with torch.cuda.stream(s):
                y, _ = ks.statescan(*base, T, keep=keep)
                got.append((y, ks.statescan_bprop(*base, T, keep, t["dY"])))
    torch.cuda.synchronize()
    for y, gr in got:
        assert torch.equal(y[rows], want[rows])
        for a, b in zip(gr, grads):
            assert a is None or torch.equal(a, b)


def test_refusals_on_the_device():
    from deepbind_amd import kangaroo_smat as ks, smat as sm
    from deepbind_amd._lib import DeepbindError
    X, W, b = torch.zeros(9, 6, device="cuda"), torch.zeros(4, 6, device="cuda"), torch.zeros(1, 6, device="cuda")
    T = regions([[0, 9]])
    for f in (lambda: sm.layernorm(X, b, b, out=X), lambda: ks.causalconv(X, W, b, T, out=X), lambda: ks.causalconv_bprop(X, W, b, T, X.clone(), out=(X, None, None)),
              lambda: ks.statescan(X, X, W, torch.zeros(9, 4, device="cuda"), torch.zeros(9, 4, device="cuda"), T, out=X),
              lambda: ks.causalconv(X, W, b, T.cpu())):
        with pytest.raises(DeepbindError):
            f()


# ------------------------------------------------------------------------------------------------ sizes beyond the tables above
def _many(rng, count, most):
    """Regions of 0 to `most` rows in random order, with gaps between some of them."""
    lens = rng.integers(0, most + 1, size=count)
    starts = np.cumsum(np.concatenate([[2], lens[:-1] + rng.integers(0, 2, size=count - 1)]))
    return np.stack([starts, starts + lens], 1)[rng.permutation(count)], int(starts[-1] + lens[-1]) + 3


def test_more_regions_than_workgroups_that_add_up_gradients():
    """5000 regions of up to three rows: each workgroup takes several; B and C with row strides of their own."""
    from deepbind_amd import kangaroo_smat as ks
    rng = np.random.default_rng(31)
    R, N = _many(rng, 5000, 3)
    D, S, K = 6, 3, 4
    f = lambda *s: rng.standard_normal(s)  # noqa: E731
    rows = inside(R, N)
    T = regions(R)
    X, x = put(f(N, D), torch.float32)
    dt, dtv = sliced(f(N, D), torch.float32, 2)
    B, b = sliced(f(N, S), torch.float32, 1)
    C, c = put(f(N, S), torch.float32)
    gate, gv = sliced(f(N, D), torch.float32, 5)
    dY, dy = put(f(N, D), torch.float32)
    A, a = put(-np.exp(f(S, D)), torch.float32)
    skip, sv = put(f(1, D), torch.float32)
    kw = dict(D=skip, gate=gate)
    keep = ks.kept_states(X, A)
    Y, last = ks.statescan(X, dt, A, B, C, T, keep=keep, want_state=True, **kw)
    got = ks.statescan_bprop(X, dt, A, B, C, T, keep, dY, **kw)
    want, size = ref.statescan(x, dtv, a, b, c, R, sv, gv, np.zeros((1, D)), dY=dy)
    k = 16 * (3 + 8) + S
    check(Y[rows], want[0][rows], size[0][rows], k, "float32", "Y")
    check(last, want[1], size[1], k, "float32", "last", stored=False)
    for name, g, w, z in zip(("dX", "ddt", "dA", "dB", "dC", "dD", "dgate"), got, want[2:], size[2:]):
        per_row = name in ("dX", "ddt", "dB", "dC", "dgate")
        if per_row:
            g, w, z = g[rows], w[rows], z[rows]
        check(g, w, z, 2 * k + D + (0 if per_row else len(rows)), "float32", name)
    W, wv = put(f(K, D), torch.float32)
    bias, bv = put(f(1, D), torch.float32)
    Z, _ = ks.causalconv(X, W, bias, T)
    (zr, _), (zs, _) = ref.causalconv(x, wv, bv, R)
    check(Z[rows], zr[rows], zs[rows], K + 12, "float32", "Z")
    grads = ks.causalconv_bprop(X, W, bias, T, dY)
    (dxr, dwr, dbr), (dxs, dws, dbs) = ref.causalconv_bprop(x, wv, bv, R, dy)
    check(grads[0][rows], dxr[rows], dxs[rows], 2 * (K + 12), "float32", "conv dX")
    check(grads[1], dwr, dws, K + 12 + len(rows), "float32", "conv dW")
    check(grads[2], dbr, dbs, K + 12 + len(rows), "float32", "conv db")


def test_maps_of_more_than_2_to_the_31_values():
    """The last rows of a map whose elements do not fit 31 bits give what the same rows give in a small map."""
    from deepbind_amd import kangaroo_smat as ks, smat as sm
    D, S, L = 1024, 2, 300
    N = (1 << 21) + 1000                          # N * D = 2.148e9 elements, 4.3 GB of bfloat16
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    small = lambda *s, dtype=torch.bfloat16: torch.randn(s, generator=g, device="cuda").to(dtype)  # noqa: E731
    ends = [(0, L), (N - L, N)]
    rows = {n: (small(L, D), small(L, D)) for n in ("X", "dt", "dY")}
    wb = {n: (small(L, S, dtype=torch.float32), small(L, S, dtype=torch.float32)) for n in ("B", "C")}
    big = {}
    for n, parts in list(rows.items()) + list(wb.items()):
        big[n] = torch.empty(N, parts[0].shape[1], dtype=parts[0].dtype, device="cuda")
        for (s, e), part in zip(ends, parts):
            big[n][s:e] = part
    A, W, b = -torch.rand((S, D), generator=g, device="cuda"), small(4, D, dtype=torch.float32), small(1, D, dtype=torch.float32)
    T, T1 = regions(ends), regions([[0, L]])
    out = torch.empty(N, D, dtype=torch.bfloat16, device="cuda")
    keep = ks.kept_states(big["X"], A)
    grads = (torch.empty_like(out), torch.empty_like(out), None, torch.empty(N, S, device="cuda"), torch.empty(N, S, device="cuda"), None, None, None)
    ks.statescan(big["X"], big["dt"], A, big["B"], big["C"], T, keep=keep, out=out)
    got = ks.statescan_bprop(big["X"], big["dt"], A, big["B"], big["C"], T, keep, big["dY"], out=grads)
    sums = 0
    for i, (s, e) in enumerate(ends):
        p = [rows["X"][i], rows["dt"][i], A, wb["B"][i], wb["C"][i], T1]
        k1 = ks.kept_states(p[0], A)
        y, _ = ks.statescan(*p, keep=k1)
        want = ks.statescan_bprop(*p, k1, rows["dY"][i])
        # the rows are cut differently in the two maps: two float32 ways to the same sums of some hundred terms, then bfloat16
        near = lambda u, v: float((u.double() - v.double()).abs().max()) <= 2 * 2.0 ** -8 * float(v.double().abs().max())  # noqa: E731
        assert near(out[s:e], y) and near(got[0][s:e], want[0]) and near(got[1][s:e], want[1]) and near(got[3][s:e], want[3]) and near(got[4][s:e], want[4])
        sums = sums + want[2].double()
    assert float((got[2].double() - sums).abs().max()) <= 1e-4 * float(sums.abs().max())
    del keep, grads, got
    ks.causalconv(big["X"], W, b, T, out=out)
    dX, dW, _ = ks.causalconv_bprop(big["X"], W, b, T, big["dY"], out=(torch.empty_like(out), None, None))
    for i, (s, e) in enumerate(ends):            # the same operations on the same numbers, row by row
        assert torch.equal(out[s:e], ks.causalconv(rows["X"][i], W, b, T1)[0])
        assert torch.equal(dX[s:e], ks.causalconv_bprop(rows["X"][i], W, b, T1, rows["dY"][i])[0])
    Z, stats = sm.layernorm(big["X"], nchunk=4, want_stats=True, out=out)
    for i, (s, e) in enumerate(ends):
        z, _ = sm.layernorm(rows["X"][i], nchunk=4)
        assert torch.equal(Z[s:e], z)


def test_state_may_be_named_as_its_own_successor():
    from deepbind_amd import kangaroo_smat as ks
    X, W, b = torch.randn(3, 8, device="cuda"), torch.randn(3, 8, device="cuda"), torch.randn(1, 8, device="cuda")
    s0 = torch.randn(3, 2, 8, device="cuda")
    s1, s2 = s0.clone(), s0.clone()
    assert torch.equal(ks.causalconv_step(X, W, b, s1), ks.causalconv_step(X, W, b, s2, into=s2)) and torch.equal(s1, s2)
    A, B = -torch.rand(4, 8, device="cuda"), torch.randn(3, 4, device="cuda")
    h0 = torch.randn(3, 4, 8, device="cuda")
    h1, h2 = h0.clone(), h0.clone()
    assert torch.equal(ks.statescan_step(X, X, A, B, B, h1), ks.statescan_step(X, X, A, B, B, h2, into=h2)) and torch.equal(h1, h2) and not torch.equal(h0, h1)


@pytest.mark.parametrize("kind", ["float32", "float64"])
@pytest.mark.parametrize("gated", [False, True])
def test_statescan_gradient_of_a_state_that_overflows_at_the_last_row(kind, gated):
    """The last state enters the last row's value alone: the gradient of A holds no product with it and stays what it is, also
    where rows are taken several at a time and the region ends among them."""
    from deepbind_amd import kangaroo_smat as ks
    t, v, R, N, rows = scan_inputs(kind, "ragged", 70, 1, 16, 0)
    T = regions(R)
    for s, e in ref.rows_of(R, N):
        if e > s:
            t["X"][e - 1, 3] = v["X"][e - 1, 3] = float("inf")
    kw = dict(gate=t["gate"] if gated else None)
    base = [t[n] for n in ("X", "dt", "A", "B", "C")]
    keep = ks.kept_states(t["X"], t["A"])
    ks.statescan(*base, T, keep=keep, **kw)
    dA = ks.statescan_bprop(*base, T, keep, t["dY"], **kw)[2]
    with np.errstate(invalid="ignore"):
        (_, _, *grads), (_, _, *sizes) = ref.statescan(*[v[n] for n in ("X", "dt", "A", "B", "C")], R, np.zeros((1, 70)), v["gate"] if gated else None,
                                                       np.zeros((1, 70)), True, dY=v["dY"])
    assert np.isfinite(grads[2]).all()
    longest = max(e - s for s, e in ref.rows_of(R, N))
    # (the same roundings as in the other tests of the gradients)
    check(dA, grads[2], sizes[2], 2 * (16 * (longest + 8) + 16) + 70 + len(rows), kind, "dA", stored=False)


def test_as_many_sequences_as_a_launch_takes():
    """Single rows of nearly 2^24 sequences, each against its own formula (one channel, one state: a few roundings, k = 16 as elsewhere)."""
    from deepbind_amd import kangaroo_smat as ks
    n = (1 << 24) - 4096
    g = torch.Generator(device="cuda").manual_seed(3)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    X, dt, B, C, A, state, W = f(n, 1), f(n, 1).abs(), f(n, 1), f(n, 1), -f(1, 1).abs(), f(n, 1, 1), f(2, 1)
    i = torch.arange(n, dtype=torch.int64)
    R = torch.stack([i, i + 1], 1).to(torch.uint32).cuda()
    x, d, b, c, a, w = (v.double() for v in (X, dt, B, C, A, W))

    def near(got, want, size):
        return bool(((got.double() - want).abs() <= 16 * 2.0 ** -24 * size + 1e-35).all())

    h = torch.exp(d * a)
    for s in (state, None):
        before = 0 if s is None else s.double().view(n, 1)
        now, size = h * before + d * x * b, h * (1 + (d * a).abs()) * abs(before) + (d * x * b).abs()
        Y = ks.statescan(X, dt, A, B, C, R, softplus=False)[0] if s is None else ks.statescan_step(X, dt, A, B, C, s, softplus=False, into=torch.empty_like(s))
        assert near(Y, c * now, c.abs() * size)
    assert near(ks.causalconv(X, W, None, R, silu=False)[0], x * w[1], (x * w[1]).abs())
    last = state.clone()
    Z = ks.causalconv_step(X, W, None, last, silu=False)
    assert near(Z, x * w[1] + state.double().view(n, 1) * w[0], (x * w[1]).abs() + (state.double().view(n, 1) * w[0]).abs()) and torch.equal(last.view(n, 1), X)
    dX, dW, _ = ks.causalconv_bprop(X, W, None, R, dt, silu=False)
    assert near(dX, d * w[1], (d * w[1]).abs()) and not bool(dW[0].any())
    # (each of 2048 workgroups adds 8192 products one after another, at most: n roundings bound it)
    assert abs(float(dW[1]) - float((d * x).sum())) <= 16384 * 2.0 ** -24 * float((d * x).abs().sum())
