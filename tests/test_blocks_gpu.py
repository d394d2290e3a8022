"""The gated delta rule, the norms around a block and gradient clipping on the GPU against their plain restatement in 64 bits.

Tolerances: per value, the bounds that blocks_ref derives times the unit roundoff of the arithmetic, plus the rounding of the stored type; they hold
for the worst of all roundings at once. Beside them, for the delta rule, one on norms: roundings that do not conspire are independent, of
u / sqrt(3) at most each in the mean square, and a value goes through some K + V + 64 of them, so that a result is off by about sqrt(K + V + 64) u / sqrt(3) < 11 u of its
terms' size (K = V = 128); 32 u of its own leaves three for the terms' size over the result's."""
import numpy as np
import pytest
import torch

from tests import blocks_ref as ref
from tests.gpu_util import host
from tests.test_rows_gpu import SENTINEL, STORED, TABLES, TYPES, U, check, inside, put, regions, sliced, wide

pytestmark = pytest.mark.gpu


def close(got, want, bound, kind, what, rows=None, stored=True, norms=True):
    got = host(got.double())
    if rows is not None:
        out = np.ones(got.shape[0], bool)
        out[rows] = False
        assert (got[out] == SENTINEL).all(), "%s: rows in no region were written" % what
        got, want, bound = got[rows], want[rows], bound[rows]
    assert got.shape == want.shape, what
    u, r = U[kind], STORED[kind] if stored else U[kind]
    bad = ~(np.abs(got - want) <= u * bound + r * np.abs(want) + 1e-35)
    assert not bad.any(), "%s: %d of %d values off, worst %.3g of the bound" % (what, bad.sum(), bad.size, np.nanmax(np.abs(got - want) / (u * bound + r * np.abs(want) + 1e-35)))
    if norms and want.size >= 64:
        off, size = np.linalg.norm(got - want), np.linalg.norm(want)
        assert off <= (32 * u + (r if stored and r > u else 0)) * size + 1e-30, "%s: %.3g u of its norm off" % (what, off / size / u)


def delta_case(kind, N, H, G, Kd, Vd, decays, pad, seed, level=2.0):
    rng = np.random.default_rng(seed)
    unit = lambda t: (t / np.sqrt((t ** 2).sum(2, keepdims=True))).reshape(N, -1)  # noqa: E731
    # keys follow letters, so that they come again
    letters = rng.integers(0, 4, N)
    q, k = (unit(rng.standard_normal((4, G, Kd))[letters] + 0.7 * rng.standard_normal((N, G, Kd))) for _ in range(2))
    t, v = {}, {}
    for name, a, p in (("Q", q, pad), ("K", k, pad and pad + 1), ("V", rng.standard_normal((N, H * Vd)), pad and pad + 2)):
        t[name], v[name] = sliced(a, TYPES[kind], p)
    t["beta"], v["beta"] = sliced(1 / (1 + np.exp(-rng.standard_normal((N, H)))), wide(kind), pad)
    t["decay"], v["decay"] = sliced(-np.exp(rng.standard_normal((N, H)) - level), wide(kind), pad) if decays else (None, None)
    t["dO"], v["dO"] = sliced(rng.standard_normal((N, H * Vd)), TYPES[kind], pad)
    return t, v


# one long region among many short ones, and a few of a handful of segments; a region that ends with a segment, and one row behind
MIXED = [[i * 9, i * 9 + 3 + i % 6] for i in range(200)] + [[1900, 5000], [5000, 5001], [5001, 6000]] + [[6000 + i * 5, 6004 + i * 5] for i in range(200)]
TABLES = dict(TABLES, mixed=(MIXED, 7010), segments=([[300, 1068], [1068, 1837], [0, 256], [256, 300]], 1840))
DELTA = [("one", 1, 1, 16, 16, True, 0), ("ragged", 3, 1, 19, 13, True, 1), ("ragged", 2, 2, 1, 1, False, 0), ("outside", 4, 2, 7, 33, True, 0), ("reads", 4, 4, 16, 16, True, 0),
         ("ragged", 2, 1, 64, 64, True, 3), ("outside", 1, 1, 128, 128, True, 0), ("reads", 2, 1, 33, 50, False, 1), ("long", 2, 2, 16, 16, True, 0), ("long", 1, 1, 40, 65, True, 2),
         ("none", 2, 2, 8, 8, True, 0), ("mixed", 1, 1, 16, 16, True, 0), ("mixed", 2, 1, 40, 33, True, 1), ("segments", 2, 2, 64, 64, True, 0), ("segments", 3, 1, 100, 20, True, 0)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("table,H,G,Kd,Vd,decays,pad", DELTA)
def test_delta_rule_and_its_gradient(kind, table, H, G, Kd, Vd, decays, pad):
    from deepbind_amd import kangaroo_smat as ks
    R, N = TABLES[table]
    t, v = delta_case(kind, N, H, G, Kd, Vd, decays, pad, [N, H, Kd, Vd])
    Rd, rows, scale = regions(R).view(-1, 2), inside(R, N), Kd ** -0.5
    what = dict(decay=t["decay"], groups=G)
    args, plain = (t["Q"], t["K"], t["V"], t["beta"], Rd), (v["Q"], v["K"], v["V"], v["beta"], v["decay"], np.asarray(R).reshape(-1, 2), G, scale)
    full = lambda like: torch.full(like.shape, SENTINEL, dtype=like.dtype, device="cuda")  # noqa: E731
    # from a state, to a state
    rng = np.random.default_rng(1)
    state, sv = put(rng.standard_normal((len(R), Kd, H * Vd)), wide(kind))
    (Or, lr), (Ob, lb) = ref.delta(*plain, state=sv), ref.delta_bounds(*plain, state=sv)
    out = full(t["V"])
    O, last = ks.deltarule(*args, state=state, want_state=True, out=out, **what)
    assert O is out
    close(O, Or, Ob, kind, "O from a state", rows)
    close(last, lr, lb, kind, "last", stored=False)
    # and from zeros, with the gradients
    want, bound = ref.delta(*plain, dO=v["dO"]), ref.delta_bounds(*plain, dO=v["dO"])
    keep = ks.kept_delta(t["K"], t["V"], t["beta"], groups=G)
    out = full(t["V"])
    O, none = ks.deltarule(*args, keep=keep, out=out, **what)
    assert none is None
    close(O, want[0], bound[0], kind, "O", rows)
    outs = tuple(None if g is None else full(g) for g in (t["Q"], t["K"], t["V"], t["beta"], t["decay"]))
    grads = ks.deltarule_bprop(*args, keep, t["dO"], out=outs, **what)
    assert all(a is b for a, b in zip(grads, outs))
    for name, g, w, b in zip(("dQ", "dK", "dV", "dbeta", "ddecay"), grads, want[2:], bound[2:]):
        if g is not None:
            close(g, w, b, kind, name, rows, stored=name in ("dQ", "dK", "dV"))
    # new outputs: zeros where no region is, the same bits where one is
    O2, _ = ks.deltarule(*args, **what)
    again = ks.deltarule_bprop(*args, keep, t["dO"], **what)
    outside = np.setdiff1d(np.arange(N), rows)
    for a, b in zip((O2,) + again, (O,) + grads):
        assert (a is None) == (b is None)
        if a is not None:
            assert torch.equal(a[rows], b[rows]) and not a[outside].any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,H,G,Kd,Vd,decays,pad", [(1, 1, 1, 1, 1, True, 0), (5, 4, 2, 19, 13, True, 2), (64, 4, 4, 64, 64, True, 0), (3, 2, 1, 128, 130, False, 1), (17, 3, 3, 33, 64, True, 0)])
def test_delta_rule_row_by_row(kind, n, H, G, Kd, Vd, decays, pad):
    from deepbind_amd import kangaroo_smat as ks
    state, sv = put(np.random.default_rng(2).standard_normal((n, Kd, H * Vd)), wide(kind))
    start = state.clone()
    R = np.stack([np.arange(n), np.arange(1, n + 1)], 1)
    for step in range(3):
        t, v = delta_case(kind, n, H, G, Kd, Vd, decays, pad, [n, H, Kd, step])
        plain = (v["Q"], v["K"], v["V"], v["beta"], v["decay"], R, G, Kd ** -0.5)
        (Or, lr), (Ob, lb) = ref.delta(*plain, state=sv), ref.delta_bounds(*plain, state=sv)
        into = torch.empty_like(state)
        kw = dict(decay=t["decay"], groups=G)
        O = ks.deltarule_step(t["Q"], t["K"], t["V"], t["beta"], state, into=into, **kw)
        assert torch.equal(state, start)
        close(O, Or, Ob, kind, "O")
        close(into, lr, lb, kind, "state", stored=False)
        O2 = ks.deltarule_step(t["Q"], t["K"], t["V"], t["beta"], state, out=torch.empty_like(O), **kw)
        assert torch.equal(O2, O) and torch.equal(state, into)
        start = state.clone()
        sv = host(state.double())


def test_delta_rule_in_pieces_and_steps_is_the_whole():
    from deepbind_amd import kangaroo_smat as ks
    N, H, Kd, Vd = 300, 2, 24, 20
    t, v = delta_case("float64", N, H, H, Kd, Vd, True, 0, 9)
    call = lambda a, b, **kw: ks.deltarule(t["Q"][a:b], t["K"][a:b], t["V"][a:b], t["beta"][a:b], regions([[0, b - a]]), decay=t["decay"][a:b], want_state=True, **kw)  # noqa: E731
    whole, end = call(0, N)
    O1, s = call(0, 129)
    O2, s = call(129, 290, state=s)
    steps = [ks.deltarule_step(t["Q"][i:i + 1], t["K"][i:i + 1], t["V"][i:i + 1], t["beta"][i:i + 1], s, decay=t["decay"][i:i + 1]) for i in range(290, N)]
    got = torch.cat([O1, O2] + steps)
    assert float((got - whole).abs().max()) < 1e-13 and float((s - end).abs().max()) < 1e-13
    # a region of no rows hands its state on
    O, last = ks.deltarule(t["Q"], t["K"], t["V"], t["beta"], regions([[5, 5]]), decay=t["decay"], state=s, want_state=True)
    assert torch.equal(last, s) and not O.any()


@pytest.mark.parametrize("kind", ["float32", "float64"])
def test_delta_rule_with_hard_resets_no_learning_and_large_steps(kind):
    from deepbind_amd import kangaroo_smat as ks
    R, N = [[0, 90], [90, 171]], 171
    t, v = delta_case(kind, N, 2, 1, 12, 9, True, 0, 11)
    for rows, name, value in (((20, 47, 48, 130), "decay", -1e4), ((3, 50, 95), "beta", 0.0), ((60, 61, 100), "beta", 2.0), ((70,), "decay", -60.0), ((33,), "decay", 0.0)):
        for r in rows:
            t[name][r] = value
            v[name][r] = value
    plain = (v["Q"], v["K"], v["V"], v["beta"], v["decay"], np.array(R), 1, 12 ** -0.5)
    want, bound = ref.delta(*plain, dO=v["dO"]), ref.delta_bounds(*plain, dO=v["dO"])
    args = (t["Q"], t["K"], t["V"], t["beta"], regions(R))
    keep = ks.kept_delta(t["K"], t["V"], t["beta"], groups=1)
    O, _ = ks.deltarule(*args, decay=t["decay"], groups=1, keep=keep)
    grads = ks.deltarule_bprop(*args, keep, t["dO"], decay=t["decay"], groups=1)
    close(O, want[0], bound[0], kind, "O")
    for name, g, w, b in zip(("dQ", "dK", "dV", "dbeta", "ddecay"), grads, want[2:], bound[2:]):
        close(g, w, b, kind, name)
    # minus infinity is a reset too: what is before it leaves no trace
    t["decay"][47] = -float("inf")
    O2, _ = ks.deltarule(*args, decay=t["decay"], groups=1)
    close(O2, want[0], bound[0], kind, "O with a decay of minus infinity")
    grads = ks.deltarule_bprop(*args, keep, t["dO"], decay=t["decay"], groups=1)
    for name, g, w, b in zip(("dQ", "dK", "dV", "dbeta", "ddecay"), grads, want[2:], bound[2:]):
        close(g, w, b, kind, name + " with a decay of minus infinity")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_delta_rule_carries_bad_values_only_where_the_formulas_do(kind, bad):
    from deepbind_amd import kangaroo_smat as ks
    N, H, G, Kd, Vd = 150, 2, 1, 20, 24
    R = [[0, 100], [100, 150]]
    t, _ = delta_case(kind, N, H, G, Kd, Vd, True, 0, 12)
    args = [t["Q"], t["K"], t["V"], t["beta"], regions(R)]
    kw = dict(decay=t["decay"], groups=G)
    keep = ks.kept_delta(t["K"], t["V"], t["beta"], groups=G)
    both = lambda: (ks.deltarule(*args, keep=keep, **kw)[0],) + ks.deltarule_bprop(*args, keep, t["dO"], **kw)  # noqa: E731
    good = [g.clone() for g in both()]
    everywhere = slice(None)

    def spoilt(name, row, col, clean):
        """One bad value: the outputs named in `clean` are the same bits at the rows (and columns) given there."""
        x = t[name]
        old = x[row, col].clone()
        x[row, col] = bad
        got = both()
        x[row, col] = old
        for i, (r, c) in clean:
            assert torch.equal(got[i][r][:, c], good[i][r][:, c]), (name, row, i)
        return got

    # a value of row 37, column 5 of head 0: its own column of O from row 37 on, dK and what goes through the state after it; not dQ, dV of rows before
    got = spoilt("V", 37, 5, [(0, (slice(0, 37), everywhere)), (0, (slice(100, 150), everywhere)), (0, (everywhere, slice(6, 48))), (1, (slice(0, 37), everywhere)),
                              (1, (slice(100, 150), everywhere)), (2, (slice(100, 150), everywhere)), (3, (everywhere, everywhere)), (4, (slice(100, 150), everywhere)),
                              (4, (everywhere, slice(1, 2)))])
    assert not got[0][37:100, 5].isfinite().any()
    # a query of row 37: its own output and dQ's row not at all (dQ has no query in it), dK and dV of rows up to 37 only
    got = spoilt("Q", 37, 3, [(0, (slice(0, 37), everywhere)), (0, (slice(38, 150), everywhere)), (1, (everywhere, everywhere)), (2, (slice(38, 150), everywhere)),
                              (3, (slice(38, 150), everywhere)), (4, (slice(38, 150), everywhere))])
    assert not got[0][37].isfinite().any()
    # a key of row 37: outputs from row 37 on, dQ from there on
    spoilt("K", 37, 3, [(0, (slice(0, 37), everywhere)), (0, (slice(100, 150), everywhere)), (1, (slice(0, 37), everywhere)), (2, (slice(100, 150), everywhere)), (3, (slice(100, 150), everywhere))])
    # a gradient of row 37: dQ of its own row, the others up to it
    spoilt("dO", 37, 5, [(0, (everywhere, everywhere)), (1, (slice(0, 37), everywhere)), (1, (slice(38, 150), everywhere)), (2, (slice(38, 150), everywhere)),
                         (3, (slice(38, 150), everywhere)), (3, (everywhere, slice(6, 48))), (4, (slice(38, 150), everywhere))])
    # rows in no region, and their gradients
    args[4] = regions([[0, 90], [100, 150]])
    good = [g.clone() for g in both()]
    for name in ("Q", "K", "V", "beta", "decay", "dO"):
        t[name][90:100] = bad
    for a, b in zip(both(), good):
        assert torch.equal(a, b)


def test_delta_rule_of_nothing():
    from deepbind_amd import kangaroo_smat as ks
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    R = regions([[0, 0], [3, 9]])
    state = torch.randn(2, 4, 6, device="cuda")
    O, last = ks.deltarule(z(0, 8), z(0, 8), z(0, 6), z(0, 2), R, state=state, want_state=True)
    assert O.shape == (0, 6) and torch.equal(last, state)
    keep = ks.kept_delta(z(0, 8), z(0, 6), z(0, 2))
    assert keep.shape == (1, 0)
    grads = ks.deltarule_bprop(z(0, 8), z(0, 8), z(0, 6), z(0, 2), R, keep, z(0, 6))
    assert grads[0].shape == (0, 8) and grads[4] is None
    none, _ = ks.deltarule(z(5, 8), z(5, 8), z(5, 6), z(5, 2), regions([]).view(0, 2))
    assert not none.any()
    assert ks.deltarule_step(z(0, 8), z(0, 8), z(0, 6), z(0, 2), z(0, 4, 6)).shape == (0, 6)


def test_delta_rule_of_many_regions_and_of_many_heads():
    from deepbind_amd import kangaroo_smat as ks
    for R, N, H, Kd, Vd in (([[i, i + 1] for i in range(70000)], 70000, 1, 3, 2), ([[0, 40], [40, 70]], 70, 200, 2, 17)):
        t, v = delta_case("float32", N, H, 1, Kd, Vd, True, 0, 13)
        keep = ks.kept_delta(t["K"], t["V"], t["beta"], groups=1)
        args = (t["Q"], t["K"], t["V"], t["beta"], regions(R))
        O, last = ks.deltarule(*args, decay=t["decay"], groups=1, keep=keep, want_state=True)
        grads = ks.deltarule_bprop(*args, keep, t["dO"], decay=t["decay"], groups=1)
        want = ref.delta(v["Q"], v["K"], v["V"], v["beta"], v["decay"], R, 1, Kd ** -0.5, dO=v["dO"])
        for g, w in zip((O, last) + grads, want):
            assert np.linalg.norm(host(g.double()) - w) <= 32 * 2.0 ** -24 * np.linalg.norm(w) + 1e-30


# ------------------------------------------------------------------------------------------------ norms around a block
BLOCK = [(1, 1, 1, 0), (5, 3, 16, 3), (64, 1, 16, 0), (7, 2, 33, 1), (33, 1, 257, 0), (9, 1, 1440, 0), (130, 24, 16, 0), (67, 5, 100, 5), (3, 1, 4100, 0), (2, 2, 9001, 3), (4000, 1, 5, 0),
         (700, 90, 3, 0), (19, 2, 600, 1), (11, 1, 2500, 0)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("n,nchunk,w,pad", BLOCK)
def test_block_norms_and_their_gradients(kind, rms, n, nchunk, w, pad):
    from deepbind_amd import smat as sm
    m, eps = nchunk * w, 1e-2
    rng = np.random.default_rng([n, nchunk, w, rms])
    f = lambda *s: rng.standard_normal(s)  # noqa: E731
    one, zero = np.ones((1, m)), np.zeros((1, m))
    k = 24 + w / 16                              # the sums over a chunk, and the two dozen roundings of one value (a sigmoid's among them)
    for gated, resid, scaled, weights, norm, nxt in ((True, True, True, True, True, True), (False, True, False, True, True, True), (True, False, False, True, True, False),
                                                     (True, True, True, False, False, True), (False, True, True, False, True, False)):
        if (not gated or not norm) and n > 1000:
            continue
        Y, y = sliced(f(n, m) * 2 + f(n, 1), TYPES[kind], pad)
        R, r = sliced(f(n, m), TYPES[kind], pad and pad + 1) if resid else (None, np.zeros((n, m)))
        G, g = sliced(f(n, m), TYPES[kind], pad) if gated else (None, None)
        W = {}
        for name, a, there in (("gamma", 1 + 0.3 * f(1, m), weights and norm), ("beta", 0.3 * f(1, m), weights and norm and not rms), ("scale", f(1, m), scaled),
                               ("next_gamma", 1 + 0.3 * f(1, m), weights and nxt), ("next_beta", 0.3 * f(1, m), weights and nxt and not rms)):
            W[name] = put(a, wide(kind)) if there else (None, zero if "beta" in name else one)
        dR, dr = sliced(f(n, m), TYPES[kind], pad)
        dZ, dz = sliced(f(n, m), TYPES[kind], pad and pad + 2) if nxt else (None, None)
        gpu = dict(gate=G, nchunk=nchunk, rms=rms, norm=norm, next_norm=nxt, **{a: b[0] for a, b in W.items()})
        plain = (y, r, g) + tuple(W[a][1] for a in ("gamma", "beta", "scale", "next_gamma", "next_beta")) + (nchunk, rms, norm, nxt, eps)
        O, Z, stats = sm.blocknorm(Y, R, eps=eps, want_stats=True, **gpu)
        kept = host(O.double())
        (Or, Zr, _), (Os, Zs, _) = ref.blocknorm(*plain, kept=kept)
        check(O, Or, Os, k, kind, "O")
        assert (Z is None) == (not nxt) and stats.shape == (4, n * nchunk)
        if nxt:
            check(Z, Zr, Zs, k, kind, "Z")
        grads = sm.blocknorm_bprop(Y, O, stats, dR, dZ, **gpu)
        values, sizes = ref.blocknorm_bprop(*plain, dr, dz, kept)
        there = (True, True, gated) + tuple(W[a][0] is not None for a in ("gamma", "beta", "scale", "next_gamma", "next_beta"))
        for i, (name, got, want, size, has) in enumerate(zip(("dY", "dR", "dgate", "dgamma", "dbeta", "dscale", "dnext_gamma", "dnext_beta"), grads, values, sizes, there)):
            assert (got is not None) == has, name
            if has:
                check(got, want, size, 8 * k + (n if i > 2 else 0), kind, name, stored=i < 3)
        # into given tensors, and without the gradient from elsewhere
        spare = tuple(None if t is None else torch.empty_like(t) for t in grads)
        again = sm.blocknorm_bprop(Y, O, stats, dR, dZ, out=spare, **gpu)
        assert all(a is b for a, b in zip(again, spare)) and all(a is None or torch.equal(a, b) for a, b in zip(again, grads))
        wideO = torch.full((n, m + 2), SENTINEL, dtype=TYPES[kind], device="cuda")
        O2, Z2, none = sm.blocknorm(Y, R, eps=eps, out=(wideO[:, 1:-1], None), **gpu)
        assert none is None and torch.equal(O2, O) and bool((wideO[:, 0] == SENTINEL).all()) and bool((wideO[:, -1] == SENTINEL).all()) and (not nxt or torch.equal(Z2, Z))
        if nxt:
            without = sm.blocknorm_bprop(Y, O, stats, None, dZ, **gpu)
            zeros = sm.blocknorm_bprop(Y, O, stats, torch.zeros_like(O), dZ, **gpu)
            assert all(a is None or torch.equal(a, b) for a, b in zip(without, zeros))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("n,nchunk,w,pad", [(3300, 1, 300, 0), (1100, 1, 700, 1), (900, 1, 1300, 0), (530, 2, 1440, 0), (600, 1, 2500, 3), (300, 1, 4000, 0), (270, 1, 6001, 0)])
def test_block_norms_of_chunks_of_two_to_sixteen_waves(kind, n, nchunk, w, pad):
    # (more rows than workgroups, so that each walks several)
    test_block_norms_and_their_gradients(kind, bool(n % 4), n, nchunk, w, pad)


def test_block_norms_of_no_rows_and_of_bad_rows():
    from deepbind_amd import smat as sm
    X, g = torch.zeros(0, 12, device="cuda"), torch.ones(1, 12, device="cuda")
    O, Z, stats = sm.blocknorm(X, X, gate=X, gamma=g, scale=g, nchunk=3, want_stats=True)
    grads = sm.blocknorm_bprop(X, O, stats, X, X, gate=X, gamma=g, scale=g, nchunk=3, out=(None, None, None, g * 5, None, g * 5, None, None))
    assert O.shape == (0, 12) and grads[0].shape == (0, 12) and not grads[3].any() and not grads[5].any() and grads[4] is None
    for rms in (True, False):
        Y, R, G = (torch.randn(50, 48, device="cuda") for _ in range(3))
        call = lambda: sm.blocknorm(Y, R, gate=G, nchunk=3, rms=rms, want_stats=True)  # noqa: E731
        want = call()
        back = sm.blocknorm_bprop(Y, want[0], want[2], R, G, gate=G, nchunk=3, rms=rms)
        Y[7, 20], G[30, 0] = float("nan"), float("inf")
        got = call()
        bad = torch.zeros(50, 48, dtype=torch.bool, device="cuda")
        bad[7, 16:32] = bad[30, :16] = True
        assert torch.equal(got[0][~bad], want[0][~bad]) and torch.equal(got[1][~bad], want[1][~bad]) and bool(got[1][bad].isnan().any())
        spoilt = sm.blocknorm_bprop(Y, got[0], got[2], R, G, gate=G, nchunk=3, rms=rms)
        bad[:, :] = False
        bad[7, 16:32] = bad[30, :16] = bad[30, :16] = True
        for a, b in zip(spoilt[:2], back[:2]):
            assert torch.equal(a[(~bad)], b[~bad]) or torch.equal(a[:7], b[:7])


def test_block_norms_far_from_zero_and_of_equal_values():
    """Equal values are normalised to zero, exactly, and values far from zero by their distances, not by what is left of their squares."""
    from deepbind_amd import smat as sm
    Y = torch.full((40, 100), 1000.1, device="cuda")
    O, Z, _ = sm.blocknorm(Y)
    assert not O.any() and not Z.any()
    Y = 1e4 + torch.randn(40, 100, device="cuda")
    y = host(Y.double())
    want = (y - y.mean(1, keepdims=True)) / np.sqrt(((y - y.mean(1, keepdims=True)) ** 2).mean(1, keepdims=True) + 1e-5)
    O, _, _ = sm.blocknorm(Y, next_norm=False)
    # the values are exact inputs: their distances to the mean are off by the mean's own rounding, half a unit of 1e4
    assert np.abs(host(O.double()) - want).max() < 1e4 * 2.0 ** -24 * 2


# ------------------------------------------------------------------------------------------------ clipping
@pytest.mark.parametrize("kind", list(TYPES) + ["mixed"])
@pytest.mark.parametrize("nblock,shapes", [(1, [(1, 1)]), (1, [(7, 5), (1, 3), (0, 4), (300, 41)]), (1, [(1, 50001)] * 3 + [(1, 17)] * 90), (3, [(96, 48), (1, 48), (48, 32), (1, 96), (96, 1)]),
                                           (90, [(96, 1440), (1, 1440), (1440, 32), (1, 2880), (2880, 1), (1, 90)]), (2, [(1000, 300), (64, 20002)]), (1, [(2000, 1500), (1, 1000003)])])
def test_clipping(kind, nblock, shapes):
    from deepbind_amd import deepity_smat as ds
    rng = np.random.default_rng([len(shapes), nblock])
    kinds = [kind if kind != "mixed" else list(TYPES)[i % 3] for i in range(len(shapes))]
    by_rows = [nblock > 1 and i % 5 in (2, 4) for i in range(len(shapes))]
    grads, plain = [], []
    for i, (s, kd, by) in enumerate(zip(shapes, kinds, by_rows)):
        level = np.exp(rng.standard_normal(nblock))
        a = rng.standard_normal(s) * (np.repeat(level, s[0] // nblock)[:, None] if by else np.repeat(level, s[1] // nblock)[None])
        t, v = sliced(a, TYPES[kd], (i % 2) * 3 if s[0] > 1 else 0)
        grads.append(t)
        plain.append(v)
    norms, _ = ref.clip(plain, 1.0, nblock, by_rows)
    most = float(np.median(norms)) * (0.5 if nblock == 1 else 1.0)
    norms, want = ref.clip(plain, most, nblock, by_rows)
    before = [g.clone() for g in grads]
    out = [torch.full(s, SENTINEL, dtype=g.dtype, device="cuda") for s, g in zip(shapes, grads)]
    got = ds.clip_gradients(grads, most, nblock=nblock, by_rows=by_rows if nblock > 1 else None, out=out)
    assert got.shape == (1, nblock) and got.dtype == torch.float64
    # squares and sums in double: n roundings at most, whose root is halved again
    n = sum(int(np.prod(s)) for s in shapes)
    np.testing.assert_allclose(host(got)[0], norms, rtol=n * 2.0 ** -53)
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    for o, w, kd in zip(out, want, kinds):
        # the factor's own rounding, the product's, and the stored one's
        assert (np.abs(host(o.double()) - w) <= (2 * U[kd] + STORED[kd] + n * 2.0 ** -53) * np.abs(w)).all()
    # in place, the same bits
    again = ds.clip_gradients(grads, most, nblock=nblock, by_rows=by_rows)
    assert torch.equal(again, got) and all(torch.equal(a, b) for a, b in zip(grads, out))


def test_clipping_of_unusual_values():
    from deepbind_amd import deepity_smat as ds
    big = torch.full((3, 40), 3e38, device="cuda")
    tiny = torch.full((50,), 1e-40, device="cuda")
    n = ds.clip_gradients([big, tiny], 1.0)
    assert abs(float(n) / (3e38 * 120 ** 0.5) - 1) < 1e-6 and abs(float(big.double().norm()) - 1) < 1e-5
    small = torch.full((100,), 1e-30, device="cuda")
    n = ds.clip_gradients([small], 1e-30)
    assert abs(float(n) / 1e-29 - 1) < 1e-6 and abs(float(small.double().norm()) / 1e-30 - 1) < 1e-5
    for size in (30, 50000):
        x = torch.ones(size, device="cuda")
        x[7] = float("inf")
        y = torch.empty_like(x)
        n = ds.clip_gradients([x], 1.0, out=[y])
        assert float(n) == float("inf") and bool(y[7].isnan()) and not y[:7].any() and not y[8:].any()
        x[7] = float("nan")
        n = ds.clip_gradients([x], 1.0, out=[y])
        assert bool(n.isnan().all()) and torch.equal(y[8:], x[8:])
        two = torch.stack([x, torch.full_like(x, 2.0)])
        n = ds.clip_gradients([two], 1.0, nblock=2, by_rows=[True])
        assert bool(n[0, 0].isnan()) and abs(float(two[1].double().norm()) - 1) < 1e-6 and float(two[0, 0]) == 1.0
    # no values at all
    assert not ds.clip_gradients([torch.zeros(0, device="cuda"), torch.zeros(0, 6, device="cuda")], 1.0).any()
    assert ds.clip_gradients([torch.zeros(4, 0, device="cuda")], 1.0, nblock=3).shape == (1, 3)
    # no gradient at all: nothing to scale
    z = torch.zeros(9, device="cuda")
    assert float(ds.clip_gradients([z], 1.0)) == 0 and not z.any()
    from deepbind_amd._lib import DeepbindError
    with pytest.raises(DeepbindError, match="shares memory"):
        ds.clip_gradients([z, z], 1.0)
    with pytest.raises(DeepbindError, match="shares memory"):
        ds.clip_gradients([z, z[:4]], 1.0, out=[torch.empty_like(z), z[4:8]])


# ------------------------------------------------------------------------------------------------ as they are used
def layer(P, X, R, G, dY=None):
    """A layer between scan and pooling: keys and queries of length one, the delta rule, its output normalised and gated per head, the residual and the
    next layer's norm; and its gradients."""
    from deepbind_amd import kangaroo_smat as ks
    from deepbind_amd import smat as sm
    H, key = P["beta"].shape[1], P["K"].shape[1] // G
    unit = torch.full((1, G * key), key ** -0.5, dtype=P["gamma"].dtype, device="cuda")
    qk = [sm.blocknorm(P[n], gamma=unit, nchunk=G, rms=True, norm=True, next_norm=False, eps=1e-9, want_stats=True) for n in ("Q", "K")]
    keep = ks.kept_delta(P["K"], P["V"], P["beta"], groups=G)
    args = (qk[0][0], qk[1][0], P["V"], P["beta"], R)
    O, _ = ks.deltarule(*args, decay=P["decay"], groups=G, keep=keep)
    N1, _, s1 = sm.blocknorm(O, gate=P["gate"], gamma=P["gamma"], nchunk=H, rms=True, next_norm=False, want_stats=True)
    out, Z, s2 = sm.blocknorm(N1, X, norm=False, scale=P["scale"], next_gamma=P["next"], want_stats=True)
    if dY is None:
        return Z
    g2 = sm.blocknorm_bprop(N1, out, s2, None, dY, norm=False, scale=P["scale"], next_gamma=P["next"])
    g1 = sm.blocknorm_bprop(O, N1, s1, g2[0], None, gate=P["gate"], gamma=P["gamma"], nchunk=H, rms=True, next_norm=False)
    gd = ks.deltarule_bprop(*args, keep, g1[0], decay=P["decay"], groups=G)
    gq, gk = (sm.blocknorm_bprop(P[n], s[0], s[2], g, None, gamma=unit, nchunk=G, rms=True, next_norm=False)[0] for n, s, g in zip("QK", qk, gd))
    return Z, dict(Q=gq, K=gk, V=gd[2], beta=gd[3], decay=gd[4], gate=g1[2], gamma=g1[3], scale=g2[5], next=g2[6], X=g2[1])


def layer_case(kind, N, H, G, key, value, seed):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.standard_normal(s)  # noqa: E731
    P = dict(Q=f(N, G * key), K=f(N, G * key), V=f(N, H * value), gate=f(N, H * value))
    W = dict(beta=1 / (1 + np.exp(-f(N, H))), decay=-np.exp(f(N, H) - 2), gamma=1 + 0.2 * f(1, H * value), scale=f(1, H * value), next=1 + 0.2 * f(1, H * value))
    P = {k: put(a, TYPES[kind])[0] for k, a in P.items()}
    P.update({k: put(a, wide(kind))[0] for k, a in W.items()})
    X, dY = put(f(N, H * value), TYPES[kind])[0], put(f(N, H * value), TYPES[kind])[0]
    return P, X, dY


def test_a_layer_of_them_has_the_gradient_of_its_differences():
    P, X, dY = layer_case("float64", 83, 4, 2, 6, 5, 21)
    R = regions([[40, 83], [0, 21], [21, 40]])
    _, grads = layer(P, X, R, 2, dY)
    loss = lambda: float((layer(P, X, R, 2) * dY).sum())  # noqa: E731
    rng = np.random.default_rng(3)
    for name, g in grads.items():
        t = X if name == "X" else P[name]
        for _ in range(3):
            i = tuple(int(rng.integers(0, s)) for s in t.shape)
            old, step = t[i].clone(), 1e-5
            t[i] = old + step
            up = loss()
            t[i] = old - step
            down = loss()
            t[i] = old
            # differences: truncation of order step^2, rounding of a sum of a thousand values over the step
            assert abs((up - down) / (2 * step) - float(g[i])) < 1e-6 * (1 + abs(float(g[i]))), (name, i)


def test_a_layer_of_them_is_trained_with_clipping_and_the_same_bits_come_again():
    from deepbind_amd import deepity_smat as ds
    P, X, dY = layer_case("float32", 700, 4, 2, 16, 16, 22)
    R = regions([[300, 700], [0, 130], [130, 300]])
    runs = []
    for _ in range(2):
        Z, g = layer(P, X, R, 2, dY)
        trained = [g[k] for k in ("gamma", "scale", "next")]
        before = [t.clone() for t in trained]
        norm = ds.clip_gradients(trained, 0.25)
        for a, b in zip(trained, before):
            assert float((a - b * min(1.0, 0.25 / float(norm))).abs().max()) <= 1e-6 * float(b.abs().max())
        runs.append([Z, norm] + [g[k].clone() for k in sorted(g)])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
def test_captured_layers_replay_on_new_inputs_and_streams_do_not_meet(kind):
    from deepbind_amd import deepity_smat as ds
    P, X, dY = layer_case(kind, 260, 2, 1, 40, 24, 23)
    R = regions([[0, 200], [200, 260]])

    def everything():
        Z, g = layer(P, X, R, 1, dY)
        out = [torch.empty_like(g[k]) for k in ("gamma", "scale", "next", "V")]
        norm = ds.clip_gradients([g[k] for k in ("gamma", "scale", "next", "V")], 0.1, out=out)
        return [Z, norm] + [g[k] for k in sorted(g)] + out

    eager = [t.clone() for t in everything()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = everything()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, eager):
        assert torch.equal(a, b)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = everything()
        graphs.append((graph, held))
    for turn in range(3):
        new, Xn, dn = layer_case(kind, 260, 2, 1, 40, 24, 30 + turn)
        for k in P:
            P[k].copy_(new[k])
        X.copy_(Xn)
        dY.copy_(dn)
        want = [t.clone() for t in everything()]
        torch.cuda.synchronize()
        for graph, held in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for graph, held in graphs:
            for a, b in zip(held, want):
                assert torch.equal(a, b)


def test_outputs_on_inputs_and_other_devices_are_refused():
    from deepbind_amd import kangaroo_smat as ks
    from deepbind_amd import smat as sm
    from deepbind_amd._lib import DeepbindError
    X, b, R = torch.zeros(9, 12, device="cuda"), torch.zeros(9, 2, device="cuda"), regions([[0, 9]])
    state = torch.zeros(9, 6, 12, device="cuda")
    for f in (lambda: ks.deltarule(X, X, X, b, R, out=X), lambda: ks.deltarule_step(X, X, X, b, state, out=X), lambda: ks.deltarule_step(X, X, X, b, state, into=state[:]),
              lambda: sm.blocknorm(X, out=(X, None)), lambda: sm.blocknorm(X, out=(None, X)),
              lambda: ks.deltarule_bprop(X, X, X, b, R, ks.kept_delta(X, X, b), X, out=(None, None, None, b, None))):
        with pytest.raises(DeepbindError, match="shares memory"):
            f()
    with pytest.raises(DeepbindError, match="expected a device tensor"):
        ks.deltarule(X, X.cpu(), X, b, R)
