"""The row operators at values and sizes where they can go wrong: rows far from zero, infinities, states that grow or overflow, regions just
beyond the length that is cut, many states beside narrow groups. Tolerances as in test_rows_gpu; those of the scan come row by row from rows_bounds."""
import numpy as np
import pytest
import torch

from tests import rows_bounds, rows_ref as ref
from tests.gpu_util import host
from tests.test_rows_gpu import STORED, TYPES, U, inside, put, regions, wide

pytestmark = pytest.mark.gpu

NAMES = ("dX", "ddt", "dA", "dB", "dC", "dD", "dgate", "ddt_bias")


def near(got, want, bound, kind, what, rows=None, stored=False):
    """got against want: the same NaN and infinities, finite values within bound u (1.01: products of errors)."""
    got = host(got.double())
    if rows is not None:
        got, want, bound = got[rows], want[rows], bound[rows]
    assert got.shape == want.shape, what
    assert np.array_equal(np.isnan(got), np.isnan(want)), "%s: NaN at %s instead of %s" % (what, np.argwhere(np.isnan(got))[:4].tolist(), np.argwhere(np.isnan(want))[:4].tolist())
    inf = np.isinf(want)
    assert np.array_equal(np.isinf(got), inf) and np.array_equal(got[inf], want[inf]), "%s: other infinities" % what
    ok = np.isfinite(want)
    got, want, bound = got[ok], want[ok], np.where(np.isnan(bound), np.inf, bound)[ok]
    bound = 1.01 * U[kind] * bound + (STORED[kind] if stored else U[kind]) * np.abs(want) + 1e-35
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), "%s: %d of %d values off, worst %.3g of the bound" % (what, bad.sum(), bad.size, (np.abs(got - want) / bound).max())


def scan(kind, v, R, N, what, rows=None, soft=True, state=False, grads=True, segment=0, only=NAMES):
    """Forward, and backward from zero states, on the values v against the definition."""
    from deepbind_amd import kangaroo_smat as ks
    rows = inside(R, N) if rows is None else rows
    t = {}
    for n, a in v.items():
        t[n], v[n] = (None, None) if a is None else put(a, TYPES[kind] if n in ("X", "dt", "gate", "dY") else wide(kind))
    T = regions(np.asarray(R).reshape(-1, 2))
    D = v["A"].shape[1]
    kw = dict(D=t["D"], gate=t["gate"], dt_bias=t["bias"], softplus=soft)
    base = [t[n] for n in ("X", "dt", "A", "B", "C")]
    zero = np.zeros((1, D))
    args = [v[n] for n in ("X", "dt", "A", "B", "C")] + [R, zero if v["D"] is None else v["D"], v["gate"], zero if v["bias"] is None else v["bias"], soft]
    with np.errstate(all="ignore"):
        if state:
            Y, last = ks.statescan(*base, T, state=t["state"], want_state=True, **kw)
            (want, wl), _ = ref.statescan(*args, state=v["state"])
            bound, bl = rows_bounds.statescan(*args, state=v["state"], segment=segment)
            near(Y, want, bound, kind, what + ": Y from a state", rows, stored=True)
            near(last, wl, bl, kind, what + ": last from a state")
        keep = ks.kept_states(t["X"], t["A"]) if grads else None
        Y, last = ks.statescan(*base, T, keep=keep, want_state=True, **kw)
        want = ref.statescan(*args, dY=v["dY"] if grads else None)[0]
        bound = rows_bounds.statescan(*args, dY=v["dY"] if grads else None, segment=segment)
    near(Y, want[0], bound[0], kind, what + ": Y", rows, stored=True)
    near(last, want[1], bound[1], kind, what + ": last")
    if grads:
        got = ks.statescan_bprop(*base, T, keep, t["dY"], **kw)
        for name, g, w, b in zip(NAMES, got, want[2:], bound[2:]):
            if g is not None and name in only:
                per_row = name in ("dX", "ddt", "dB", "dC", "dgate")
                near(g, w, b, kind, "%s: %s" % (what, name), rows if per_row else None, stored=name in ("dX", "ddt", "dgate"))


def values(rng, N, P, D, G, S, gate=True):
    f = lambda *s: rng.standard_normal(s)  # noqa: E731
    return dict(X=f(N, D), dt=f(N, D), A=-np.exp(f(S, D)), B=f(N, G * S), C=f(N, G * S), D=f(1, D), gate=f(N, D) if gate else None, bias=f(1, D) - 2,
                state=f(P, S, D), dY=f(N, D))


# ------------------------------------------------------------------------------------------------ state scan
RAGGED = [[30, 61], [0, 1], [1, 3], [70, 70], [3, 30], [61, 64]]
CUTS = [[0, 128], [128, 257], [260, 420], [420, 581], [581, 582]]               # one not cut, one whose last segment is a row, five whole segments, one more row


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D,G,S", [(24, 2, 16), (48, 2, 33), (130, 2, 64), (12, 4, 17), (70, 1, 16)])
def test_statescan_of_regions_around_the_length_that_is_cut(kind, D, G, S):
    rng = np.random.default_rng([D, G, S])
    scan(kind, values(rng, 590, len(CUTS), D, G, S), CUTS, 590, "cut", state=True, segment=32)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("D,G,S", [(24, 2, 33), (64, 2, 64), (12, 4, 17), (90, 3, 20), (20, 5, 64)])
def test_statescan_of_many_states_beside_narrow_groups(kind, D, G, S):
    rng = np.random.default_rng([D, G, S])
    scan(kind, values(rng, 75, len(RAGGED), D, G, S, gate=S != 20), RAGGED, 75, "narrow", state=True)


@pytest.mark.parametrize("kind", ["float32", "bfloat16"])
@pytest.mark.parametrize("D,G,S", [(40, 2, 16), (65, 1, 7)])
def test_statescan_of_long_regions_is_as_near_as_the_decays_remember(kind, D, G, S):
    rng = np.random.default_rng([D, S])
    R = [[2000, 9001], [3, 1300], [1300, 1301]]
    v = values(rng, 9010, len(R), D, G, S)
    v["A"] = -np.exp(1.5 * np.log(-v["A"]))      # some forget in a row, some remember a thousand
    scan(kind, v, R, 9010, "long", segment=32)


def test_statescan_gradient_of_very_many_groups():
    """1024 groups of 65 channels and 64 states: a region's dB and dC are more than the workgroups of one launch take 1024 of each."""
    from deepbind_amd import kangaroo_smat as ks
    G, gs, S, N = 1024, 65, 64, 520
    D = G * gs
    g = torch.Generator(device="cuda").manual_seed(5)
    f = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    X, dt, dY, A, B, C = f(N, D), f(N, D), f(N, D), -f(S, D).abs(), f(N, G * S), f(N, G * S)
    T = regions([[i * 104, i * 104 + 104] for i in range(5)])                   # (short enough not to be cut, in either call)
    keep = ks.kept_states(X, A)
    Y, _ = ks.statescan(X, dt, A, B, C, T, keep=keep)
    got = ks.statescan_bprop(X, dt, A, B, C, T, keep, dY)
    for i in (0, 517, G - 1):
        c, w = slice(i * gs, (i + 1) * gs), slice(i * S, (i + 1) * S)
        one = [X[:, c], dt[:, c], A[:, c].contiguous(), B[:, w], C[:, w]]
        k1 = ks.kept_states(one[0], one[2])
        y1, _ = ks.statescan(*one, T, keep=k1)
        want = ks.statescan_bprop(*one, T, k1, dY[:, c])
        assert torch.equal(Y[:, c], y1)
        for name, a, b in zip(NAMES, got, want):
            if b is not None:
                near = a[:, w] if name in ("dB", "dC") else a[:, c]
                # (dA is added over another number of workgroups; the rest are the same operations)
                assert torch.equal(near, b) if name != "dA" else float((near - b).abs().max()) <= 1e-5 * float(b.abs().max()), (i, name)


# ------------------------------------------------------------------------------------------------ layer norm
def _depth(w, kind):
    """The most roundings on a value's way through a chunk's sum: one thread's values (at most 16 in registers; from 256 threads' vectors on, where the
    chunk is wider), then 256 threads in pairs."""
    per = {"float32": 4, "float64": 2, "bfloat16": 8}[kind]
    return max(4 * per, w // 256 + per) + 8


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("nchunk,w", [(1, 7), (5, 12), (3, 24), (1, 100), (2, 1440), (1, 20001), (9, 16)])
def test_layernorm_of_rows_of_one_value(kind, nchunk, w):
    """A chunk of identical values lies on its mean: its rows are beta, and the deviation is that of eps alone."""
    from deepbind_amd import smat as sm
    rng = np.random.default_rng([w, nchunk])
    n, eps = 61, 1e-5
    X, x = put(np.repeat(10 ** rng.uniform(-1, 5, (n, nchunk)) * rng.choice([-1, 1], (n, nchunk)), w, 1), TYPES[kind])
    g, gv = put(1 + 0.3 * rng.standard_normal((1, nchunk * w)), wide(kind))
    b, bv = put(0.3 * rng.standard_normal((1, nchunk * w)), wide(kind))
    Z, stats = sm.layernorm(X, g, b, nchunk=nchunk, eps=eps, want_stats=True)
    assert torch.equal(Z, b.to(TYPES[kind]).expand_as(Z))
    assert torch.equal(stats[0].view(n, nchunk), X[:, ::w].to(wide(kind)))
    # the first mean is off by e <= k u |x|; the mean of its squares less the square of their mean by (k + 4) u e^2 of eps
    k = _depth(w, kind) + 2
    e = k * U[kind] * np.abs(x[:, ::w])
    r = host(stats[1].double()).reshape(n, nchunk)
    assert (np.abs(r * np.sqrt(eps) - 1) <= 4 * U[kind] + (k + 4) * U[kind] * e * e / (2 * eps)).all()
    dX, dg, db = sm.layernorm_bprop(X, g, stats, torch.ones_like(X), nchunk=nchunk)
    assert not dg.any() and torch.equal(db, torch.full_like(db, n))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("nchunk,w", [(1, 7), (5, 12), (4, 16), (3, 100), (1, 1440), (1, 20001)])
@pytest.mark.parametrize("offset", [30.0, 1e4])
def test_layernorm_of_rows_far_from_zero(kind, nchunk, w, offset):
    from deepbind_amd import smat as sm
    rng = np.random.default_rng([w, nchunk, int(offset)])
    n, eps, u = 200 if w < 2000 else 20, 1e-5, U[kind]
    X, x = put(rng.standard_normal((n, nchunk * w)) + offset * rng.choice([-1, 1], (n, 1)), TYPES[kind])
    g, gv = put(1 + 0.3 * rng.standard_normal((1, nchunk * w)), wide(kind))
    Z, stats = sm.layernorm(X, g, None, nchunk=nchunk, eps=eps, want_stats=True)
    V = x.reshape(n, nchunk, w).astype(np.longdouble)        # (64 bits would round the mean as the kernel does)
    mean = V.mean(2, keepdims=True)
    c = V - mean
    var = (c * c).mean(2, keepdims=True)
    r = 1 / np.sqrt(var + eps)
    # the first mean is off by e; the mean of what is left corrects it up to its own rounding, u |mean|, and that of a sum of numbers of the deviation's size
    k = _depth(w, kind) + 4
    e = k * u * np.abs(V).mean(2, keepdims=True)
    spread = np.abs(c).mean(2, keepdims=True) + e
    dmean = u * np.abs(mean) + k * u * spread
    drel = 4 * u + (k + 4) * u * (var + 2 * e * e) / (2 * (var + eps))          # of the deviation's reciprocal
    assert (np.abs(host(stats[0].double()).reshape(mean.shape) - mean) <= dmean).all()
    assert (np.abs(host(stats[1].double()).reshape(mean.shape) / r - 1) <= drel).all()
    bound = np.abs(gv) * (r * (dmean + u * np.abs(c)) + np.abs(c) * r * (drel + 2 * u)).reshape(n, -1)
    want = (c * r).reshape(n, -1) * gv
    assert (np.abs(host(Z.double()) - want) <= 1.01 * bound + STORED[kind] * (np.abs(want) + bound)).all()
@pytest.mark.parametrize("kind", ["float32", "float64"])
@pytest.mark.parametrize("S", [1, 5, 16, 17, 33])
@pytest.mark.parametrize("D,G", [(5, 1), (70, 1), (24, 2)])
@pytest.mark.parametrize("one_sign", [False, True])
def test_statescan_forward_of_an_infinite_input(kind, S, D, G, one_sign):
    """A state takes an infinite input in and stays infinite; the row's other values, later rows' and other channels' are what the definition makes of it."""
    rng = np.random.default_rng([S, D, G])
    v = values(rng, 75, len(RAGGED), D, G, S)
    v["A"] = np.maximum(v["A"], -3)              # (no decay underflows: 0 * inf would be another definition's)
    if one_sign:                                 # (sums of infinities of both signs would be NaN in either way)
        v["B"], v["C"], v["D"] = np.abs(v["B"]), np.abs(v["C"]), np.abs(v["D"])
    v["X"][40, 3], v["X"][2, 0], v["X"][10, D - 1] = np.inf, -np.inf, np.inf
    scan(kind, v, RAGGED, 75, "S=%d" % S, grads=False, state=True)


@pytest.mark.parametrize("kind", ["float32", "float64"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("S", [1, 5, 16, 17])
@pytest.mark.parametrize("one_sign", [False, True])
def test_statescan_gradients_of_an_infinite_input(kind, gated, S, one_sign):
    """Where the number of states is no multiple of four: those that do not exist add nothing, whatever the others hold."""
    for name, worst in (("X", np.inf), ("dY", -np.inf)):
        rng = np.random.default_rng([S, gated])
        v = values(rng, 75, len(RAGGED), 64, 1, S, gated)
        v["A"] = np.maximum(v["A"], -3)
        if one_sign:
            v["B"], v["C"], v["D"], v["dY"] = np.abs(v["B"]), np.abs(v["C"]), np.abs(v["D"]), np.abs(v["dY"])
        v[name][40, 3], v[name][10, 7] = np.inf, worst
        scan(kind, v, RAGGED, 75, "%s, S=%d" % (name, S))


@pytest.mark.parametrize("kind", ["float32", "float64"])
@pytest.mark.parametrize("name", ["X", "dt", "dY", "gate"])
@pytest.mark.parametrize("D,G", [(5, 1), (70, 1), (24, 2), (40, 2)])
def test_statescan_gradients_of_an_infinite_last_channel(kind, name, D, G):
    """A group that does not fill its lanes: the lanes without a channel add nothing to the group's sums, whatever its last channel holds."""
    rng = np.random.default_rng([D, G, ord(name[0])])
    v = values(rng, 75, len(RAGGED), D, G, 16)
    v["A"] = np.maximum(v["A"], -3)
    v[name][12, D // G - 1], v[name][36, D - 1] = np.inf, np.inf
    scan(kind, v, RAGGED, 75, name)


@pytest.mark.parametrize("kind", ["float32", "float64"])
def test_statescan_whose_states_grow(kind):
    """A > 0 and steps as they are, in a region that is cut: nothing carried on over a segment whose growth overflows stays nothing, something small
    becomes what it becomes row by row."""
    P, N, D, S = [[3, 400]], 405, 3, 5
    rng = np.random.default_rng(8)

    def case():
        v = values(rng, N, 1, D, 1, S, gate=False)
        v["A"], v["bias"] = 2 + rng.random((S, D)), None
        return v

    big = 8 if kind == "float64" else 1          # (2^1024 is eight times 2^128)
    v = case()
    v["dt"][:] = big
    v["A"] *= 2                                  # e^(4 * 32) and more in a segment of 32 rows
    v["X"][:393], v["dY"][8:] = 0, 0             # inputs in the last rows, gradients from the first
    scan(kind, v, P, N, "zeros", soft=False, segment=32)
    v = case()
    v["dt"][:], v["A"][:] = 0, 4 * big
    v["dt"][8], v["dt"][3 + 32:3 + 64] = 1, 1    # into the first segment, through the second
    v["X"][:], v["X"][8] = 0, 1e-25 ** big * rng.standard_normal(D)
    v["D"] *= 0
    scan(kind, v, P, N, "small", soft=False, grads=False, segment=32)
    v = case()
    v["dt"][:], v["A"][:] = 0, 4 * big
    v["dt"][8], v["dt"][3 + 32:3 + 64] = 1, 1
    v["X"][:], v["dY"][:] = 0, 0
    v["dY"][80] = 1e-25 ** big
    scan(kind, v, P, N, "small gradient", soft=False, segment=32)


@pytest.mark.parametrize("kind", ["float32", "float64"])
@pytest.mark.parametrize("name", ["X", "dY"])
def test_statescan_of_an_infinite_state_that_is_carried(kind, name):
    """An infinite state stays infinite, also over segments whose decay underflows."""
    rng = np.random.default_rng(12)
    v = values(rng, 405, 1, 6, 1, 4)
    v["A"] = -1 - 6 * rng.random((4, 6))
    if kind == "float64":
        v["A"] *= 4
    v["dt"][:] = 2
    v["bias"] = np.zeros((1, 6))
    v[name][20 if name == "X" else 380, 2] = np.inf
    scan(kind, v, [[3, 400]], 405, name, segment=32, only=("dX", "dB", "dC"))


def test_statescan_gradient_of_many_regions_of_a_wide_group():
    """Groups of 130 channels, whose tiles' shares of dB and dC are added: thousands of short regions, and one just under the length that is cut."""
    rng = np.random.default_rng(19)
    lens = np.concatenate([rng.integers(0, 4, 3000), [120], rng.integers(0, 4, 500)])
    starts = np.cumsum(np.concatenate([[0], lens[:-1]]))
    R = np.stack([starts, starts + lens], 1)[rng.permutation(len(lens))].tolist()
    N = int(lens.sum()) + 5
    scan("float32", values(rng, N, len(R), 260, 2, 6), R, N, "many", segment=32)
