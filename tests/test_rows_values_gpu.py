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
