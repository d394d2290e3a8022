"""The gated delta rule, the norms around a block and clipping at values where they can go wrong: states that grow or vanish over the segments of long
regions, resets, infinities and undefined values there, bad rows in wide chunks, factors beyond a float's range. Tolerances as in test_blocks_gpu."""
import numpy as np
import pytest
import torch

from tests import blocks_ref as ref
from tests.gpu_util import host
from tests.test_blocks_gpu import delta_case
from tests.test_rows_gpu import STORED, TYPES, U, inside, put, regions, wide

pytestmark = pytest.mark.gpu

GRADS = ("dQ", "dK", "dV", "dbeta", "ddecay")
LONG = [[1030, 1100], [0, 1030]]                 # one not cut, one of four whole segments of 256 rows and a short one
SEGMENT = 256


def near(got, want, bound, kind, what, rows, stored=True, least=1e-35):
    """Within the bound, the stored type's rounding and `least`, which is what falls below the type's range."""
    got = host(got.double())
    got, want, bound = (got, want, bound) if rows is None else (got[rows], want[rows], bound[rows])
    assert got.shape == want.shape and np.isfinite(want).all(), what
    bound = 1.01 * U[kind] * bound + (STORED[kind] if stored else U[kind]) * np.abs(want) + least
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), "%s: %d of %d values off at rows %s, worst %.3g of the bound" % (what, bad.sum(), bad.size, np.unique(np.argwhere(bad)[:, 0])[:5].tolist(),
                                                                                          (np.abs(got - want) / bound).max())


def delta_as_by_rows(kind, t, v, R, G, Kd, what, least=1e-35, grads=True, state=None):
    """Forward, and backward from zero states, against the definition."""
    from deepbind_amd import kangaroo_smat as ks
    N = v["beta"].shape[0]
    T, rows = regions(R), inside(R, N)
    args = (t["Q"], t["K"], t["V"], t["beta"], T)
    kw = dict(decay=t["decay"], groups=G)
    plain = (v["Q"], v["K"], v["V"], v["beta"], v["decay"], R, G, Kd ** -0.5)
    with np.errstate(all="ignore"):
        want = ref.delta(*plain, dO=v["dO"] if grads else None, state=None if state is None else state[1])
        bound = ref.delta_bounds(*plain, dO=v["dO"] if grads else None, state=None if state is None else state[1], segment=SEGMENT)
    keep = ks.kept_delta(t["K"], t["V"], t["beta"], groups=G) if grads else None
    O, last = ks.deltarule(*args, keep=keep, want_state=True, state=None if state is None else state[0], **kw)
    near(O, want[0], bound[0], kind, what + ": O", rows, least=least)
    near(last, want[1], bound[1], kind, what + ": last", None, stored=False, least=least)
    if grads:
        for name, g, w, b in zip(GRADS, ks.deltarule_bprop(*args, keep, t["dO"], **kw), want[2:], bound[2:]):
            if g is not None:
                near(g, w, b, kind, "%s: %s" % (what, name), rows, stored=name in GRADS[:3], least=least)


def changed(t, v, name, rows, value, cols=slice(None)):
    """Rows of a map set to a value, or multiplied by it (a factor in a tuple), on the device and in the plain form."""
    t[name][rows, cols] = t[name][rows, cols] * value[0] if isinstance(value, tuple) else value
    v[name] = t[name].double().cpu().numpy()


SHAPES = [(2, 1, 16, 16), (2, 2, 40, 33), (1, 1, 128, 70), (3, 1, 20, 5)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("H,G,Kd,Vd", SHAPES)
def test_delta_rule_of_segments_whose_states_grow_and_vanish(kind, H, G, Kd, Vd):
    """A segment of a long region may grow or shrink a state by more than the type's range: what is nothing in front of it stays nothing, what is small
    or large becomes what it becomes row by row."""
    N = 1100
    big = 8 if kind == "float64" else 1          # (2^1024 is eight times 2^128)
    rate = 0.36 * big                            # e^92 in a segment of 256 rows; 16 rows stay far within the range
    case = lambda: delta_case(kind, N, H, G, Kd, Vd, True, 0, [H, Kd, Vd])  # noqa: E731
    t, v = case()
    changed(t, v, "beta", slice(0, 520), 0.0)
    changed(t, v, "decay", slice(0, 520), rate)
    delta_as_by_rows(kind, t, v, LONG, G, Kd, "nothing in front", grads=False)
    t, v = case()
    changed(t, v, "decay", slice(520, 521), -1e4)
    changed(t, v, "beta", slice(520, 1030), 0.0)
    changed(t, v, "decay", slice(521, 1030), rate)
    changed(t, v, "dO", slice(520, 1030), 0.0)
    delta_as_by_rows(kind, t, v, LONG, G, Kd, "no gradient behind")
    if kind == "float64":                        # (the bounds' norms square what is over 1e160 then)
        return
    for first, second, value, grad in ((rate, -rate, 1e-20, 1e-10), (-rate, rate, 1e15, 1e-15)):
        t, v = case()
        changed(t, v, "beta", slice(256, 768), (0.02,))
        changed(t, v, "decay", slice(256, 512), first)
        changed(t, v, "decay", slice(512, 768), second)
        changed(t, v, "V", slice(0, N), (value,))
        if first < 0:
            changed(t, v, "V", slice(256, 768), (1e-38,))                      # (1e-23: the growth behind makes it 1e17)
        changed(t, v, "dO", slice(0, N), (grad,))
        delta_as_by_rows(kind, t, v, LONG, G, Kd, "up and down" if first > 0 else "down and up")


def test_delta_rule_in_double_of_segments_whose_states_grow_and_vanish_is_that_of_shorter_pieces():
    from deepbind_amd import kangaroo_smat as ks
    N, H, Kd, Vd = 1030, 2, 40, 20
    for first, value in ((2.88, 1e-160), (-2.88, 1e120)):
        t, v = delta_case("float64", N, H, 1, Kd, Vd, True, 0, 31)
        changed(t, v, "beta", slice(256, 768), (0.02,))
        changed(t, v, "decay", slice(256, 512), first)
        changed(t, v, "decay", slice(512, 768), -first)
        changed(t, v, "V", slice(0, N), (value,))
        if first < 0:
            changed(t, v, "V", slice(256, 768), (1e-300,))
        call = lambda a, b, **kw: ks.deltarule(t["Q"][a:b], t["K"][a:b], t["V"][a:b], t["beta"][a:b], regions([[0, b - a]]), decay=t["decay"][a:b], groups=1, want_state=True, **kw)  # noqa: E731
        O, last = call(0, N)
        parts, state = [], None
        for a in range(0, N, 128):
            o, state = call(a, min(a + 128, N), state=state)
            parts.append(o)
        # both are off by at most what the bounds of the float32 cases above come to in units of their values, some 12 000
        for got, want in ((O, torch.cat(parts)), (last.view(Kd, -1), state.view(Kd, -1))):
            assert got.isfinite().all()
            assert float(((got - want).abs().amax(1) / want.abs().amax(1)).max()) < 2 * 12000 * 2.0 ** -53


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("H,G,Kd,Vd,R,rows", [(2, 1, 20, 24, [[0, 100], [100, 150]], (37, 99)), (3, 3, 16, 16, [[0, 100], [100, 150]], (37, 140)),
                                              (2, 2, 40, 20, LONG, (37, 300, 511, 512, 1029)), (2, 1, 128, 20, LONG, (300, 700))])
def test_delta_rule_carries_what_is_not_finite_exactly_as_far_as_the_formulas(kind, H, G, Kd, Vd, R, rows):
    """One value that is not finite, anywhere: what the row by row formulas, forward and backward, keep finite is the same bits as without it, and what they
    do not keep finite is not."""
    from deepbind_amd import kangaroo_smat as ks
    N = max(e for _, e in R)
    t, v = delta_case(kind, N, H, G, Kd, Vd, True, 0, 12)
    args = (t["Q"], t["K"], t["V"], t["beta"], regions(R))
    kw = dict(decay=t["decay"], groups=G)
    keep = ks.kept_delta(t["K"], t["V"], t["beta"], groups=G)

    def both():
        O, last = ks.deltarule(*args, keep=keep, want_state=True, **kw)
        return (O, last) + ks.deltarule_bprop(*args, keep, t["dO"], **kw)

    good = both()
    for row in rows:
        for name in ("V", "Q", "K", "beta", "decay", "dO"):
            for bad in (float("nan"), float("inf")):
                x, col = t[name], min(5, t[name].shape[1] - 1)
                old = x[row, col].clone()
                x[row, col] = bad
                got = both()
                x[row, col] = old
                w = {k: a.copy() if k == name else a for k, a in v.items()}
                w[name][row, col] = bad
                with np.errstate(all="ignore"):
                    want = ref.delta(w["Q"], w["K"], w["V"], w["beta"], w["decay"], R, G, Kd ** -0.5, dO=w["dO"])
                for what, g, clean, wanted in zip(("O", "last") + GRADS, got, good, want):
                    keeps = torch.from_numpy(np.isfinite(wanted)).cuda()
                    same = g == clean
                    assert bool(same[keeps].all()), "%s[%d] = %s: %s changes at rows %s" % (name, row, bad, what, np.unique(np.argwhere(host(keeps & ~same))[:, 0]).tolist()[:20])
                    left = g.isfinite() & ~keeps
                    assert not bool(left.any()), "%s[%d] = %s: %s is finite at rows %s" % (name, row, bad, what, np.unique(np.argwhere(host(left))[:, 0]).tolist()[:20])


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("one", [True, False])
@pytest.mark.parametrize("H,G,Kd,Vd,R,at", [(2, 1, 16, 16, [[0, 100], [100, 150]], 0), (4, 2, 16, 20, [[0, 100], [100, 150]], 0), (5, 5, 7, 40, [[50, 150], [0, 50]], 50),
                                            (2, 2, 40, 33, LONG, 480), (2, 1, 128, 70, [[0, 130]], 0), (3, 1, 20, 20, LONG, 240)])
def test_delta_rule_whose_factors_within_a_chunk_leave_the_range(kind, one, H, G, Kd, Vd, R, at):
    """Sixteen rows may grow or shrink a state by more than the type's range, by their decays (of one head, or of all) or by keys longer than one, where the
    rows by themselves find nothing to grow, or something small."""
    N = max(e for _, e in R)
    rate = 40.0 if kind == "float64" else 7.5    # e^640 and e^120 in a chunk: more than its matrices are let hold, and in single precision than they can
    heads = slice(0, 1) if one else slice(0, H)
    end = max(e for s, e in R if s <= at < e)
    case = lambda: delta_case(kind, N, H, G, Kd, Vd, True, 0, [H, Kd, Vd])  # noqa: E731
    rows = lambda a, b: slice(at + a, at + b)  # noqa: E731
    t, v = case()
    start = max(s for s, e in R if s <= at < e)
    changed(t, v, "beta", slice(start, at + 40), 0.0, heads)
    changed(t, v, "decay", slice(start, at + 40), rate, heads)
    delta_as_by_rows(kind, t, v, R, G, Kd, "nothing in front", grads=False)
    t, v = case()
    changed(t, v, "decay", rows(50, 51), -1e4, heads)
    changed(t, v, "beta", slice(at + 50, end), 0.0, heads)
    changed(t, v, "decay", slice(at + 51, end), rate, heads)
    changed(t, v, "dO", slice(at + 50, end), 0.0, slice(0, (heads.stop - heads.start) * Vd))
    delta_as_by_rows(kind, t, v, R, G, Kd, "no gradient behind")
    if kind == "float64":                        # (the bounds' norms square what is over 1e160 then, and keys would have to be 1e10 long)
        return
    for first, value, between, grad in ((rate, 1e-25, 1.0, 1e-15), (-rate, 1e18, 1e-38, 1e-18)):
        t, v = case()
        changed(t, v, "beta", rows(33, 61), (0.02,), heads)
        changed(t, v, "decay", rows(33, 47), first, heads)
        changed(t, v, "decay", rows(47, 61), -first, heads)
        cols = slice(0, (heads.stop - heads.start) * Vd)
        changed(t, v, "V", slice(0, N), (value,), cols)
        changed(t, v, "V", rows(33, 61), (between,), cols)
        changed(t, v, "dO", slice(0, N), (grad,), cols)
        # (heads that share a key add their gradients of it: the others' are no smaller than these)
        delta_as_by_rows(kind, t, v, R, G, Kd, "up and down" if first > 0 else "down and up")
    # (long keys that find nothing, and send nothing back, change nothing: the plain form goes without them)
    t, v = case()
    changed(t, v, "V", slice(start, at + 31), 0.0)
    changed(t, v, "beta", rows(10, 31), 1.0)
    t["K"][rows(10, 31)] *= 100.0
    delta_as_by_rows(kind, t, v, R, G, Kd, "long keys, nothing in front", grads=False)
    t, v = case()
    changed(t, v, "decay", rows(45, 46), -1e4)
    changed(t, v, "V", slice(at + 45, end), 0.0)
    changed(t, v, "beta", slice(at + 47, end), 1.0)
    changed(t, v, "dO", slice(at + 45, end), 0.0)
    t["K"][at + 47:end] *= 100.0
    delta_as_by_rows(kind, t, v, R, G, Kd, "long keys, no gradient behind")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("H,G,Kd,Vd", SHAPES)
def test_delta_rule_with_resets_and_large_steps_over_segments(kind, H, G, Kd, Vd):
    """Hard resets at, before and behind the borders of segments, rows that learn nothing and rows that turn what they find around; minus infinity resets too."""
    t, v = delta_case(kind, 1100, H, G, Kd, Vd, True, 0, [H, Kd])
    for name, rows, value in (("decay", [20, 255, 256, 511, 700, 1029, 1030], -1e4), ("decay", [300, 769], -60.0), ("beta", [3, 257, 512], 0.0), ("beta", [60, 61, 510, 768, 1050], 2.0),
                              ("decay", [33, 257], 0.0)):
        changed(t, v, name, rows, value)
    delta_as_by_rows(kind, t, v, LONG, G, Kd, "resets")
    state = put(np.random.default_rng(3).standard_normal((2, Kd, H * Vd)), wide(kind))
    delta_as_by_rows(kind, t, v, LONG, G, Kd, "from a state", grads=False, state=state)
    changed(t, v, "decay", [255, 700], -float("inf"))
    # (the bounds' running products go without it; what it leaves is what -1e4 leaves)
    v["decay"][[255, 700]] = -1e4
    delta_as_by_rows(kind, t, v, LONG, G, Kd, "minus infinity")


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("H,G,Kd,Vd,R", [(4, 2, 40, 130, [[30, 100], [0, 30], [100, 101]]), (4, 2, 128, 130, [[300, 1068], [0, 256], [256, 300]]), (6, 2, 16, 70, [[0, 600]]),
                                        (2, 1, 100, 129, [[5, 700]])])
def test_delta_rule_of_shared_heads_with_values_in_parts(kind, H, G, Kd, Vd, R):
    """Gradients of a key that heads share, each of whose values takes several teams of waves."""
    N = max(e for _, e in R) + 3
    t, v = delta_case(kind, N, H, G, Kd, Vd, True, 1, [H, Kd, Vd])
    delta_as_by_rows(kind, t, v, R, G, Kd, "shared")


def test_delta_rule_on_two_streams_at_once():
    """Calls with everything in their scratch (segments, transitions, carried states, heads' shares, marked heads) in flight on two streams, on their own data each."""
    from deepbind_amd import kangaroo_smat as ks
    R, sides = regions([[0, 3000], [3000, 3300]]), []
    for seed in (41, 42):
        t, _ = delta_case("bfloat16" if seed == 41 else "float32", 3300, 4, 2, 64, 80, True, 0, seed)
        if seed == 42:
            t["beta"][3000:3050, 0], t["decay"][3000:3050, 0] = 0.0, 8.0
        sides.append(t)

    def both(t):
        kw = dict(decay=t["decay"], groups=2)
        keep = ks.kept_delta(t["K"], t["V"], t["beta"], groups=2)
        O, last = ks.deltarule(t["Q"], t["K"], t["V"], t["beta"], R, keep=keep, want_state=True, **kw)
        return (O, last) + ks.deltarule_bprop(t["Q"], t["K"], t["V"], t["beta"], R, keep, t["dO"], **kw)

    want = [both(t) for t in sides]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(4):
        for t, s in zip(sides, streams):
            with torch.cuda.stream(s):
                got.append(both(t))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        # (the marked head's gradients grow by e^400 over its fifty rows, beyond the range, by the formulas too)
        for a, b in zip(g, want[i % 2]):
            assert bool(((a == b) | (a.isnan() & b.isnan())).all())
        assert g[0].isfinite().all() and g[1].isfinite().all()


def test_captured_delta_rule_keeps_no_marks_from_one_replay_to_the_next():
    """Ordinary rows, rows whose states grow over a segment, rows that leave the range within a chunk, in turn through the same captured call and the same kept buffer."""
    from deepbind_amd import kangaroo_smat as ks
    H, Kd, Vd, N = 3, 20, 20, 1100
    t, v = delta_case("float32", N, H, 1, Kd, Vd, True, 0, 51)
    plain = {k: x.clone() for k, x in t.items()}
    R = regions(LONG)
    keep = ks.kept_delta(t["K"], t["V"], t["beta"], groups=1)

    def both(keep):
        kw = dict(decay=t["decay"], groups=1)
        O, last = ks.deltarule(t["Q"], t["K"], t["V"], t["beta"], R, keep=keep, want_state=True, **kw)
        return (O, last) + ks.deltarule_bprop(t["Q"], t["K"], t["V"], t["beta"], R, keep, t["dO"], **kw)

    both(keep)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(keep)
    for turn in (0, 1, 0, 2, 1, 2, 0):
        for k, x in plain.items():
            t[k].copy_(x)
        if turn == 1:
            t["decay"][520, 1], t["decay"][521:1030, 1] = -1e4, 0.36
        elif turn == 2:
            t["decay"][520, 0], t["decay"][521:560, 0] = -1e4, 7.5
        if turn:
            t["beta"][520:1030], t["dO"][520:1030] = 0.0, 0.0
        graph.replay()
        torch.cuda.synchronize()
        want = both(torch.full_like(keep, float("nan")))
        for a, b in zip(held, want):
            assert b.isfinite().all() and torch.equal(a, b), turn


# ------------------------------------------------------------------------------------------------ norms around a block
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rms", [True, False])
@pytest.mark.parametrize("n,nchunk,w", [(50, 3, 16), (50, 2, 5), (2300, 1, 300), (700, 2, 700), (600, 1, 1440), (560, 1, 2500), (530, 1, 5000), (520, 2, 9001)])
def test_block_norms_and_their_gradients_keep_a_bad_row_to_its_chunk(kind, rms, n, nchunk, w):
    """What is not finite in a chunk of a row, of any map, reaches that chunk's outputs and row gradients, and the weights' gradients of its columns, and nothing else."""
    from deepbind_amd import smat as sm
    gen = torch.Generator(device="cuda").manual_seed(n + w)
    m, wd = nchunk * w, wide(kind)
    f = lambda *s: torch.randn(*s, generator=gen, device="cuda", dtype=wd)  # noqa: E731
    t = {k: f(n, m).to(TYPES[kind]) for k in ("Y", "R", "gate", "dR", "dZ")}
    W = {k: f(1, m) for k in ("gamma", "scale", "next_gamma") + (() if rms else ("beta", "next_beta"))}
    kw = dict(nchunk=nchunk, rms=rms, **W)

    def both():
        O, Z, stats = sm.blocknorm(t["Y"], t["R"], gate=t["gate"], want_stats=True, **kw)
        return (O, Z) + sm.blocknorm_bprop(t["Y"], O, stats, t["dR"], t["dZ"], gate=t["gate"], **kw)

    want = both()
    assert all(x is None or x.isfinite().all() for x in want)
    last = n - 1                                 # (rows that workgroups reach first and last)
    for name, row, col, bad in (("Y", 7, w - 1, float("nan")), ("R", last, 0, float("inf")), ("gate", 30, 2, float("inf")), ("dZ", last, m - 1, float("nan")), ("dR", 0, 1, float("-inf"))):
        old = t[name][row, col].clone()
        t[name][row, col] = bad
        got = both()
        t[name][row, col] = old
        chunk = slice(col // w * w, col // w * w + w)
        rows = torch.zeros(n, m, dtype=torch.bool, device="cuda")
        rows[row, chunk] = True
        for i, (a, b) in enumerate(zip(got, want)):
            if a is None:
                continue
            away = ~rows if i < 5 else ~rows[row:row + 1]
            assert torch.equal(a[away], b[away]), (name, i)
            if i < 2 and name in ("dZ", "dR"):
                assert torch.equal(a, b)
        # and where it cannot but be seen
        seen = {"Y": (0, 1, 2, 3), "R": (0, 1, 2, 3), "gate": (0, 1, 2, 3, 4), "dZ": (2, 3, 4), "dR": (2, 3, 4)}[name]
        for i in seen:
            assert not got[i][row, chunk].isfinite().all(), (name, i)


# ------------------------------------------------------------------------------------------------ clipping
@pytest.mark.parametrize("nblock", [1, 3])
@pytest.mark.parametrize("size", [120, 60000])
@pytest.mark.parametrize("kind,value,most", [("float32", 1e36, 1e-4), ("float32", 1e30, 1e-12), ("float32", 1e38, 1e-6), ("float32", 3e38, 1.0), ("float32", 1e37, 1e-30), ("bfloat16", 1e38, 1e-6),
                                             ("bfloat16", 1e30, 1e-12), ("float64", 1e140, 1e-150), ("float64", 1e150, 1e-170), ("float32", 1.0, 0.5)])
def test_clipping_by_factors_below_the_types_range(kind, value, most, size, nblock):
    """The factor may be far smaller than the smallest number of the gradients' type; what it makes of them is not."""
    from deepbind_amd import deepity_smat as ds
    rng = np.random.default_rng(4)
    # of one magnitude, so that every result is an ordinary number
    grads, plain = zip(*(put(value * rng.choice([-1, 1], s) * (1 + rng.random(s)) / 2, TYPES[kind]) for s in ((size // 12, 6), (1, size // 2))))
    norms, _ = ref.clip(plain, most, nblock, [False] * 2)
    want = [(p.astype(np.longdouble) * np.longdouble(most) / np.repeat(norms, p.shape[1] // nblock)).astype(float) for p in plain]
    out = [torch.empty_like(g) for g in grads]
    got = ds.clip_gradients(grads, most, nblock=nblock, out=out)
    n = size * 2.0 ** -53
    np.testing.assert_allclose(host(got)[0], norms, rtol=n)
    for o, w in zip(out, want):
        # the factor's own rounding, the product's, and the stored one's (a small factor is two: one more product); below the range half a step of it
        least = {"float32": 2.0 ** -150, "bfloat16": 2.0 ** -134, "float64": 0.0}[kind]
        assert (np.abs(host(o.double()) - w) <= (3 * U[kind] + STORED[kind] + n) * np.abs(w) + least).all()
    again = ds.clip_gradients(grads, most, nblock=nblock)
    assert torch.equal(again, got) and all(torch.equal(a, b) for a, b in zip(grads, out))
