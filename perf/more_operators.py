"""More operators of the layers along a map's rows and of their training, as cases that can be timed one by one: the gated delta
rule over the regions of a packed map, the norms around a block with its gate and residual, and clipping by the gradient's norm.

A map is an (N, channels) matrix whose rows are the positions of packed sequences; regions (P, 2) give every sequence's rows,
as for the pooling operators. Channels belong to heads, or to models laid side by side, as the motif scan's filters do.

kind    what a program calls
delta   S[t] = a[t] (I - b[t] k[t] k[t]') S[t-1] + b[t] k[t] v[t]', o[t] = scale S[t]' q[t] of every head along the rows of every
        region, a = exp(decay): a whole batch, forward and backward, or one new row per sequence ("token")
block   r' = r + scale * norm(y) * g sigmoid(g) and z = norm(r'), every row's (or model's block's) own norms: forward, or forward and backward
clip    the 2-norm of all gradients together (of every model's, where models lie side by side), and the gradients scaled down to a largest norm

`own = False` computes them in their plain form, elementary torch operations; `own = True` calls the package.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16}
EPS = 1e-5
CHUNK = 32                   # rows that the plain form of the delta rule takes at once


def listed():
    return [
        # a minibatch of reads through four heads of 64, scoring
        dict(name="delta_reads", kind="delta", call="forward", type="float32", count=2048, lo=63, hi=124, heads=4, groups=4, key=64, value=64,
             decay=True, shuffled=False, carried=False),
        # the next pieces of three long stretches, in half the width, going on from the states of the pieces before
        dict(name="delta_long", kind="delta", call="forward", type="bfloat16", count=3, lo=8000, hi=16000, heads=8, groups=8, key=128, value=128,
             decay=True, shuffled=False, carried=True),
        # 24 models of 16 filters trained on reads, a head for each
        dict(name="delta_train_models", kind="delta", call="train", type="float32", count=512, lo=63, hi=124, heads=24, groups=24, key=16, value=16,
             decay=True, shuffled=False, carried=False),
        # two long stretches, training in half the width; four value heads share each key
        dict(name="delta_train_long", kind="delta", call="train", type="bfloat16", count=2, lo=6000, hi=9000, heads=16, groups=4, key=64, value=64,
             decay=True, shuffled=False, carried=False),
        # 128 streams, one new row each
        dict(name="delta_token", kind="delta", call="token", type="float32", count=128, lo=1, hi=1, heads=16, groups=16, key=64, value=64,
             decay=True, shuffled=False, carried=True),
        # a gradient check in double precision: few short ragged sequences, odd sizes, no decay
        dict(name="delta_train_double", kind="delta", call="train", type="float64", count=17, lo=1, hi=77, heads=3, groups=1, key=19, value=13,
             decay=False, shuffled=True, carried=False),
        # the pooled features of one request scored by one model of 16 filters: what a service pays per call
        dict(name="block_pooled", kind="block", call="forward", type="float32", rows=64, models=1, width=16, rms=False, gate=True),
        # 64 models of 16 filters trained side by side, every model's own features normalised per position
        dict(name="block_train_models", kind="block", call="train", type="float32", rows=50021, models=64, width=16, rms=True, gate=False),
        # the map of a calibration batch's 1440 filters in half the width, as one row, trained
        dict(name="block_train_wide", kind="block", call="train", type="bfloat16", rows=130003, models=1, width=1440, rms=True, gate=True),
        # one motif model's gradients: a few small tensors
        dict(name="clip_small", kind="clip", type="float32", models=1, filters=16, taps=24, hidden=32),
        # a calibration batch: the gradients of 90 models side by side, each clipped by its own norm
        dict(name="clip_models", kind="clip", type="float32", models=90, filters=16, taps=24, hidden=32),
        # a large model's gradients in 40 tensors, matrices and vectors
        dict(name="clip_large", kind="clip", type="float32", tensors=40, most=6000000),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithm, capped so that none costs more than the largest listed."""
    kind = rng.choice(("delta", "delta", "delta", "block", "block", "clip"))
    kept = rng.choice(("float32", "float32", "bfloat16", "float64"))
    if kind == "clip":
        if rng.random() < 0.5:
            return dict(kind=kind, type=kept, models=rng.choice((1, _log(rng, 2, 96))), filters=_log(rng, 4, 64), taps=rng.randint(4, 32), hidden=_log(rng, 1, 64))
        return dict(kind=kind, type=kept, tensors=_log(rng, 1, 60), most=_log(rng, 10, 3000000))
    if kind == "block":
        models = rng.choice((1, 1, _log(rng, 2, 90)))
        width = _log(rng, 8, 4096) if models == 1 else _log(rng, 8, 64)
        return dict(kind=kind, call=rng.choice(("forward", "train")), type=kept, rows=_log(rng, 1, min(130000, 100000000 // (models * width))), models=models,
                    width=width, rms=rng.random() < 0.5, gate=rng.random() < 0.6)
    call = rng.choice(("forward", "train", "train", "token"))
    groups = _log(rng, 1, 8)
    heads = groups * rng.choice((1, 1, 2, 4))
    key = rng.choice((16, 32, 64, 64, 128, _log(rng, 2, 128)))
    value = rng.choice((key, key, 64, 128, _log(rng, 1, 160)))
    if call == "token":
        count, lo, hi = _log(rng, 1, 256), 1, 1
    else:
        lo = _log(rng, 1, 8000)
        hi = lo if rng.random() < 0.3 else lo + rng.randint(0, lo)
        most = 120000000 if kept == "float64" else 480000000                    # rows x heads x key x value
        count = _log(rng, 1, max(1, min(4096, most // (hi * heads * key * value))))
    return dict(kind=kind, call=call, type=kept, count=count, lo=lo, hi=hi, heads=heads, groups=groups, key=key, value=value, decay=rng.random() < 0.8,
                shuffled=call != "token" and rng.random() < 0.3, carried=call == "token" or (call == "forward" and rng.random() < 0.5))


# ---------------------------------------------------------------------------------------------- inputs
def _plan(case):
    """What belongs to the case and not to its data: the regions' lengths and their order in the table."""
    g = np.random.default_rng([case["count"], case["lo"], case["hi"], case["heads"]])
    lens = g.integers(case["lo"], case["hi"] + 1, size=case["count"])
    edges = np.concatenate([[0], np.cumsum(lens)])
    table = np.stack([edges[:-1], edges[1:]], 1)
    return table[g.permutation(case["count"])] if case["shuffled"] else table


def _gradients(case):
    """Shapes of the tensors of a clip case, and for each whether models' blocks are blocks of rows (else of columns)."""
    if "tensors" in case:
        g = np.random.default_rng([case["tensors"], case["most"]])
        sizes = [case["most"]] + [max(1, int(case["most"] * 10 ** -e)) for e in 2.5 * g.random(case["tensors"] - 1) ** 2]
        return [(1, n) if i % 3 == 2 or n < 64 else (n // int(n ** 0.5), int(n ** 0.5)) for i, n in enumerate(sizes)], [False] * len(sizes)
    M, F, H = case["models"], case["filters"], case["hidden"]
    return [(4 * case["taps"], M * F), (1, M * F), (F * M, H), (1, H * M), (H * M, 1), (1, M)], [False, False, True, False, True, False]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    kept = TYPES[case["type"]]
    wide = torch.float64 if kept == torch.float64 else torch.float32            # weights, states and sums
    normal = lambda *shape, dtype=wide: torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)  # noqa: E731
    uniform = lambda *shape: torch.rand(shape, generator=gen, device=DEVICE, dtype=torch.float32)  # noqa: E731
    s = dict(case)
    if case["kind"] == "clip":
        shapes, s["by_rows"] = _gradients(case)
        s["nblock"] = case.get("models", 1)
        # gradients of different sizes: about half the models (three in four where there is one) are over the largest norm
        total = sum(r * c for r, c in shapes)
        M = s["nblock"]
        level = torch.exp(1.5 * normal(M, dtype=torch.float32) + (1.0 if M == 1 else 0.0)) / math.sqrt(total / M)
        spread = lambda r, c, by: level.repeat_interleave(r // M)[:, None] if by else level.repeat_interleave(c // M)[None] if M > 1 else level  # noqa: E731
        s["grads"] = [(normal(r, c, dtype=torch.float32) * spread(r, c, by)).to(kept) for (r, c), by in zip(shapes, s["by_rows"])]
        s["max_norm"] = 1.0
        s["out"] = [torch.empty_like(t) for t in s["grads"]]
        return s
    if case["kind"] == "block":
        n, m = case["rows"], case["models"] * case["width"]
        s["Y"] = (normal(n, m, dtype=torch.float32) * 1.5 + 0.5 * normal(n, 1, dtype=torch.float32)).to(kept)
        s["R"] = (2 * normal(n, m, dtype=torch.float32)).to(kept)
        # the gate is the second half of a projection's output
        s["gate"] = normal(n, 2 * m, dtype=kept)[:, m:] if case["gate"] else None
        for k in ("gamma", "next_gamma"):
            s[k] = 1 + 0.2 * normal(1, m)
        s["scale"] = 0.3 + 0.1 * normal(1, m)
        s["beta"], s["next_beta"] = (None, None) if case["rms"] else (0.2 * normal(1, m), 0.2 * normal(1, m))
        s["out"] = (torch.empty_like(s["Y"]), torch.empty_like(s["Y"]))
        if case["call"] == "train":
            s["dR"], s["dZ"] = normal(n, m, dtype=kept), normal(n, m, dtype=kept)
            empty = lambda k: None if s[k] is None else torch.empty(s[k].shape, dtype=s[k].dtype, device=DEVICE)  # noqa: E731
            s["dout"] = tuple(empty(k) for k in ("Y", "R", "gate", "gamma", "beta", "scale", "next_gamma", "next_beta"))
        return s
    P, H, G, Kd, Vd = (case[k] for k in ("count", "heads", "groups", "key", "value"))
    table = _plan(case)
    tail = 0 if case["call"] == "token" else 23          # the padding after the last sequence, in no region
    n = int(table.max()) + tail
    s["longest"] = int((table[:, 1] - table[:, 0]).max())
    s["R"] = torch.from_numpy(table.astype(np.int32)).to(DEVICE)
    # keys follow the letters that they stand for, so that a key comes again and again
    letters = torch.randint(0, 4, (n,), generator=gen, device=DEVICE)
    unit = lambda t: (t / t.norm(dim=2, keepdim=True)).reshape(n, G * Kd).to(kept)  # noqa: E731
    s["K"] = unit(normal(4, G, Kd, dtype=torch.float32)[letters] + 0.7 * normal(n, G, Kd, dtype=torch.float32))
    s["Q"] = unit(normal(4, G, Kd, dtype=torch.float32)[letters] + 0.7 * normal(n, G, Kd, dtype=torch.float32))
    s["V"] = normal(n, H * Vd, dtype=kept)
    s["beta"] = torch.sigmoid(normal(n, H))
    rates = torch.exp(uniform(1, H) * math.log(200) + math.log(1e-3))           # 0.001 to 0.2
    s["g"] = -(rates * torch.exp(0.5 * normal(n, H, dtype=torch.float32))).to(wide) if case["decay"] else None
    s["state"] = 0.3 * normal(P, Kd, H * Vd) if case["carried"] else None
    s["next"] = torch.empty_like(s["state"]) if case["carried"] else None
    s["out"] = torch.zeros((n, H * Vd), dtype=kept, device=DEVICE)
    if case["call"] == "train":
        s["dO"] = normal(n, H * Vd, dtype=kept)
        zero = lambda t: None if t is None else torch.zeros(t.shape, dtype=t.dtype, device=DEVICE)  # noqa: E731
        s["dout"] = tuple(zero(s[k]) for k in ("Q", "K", "V", "beta", "g"))
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _up(t):
    return t if t is None or t.dtype == torch.float64 else t.float()


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _normed(X, s):
    """Every chunk's values less their mean (not with rms) over their deviation, and the reciprocal deviations."""
    V = X.view(X.shape[0], -1, s["width"])
    c = V if s["rms"] else V - V.mean(2, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(2, keepdim=True) + EPS)
    return (c * r).view(X.shape), r


def _normed_back(q, h, r, s):
    q, H = q.view(q.shape[0], -1, s["width"]), h.view(h.shape[0], -1, s["width"])
    d = q - H * (q * H).mean(2, keepdim=True)
    return (r * (d if s["rms"] else d - q.mean(2, keepdim=True))).view(h.shape)


def _block(s):
    kept = s["Y"].dtype
    Y, R, gate = _up(s["Y"]), _up(s["R"]), _up(s["gate"])
    h1, r1 = _normed(Y, s)
    P = h1 * s["gamma"] if s["rms"] else h1 * s["gamma"] + s["beta"]
    sig = None if gate is None else _sigmoid(gate)
    act = 1.0 if gate is None else gate * sig
    Rn = (R + s["scale"] * P * act).to(kept)
    h2, r2 = _normed(_up(Rn), s)                         # (of the residual as it is kept)
    Z = (h2 * s["next_gamma"] if s["rms"] else h2 * s["next_gamma"] + s["next_beta"]).to(kept)
    if s["call"] == "forward":
        return Rn, Z
    dR, dZ = _up(s["dR"]), _up(s["dZ"])
    total = dR + _normed_back(dZ * s["next_gamma"], h2, r2, s)
    dP = total * s["scale"] * act
    rows = lambda t: t.sum(0, keepdim=True)  # noqa: E731
    dgate = 0.0 if gate is None else (total * s["scale"] * P * sig * (1 + gate * (1 - sig))).to(kept)
    return (Rn, Z, _normed_back(dP * s["gamma"], h1, r1, s).to(kept), total.to(kept), dgate, rows(dP * h1), 0.0 if s["rms"] else rows(dP),
            rows(total * P * act), rows(dZ * h2), 0.0 if s["rms"] else rows(dZ))


def _clip(s):
    M = s["nblock"]
    blocks = [t.view(M, -1, t.shape[1]) if by else t.view(t.shape[0], M, -1).transpose(0, 1) for t, by in zip(s["grads"], s["by_rows"])]
    norms = sum((t.double() ** 2).sum((1, 2)) for t in blocks).sqrt()
    factor = torch.where(norms > s["max_norm"], s["max_norm"] / norms, 1.0)
    out = [(_up(t) * factor.to(_up(t).dtype)[:, None, None]).to(t.dtype) for t in blocks]
    return norms.view(1, M), [(o if by else o.transpose(0, 1)).reshape(t.shape) for o, t, by in zip(out, s["grads"], s["by_rows"])]


def _rows(s):
    """Row numbers (regions, whole chunks of rows) of every region and which of them exist."""
    R = s["R"].long()
    at = torch.arange(-(-s["longest"] // CHUNK) * CHUNK, device=R.device)
    ok = at[None, :] < (R[:, 1] - R[:, 0])[:, None]
    return torch.where(ok, R[:, :1] + at, 0), ok


def _heads(t, rows, ok, n, H):
    """(N, n x width) rows to (regions, H, chunks, CHUNK, width), zeros where no row is; n heads are spread over H."""
    v = torch.where(ok[:, :, None], _up(t)[rows], 0)
    v = v.view(v.shape[0], -1, CHUNK, n, v.shape[2] // n).permute(0, 3, 1, 2, 4)
    return v.repeat_interleave(H // n, 1).contiguous()


def _packed(v, rows, ok, like, n):
    """The way back: rows at their places in a map that is zero elsewhere; heads that share are summed."""
    v = v.view(v.shape[0], n, -1, *v.shape[2:]).sum(2) if v.shape[1] > n else v
    v = v.permute(0, 2, 3, 1, 4).reshape(ok.shape[0], ok.shape[1], -1)
    out = torch.zeros(like.shape, dtype=like.dtype, device=like.device)
    out[rows[ok]] = v[ok].to(like.dtype)
    return out


def _T(t):
    return t.transpose(-1, -2).contiguous()


def _unit_lower_inverse(L):
    """(I + L)^-1 of strictly lower triangles: inverses of blocks of 1, 2, 4, ... on the diagonal."""
    n, k = L.shape[-1], 1
    at = torch.arange(n, device=L.device)
    A = torch.eye(n, dtype=L.dtype, device=L.device).expand(L.shape).contiguous()
    while k < n:
        below = (at[:, None] // (2 * k) == at[None, :] // (2 * k)) & (at[:, None] // k > at[None, :] // k)
        A = A - A @ (torch.where(below, L, 0) @ A)
        k *= 2
    return A


def _delta(s):
    H, G, kept = s["heads"], s["groups"], s["V"].dtype
    scale = s["key"] ** -0.5
    if s["call"] == "token":
        P = s["count"]
        q, k = (_up(s[n]).view(P, G, -1).repeat_interleave(H // G, 1) for n in ("Q", "K"))
        v = _up(s["V"]).view(P, H, -1)
        S = s["state"].view(P, s["key"], H, -1).transpose(1, 2)
        S = S * torch.exp(s["g"])[:, :, None, None] if s["g"] is not None else S
        u = s["beta"][:, :, None] * (v - (k[..., None] * S).sum(2))
        S = S + k[..., None] * u[:, :, None]
        return (scale * (q[..., None] * S).sum(2)).reshape(P, -1).to(kept), S.transpose(1, 2).reshape(s["state"].shape)
    rows, ok = _rows(s)
    q, k = (_heads(s[n], rows, ok, G, H) for n in ("Q", "K"))
    v, b = _heads(s["V"], rows, ok, H, H), _heads(s["beta"], rows, ok, H, H)
    at = torch.arange(CHUNK, device=q.device)
    lower, strictly = at[:, None] >= at, at[:, None] > at
    if s["g"] is not None:
        c = _heads(s["g"], rows, ok, H, H).cumsum(3)     # (rows that do not exist do not decay)
        D = torch.where(lower, torch.exp(c - _T(c)), 0)
        first, last = torch.exp(c), torch.exp(c[..., -1:, :] - c)
    else:
        D, first, last = lower.to(q.dtype), torch.ones_like(b), torch.ones_like(b)
    M, A = k @ _T(k), q @ _T(k)
    N_, Pm = torch.where(strictly, M * D, 0), A * D
    T = _unit_lower_inverse(b * N_)
    n = q.shape[2]
    S = q.new_zeros(q.shape[0], H, s["key"], s["value"])
    if s["state"] is not None:
        S = s["state"].view(-1, s["key"], H, s["value"]).transpose(1, 2).contiguous()
    us, xs, Ss, os = [], [], [], []
    kl = _T(k * last)
    for i in range(n):
        W = k[:, :, i] @ S
        x = v[:, :, i] - first[:, :, i] * W
        u = T[:, :, i] @ (b[:, :, i] * x)
        os.append(scale * (first[:, :, i] * (q[:, :, i] @ S) + Pm[:, :, i] @ u))
        us.append(u), xs.append(x), Ss.append(S)
        S = first[:, :, i, -1:] * S + kl[:, :, i] @ u
    O = _packed(torch.stack(os, 2), rows, ok, s["V"], H)
    if s["call"] == "forward":
        return (O, S.transpose(1, 2).reshape(s["state"].shape)) if s["state"] is not None else O
    do = scale * _heads(s["dO"], rows, ok, H, H)
    u, x, S0 = torch.stack(us, 2), torch.stack(xs, 2), torch.stack(Ss, 2)
    W = (v - x)                                          # first * (k S)
    Tt, Pt, kt, qt = _T(T), _T(Pm), _T(k), _T(q * first)
    dS, dSs, dys = torch.zeros_like(S), [], []
    for i in range(n - 1, -1, -1):
        dy = Tt[:, :, i] @ (Pt[:, :, i] @ do[:, :, i] + last[:, :, i] * (k[:, :, i] @ dS))
        dSs.append(dS), dys.append(dy)
        dS = first[:, :, i, -1:] * dS - kt[:, :, i] @ (first[:, :, i] * b[:, :, i] * dy) + qt[:, :, i] @ do[:, :, i]
    dy, dS1 = torch.stack(dys[::-1], 2), torch.stack(dSs[::-1], 2)
    dx = b * dy
    ut, S0t = _T(u), _T(S0)
    dPm, dL = torch.where(lower, do @ ut, 0), torch.where(strictly, -(dy @ ut), 0)
    dM, dA = dL * b * D, dPm * D
    dq = dA @ k + (do * first) @ S0t
    dk = _T(dA) @ q + (dM + _T(dM)) @ k - (dx * first) @ S0t + (last * u) @ _T(dS1)
    db = (dy * x).sum(-1, keepdim=True) + (dL * N_).sum(-1, keepdim=True)
    grads = (_packed(dq, rows, ok, s["Q"], G), _packed(dk, rows, ok, s["K"], G), _packed(dx, rows, ok, s["V"], H), _packed(db, rows, ok, s["beta"], H))
    if s["g"] is None:
        return (O,) + grads
    # a row's decay acts on every pair of rows around it, on what comes from the state before the chunk and on what goes to the state behind it
    E = dPm * Pm + dL * b * N_
    pairs = _inside(E)
    into = (do * first * (q @ S0)).sum(-1) - (dx * W).sum(-1)
    out = (last * u * (k @ dS1)).sum(-1)
    through = first[..., -1, 0] * (dS1 * S0).sum((-1, -2))
    dg = pairs + into.flip(3).cumsum(3).flip(3) + (out.cumsum(3) - out) + through[..., None]
    return (O,) + grads + (_packed(dg[..., None], rows, ok, s["g"], H),)


def _inside(E):
    """sum over i >= m > j of E[i, j], for every m."""
    at = torch.arange(E.shape[-1], device=E.device)
    upto = (E @ (at[:, None] < at).to(E.dtype))          # [i, m]: sum over j < m
    return torch.where(at[:, None] >= at, upto, 0).sum(-2)


# ---------------------------------------------------------------------------------------------- the package's calls
def _own_delta(s):
    from deepbind_amd import kangaroo_smat as ks
    more = dict(decay=s["g"], groups=s["groups"])
    if s["call"] == "token":
        return ks.deltarule_step(s["Q"], s["K"], s["V"], s["beta"], s["state"], into=s["next"], out=s["out"], **more), s["next"]
    if s["call"] == "forward":
        O, last = ks.deltarule(s["Q"], s["K"], s["V"], s["beta"], s["R"], state=s["state"], want_state=s["state"] is not None, out=s["out"], **more)
        return O if last is None else (O, last)
    keep = ks.kept_delta(s["K"], s["V"], s["beta"], groups=s["groups"])
    O, _ = ks.deltarule(s["Q"], s["K"], s["V"], s["beta"], s["R"], keep=keep, out=s["out"], **more)
    grads = ks.deltarule_bprop(s["Q"], s["K"], s["V"], s["beta"], s["R"], keep, s["dO"], out=s["dout"], **more)
    return (O,) + tuple(g for g in grads if g is not None)


def _own_block(s):
    from deepbind_amd import smat as sm
    what = dict(gate=s["gate"], gamma=s["gamma"], scale=s["scale"], next_gamma=s["next_gamma"], nchunk=s["models"], rms=s["rms"])
    Rn, Z, stats = sm.blocknorm(s["Y"], s["R"], beta=s["beta"], next_beta=s["next_beta"], eps=EPS, want_stats=s["call"] == "train", out=s["out"], **what)
    if s["call"] == "forward":
        return Rn, Z
    grads = sm.blocknorm_bprop(s["Y"], Rn, stats, s["dR"], s["dZ"], beta=s["beta"], next_beta=s["next_beta"], out=s["dout"], **what)
    return (Rn, Z) + tuple(0.0 if g is None else g for g in grads)


def _own_clip(s):
    from deepbind_amd import deepity_smat as ds
    norms = ds.clip_gradients(s["grads"], s["max_norm"], nblock=s["nblock"], by_rows=s["by_rows"], out=s["out"])
    return norms, s["out"]


def run(state):
    if own:
        return {"delta": _own_delta, "block": _own_block, "clip": _own_clip}[state["kind"]](state)
    return {"delta": _delta, "block": _block, "clip": _clip}[state["kind"]](state)


def work(case):
    b = {"float32": 4, "float64": 8, "bfloat16": 2}[case["type"]]
    wb = 8 if b == 8 else 4
    if case["kind"] == "clip":
        n = sum(r * c for r, c in _gradients(case)[0])
        return {"bytes": 2 * n * b, "flops": 3 * n}
    train = case["call"] == "train"
    if case["kind"] == "block":
        e, gate = case["rows"] * case["models"] * case["width"], 1 if case["gate"] else 0
        # Y, R, gate in, the new R and Z out; and dR, dZ in, dY, dR, dgate out
        return {"bytes": e * b * ((8 + 2 * gate) if train else 4 + gate), "flops": e * ((50 + 20 * gate) if train else 18 + 6 * gate)}
    table = _plan(case)
    rows = int((table[:, 1] - table[:, 0]).sum())
    H, G, Kd, Vd = (case[k] for k in ("heads", "groups", "key", "value"))
    rates = rows * H * wb * (2 if case["decay"] else 1)
    state = 2 * case["count"] * Kd * H * Vd * wb if case["carried"] else 0
    # per row and head: the state's decay, what the key finds, what is added and what the query finds, 7 operations a value of the state; 15 backward
    if train:
        return {"bytes": rows * b * (4 * G * Kd + 4 * H * Vd) + 2 * rates, "flops": rows * H * Kd * Vd * 22}
    return {"bytes": rows * b * (2 * G * Kd + 2 * H * Vd) + rates + state, "flops": rows * H * Kd * Vd * 7}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed).items()
         if k not in ("out", "dout", "next")}
    return {"delta": _exact_delta, "block": _exact_block, "clip": _exact_clip}[case["kind"]](case, s)


def _exact_clip(case, s):
    M, grads = s["nblock"], [t.double() for t in s["grads"]]
    owners = []
    for t, by in zip(grads, s["by_rows"]):
        per = (t.shape[0] if by else t.shape[1]) // M
        one = torch.arange(M * per, device=DEVICE) // per
        owners.append((one[:, None] if by else one[None, :]).expand(t.shape) if M > 1 else torch.zeros(t.shape, dtype=torch.long, device=DEVICE))
    squares = torch.zeros(M, dtype=torch.float64, device=DEVICE)
    for t, o in zip(grads, owners):
        for m in range(M):
            squares[m] += (t[o == m] ** 2).sum() if M > 1 else (t * t).sum()
    norms = squares ** 0.5
    down = torch.clamp(s["max_norm"] / norms, max=1.0)
    return norms[None], [t * down[o] for t, o in zip(grads, owners)]


def _exact_block(case, s):
    w, Y, R = case["width"], s["Y"], s["R"]
    kept, train = TYPES[case["type"]], case["call"] == "train"
    out = {k: [] for k in ("R", "Z", "dY", "dR", "dgate", "dgamma", "dbeta", "dscale", "dnext_gamma", "dnext_beta")}

    def norm(x):
        c = x if case["rms"] else x - x.sum(1, keepdim=True) / w
        r = ((c ** 2).sum(1, keepdim=True) / w + EPS) ** -0.5
        return c * r, r

    def back(d, h, r):
        sent = r * (d - h * ((d * h).sum(1, keepdim=True) / w))
        return sent if case["rms"] else sent - r * (d.sum(1, keepdim=True) / w)

    for i in range(case["models"]):
        at = slice(i * w, (i + 1) * w)
        part = {k: None if s[k] is None else s[k][:, at] for k in ("gamma", "beta", "scale", "next_gamma", "next_beta", "gate")}
        h, r = norm(Y[:, at])
        p = h * part["gamma"] + (0 if part["beta"] is None else part["beta"])
        g = part["gate"]
        e = None if g is None else 1 / (1 + torch.exp(-g))
        open_ = torch.ones_like(p) if g is None else g * e
        new = R[:, at] + part["scale"] * p * open_
        # the second norm is of the residual as it is kept: that rounding is part of the definition
        h2, r2 = norm(new.to(kept).double())
        out["R"].append(new)
        out["Z"].append(h2 * part["next_gamma"] + (0 if part["next_beta"] is None else part["next_beta"]))
        if not train:
            continue
        dZ = s["dZ"][:, at]
        t = s["dR"][:, at] + back(dZ * part["next_gamma"], h2, r2)
        dp = t * part["scale"] * open_
        out["dR"].append(t)
        out["dY"].append(back(dp * part["gamma"], h, r))
        if g is not None:
            out["dgate"].append(t * part["scale"] * p * (e + g * e * (1 - e)))
        sums = dict(dgamma=dp * h, dscale=t * p * open_, dnext_gamma=dZ * h2)
        if not case["rms"]:
            sums.update(dbeta=dp, dnext_beta=dZ)
        for k, v in sums.items():
            out[k].append(v.sum(0, keepdim=True))
    whole = lambda k: torch.cat(out[k], 1) if out[k] else 0.0  # noqa: E731
    if not train:
        return whole("R"), whole("Z")
    return tuple(whole(k) for k in ("R", "Z", "dY", "dR", "dgate", "dgamma", "dbeta", "dscale", "dnext_gamma", "dnext_beta"))


def _exact_delta(case, s):
    P, H, G, Kd, Vd = (case[k] for k in ("count", "heads", "groups", "key", "value"))
    R, scale = _plan(case), case["key"] ** -0.5
    start, length = torch.from_numpy(R[:, 0]).to(DEVICE), torch.from_numpy(R[:, 1] - R[:, 0]).to(DEVICE)
    longest, n, train = int(length.max()), s["V"].shape[0], case["call"] == "train"
    if longest > 25000 or (train and (longest * P * H * Kd * Vd * 8 > 60e9 or longest > 10000)):    # (every step's states are held)
        return None
    of = torch.arange(H, device=DEVICE) // (H // G)
    q, k = s["Q"].view(n, G, Kd)[:, of], s["K"].view(n, G, Kd)[:, of]
    v, b = s["V"].view(n, H, Vd), s["beta"]
    a = torch.ones_like(b) if s["g"] is None else torch.exp(s["g"])
    by_length = torch.argsort(length, descending=True)   # so that the regions that still run are the first ones
    start, length = start[by_length], length[by_length]
    alive = (length[None, :] > torch.arange(longest, device=DEVICE)[:, None]).sum(1).tolist()
    S = torch.zeros((P, H, Kd, Vd), dtype=torch.float64, device=DEVICE)
    if s["state"] is not None:
        S = s["state"].view(P, Kd, H, Vd).transpose(1, 2)[by_length].contiguous()
    O, held = torch.zeros_like(v), []
    found = lambda state, row: torch.matmul(row[:, :, None], state)[:, :, 0]  # row' S  # noqa: E731
    for t in range(longest):
        m = alive[t]
        at = start[:m] + t
        old = S[:m] * a[at][:, :, None, None]
        held.append(S[:m].clone() if train else None)
        u = b[at][..., None] * (v[at] - found(old, k[at]))
        new = old + k[at][..., None] * u[:, :, None]
        O[at] = scale * found(new, q[at])
        S[:m] = new
    O = O.view(n, H * Vd)
    if not train:
        last = torch.empty((P, Kd, H * Vd), dtype=torch.float64, device=DEVICE)
        last[by_length] = S.transpose(1, 2).reshape(P, Kd, H * Vd)
        return (O, last) if s["state"] is not None else O
    dO = s["dO"].view(n, H, Vd) * scale
    dq, dk, dv, db, da = (torch.zeros_like(t) for t in (q, k, v, b, a))
    dS = torch.zeros_like(S)
    for t in range(longest - 1, -1, -1):
        m = alive[t]
        at = start[:m] + t
        kt, vt, bt = k[at], v[at], b[at][..., None]
        old = held[t] * a[at][:, :, None, None]
        miss = vt - found(old, kt)
        new = old + kt[..., None] * (bt * miss)[:, :, None]
        dq[at] = torch.matmul(new, dO[at][..., None])[..., 0]
        dnew = dS[:m] + q[at][..., None] * dO[at][:, :, None]
        du = found(dnew, kt)
        dmiss = bt * du
        dv[at] = dmiss
        db[at] = (du * miss).sum(-1)
        dk[at] = torch.matmul(dnew, (bt * miss)[..., None])[..., 0] - torch.matmul(old, dmiss[..., None])[..., 0]
        dold = dnew - kt[..., None] * dmiss[:, :, None]
        da[at] = (dold * held[t]).sum((-1, -2))
        dS[:m] = dold * a[at][:, :, None, None]
        held[t] = None
    shared = lambda t: t.view(n, G, H // G, Kd).sum(2).view(n, G * Kd)  # noqa: E731
    grads = (O, shared(dq), shared(dk), dv.view(n, H * Vd), db)
    return grads if s["g"] is None else grads + (da * a,)
