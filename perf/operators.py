"""The sequence-layer operators as cases that can be timed one by one: row normalisation, the short causal convolution and
the selective state space scan over the regions of a packed map.

A map is an (N, channels) matrix whose rows are the positions of packed sequences; regions (P, 2) give every sequence's rows,
as for the pooling operators. Channels belong to models laid side by side, as the motif scan's filters do.

kind    what a program calls
norm    layer norm of every row (of every model's block of a row): forward, or forward and backward ("train")
conv    causal convolution of up to four taps along the rows of every region, with bias and x * sigmoid(x): a whole batch,
        forward and backward, or one new row per sequence ("token")
scan    h[t] = exp(d[t] A) h[t-1] + d[t] B[t] x[t], y[t] = C[t] . h[t] + D x[t], times g sigmoid(g) of a gate, along the rows
        of every region, d = softplus(dt + bias): a whole batch, forward and backward, or one new row per sequence

`own = False` computes them in their plain form, elementary torch operations; `own = True` calls the package.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda" if torch.cuda.is_available() else "cpu"
TYPES = {"float32": torch.float32, "float64": torch.float64, "bfloat16": torch.bfloat16}
EPS = 1e-5


def listed():
    return [
        # the pooled features of one request scored by one model of 16 filters: what a service pays per call
        dict(name="norm_pooled", kind="norm", call="forward", type="float32", rows=64, models=1, width=16),
        # 64 models of 16 filters trained side by side, every model's own features normalised per position
        dict(name="norm_train_models", kind="norm", call="train", type="float32", rows=50021, models=64, width=16),
        # the map of a calibration batch's 1440 filters in half the width, normalised as one row, trained
        dict(name="norm_train_wide", kind="norm", call="train", type="bfloat16", rows=130003, models=1, width=1440),
        # a minibatch of reads through the short convolution, scoring
        dict(name="conv_reads", kind="conv", call="forward", type="float32", count=2048, lo=63, hi=124, channels=256, taps=4, shuffled=False),
        # a few long stretches of a genome, training in half the width
        dict(name="conv_train_long", kind="conv", call="train", type="bfloat16", count=6, lo=9000, hi=30000, channels=1024, taps=4, shuffled=False),
        # sequences scored letter by letter as they arrive: 64 streams, one row each
        dict(name="conv_token", kind="conv", call="token", type="float32", count=64, lo=1, hi=1, channels=512, taps=4, shuffled=False),
        # a minibatch of reads through the scan, scoring
        dict(name="scan_reads", kind="scan", call="forward", type="float32", count=2048, lo=63, hi=124, channels=256, groups=1, states=16,
             gate=True, shuffled=False, carried=False),
        # the next pieces of three long stretches, in half the width, going on from the state of the pieces before
        dict(name="scan_long", kind="scan", call="forward", type="bfloat16", count=3, lo=8000, hi=16000, channels=1024, groups=1, states=16,
             gate=True, shuffled=False, carried=True),
        # 24 models of 16 filters trained on reads; every model has its own input and output weights
        dict(name="scan_train_models", kind="scan", call="train", type="float32", count=512, lo=63, hi=124, channels=384, groups=24, states=16,
             gate=False, shuffled=False, carried=False),
        # two long stretches, training in half the width
        dict(name="scan_train_long", kind="scan", call="train", type="bfloat16", count=2, lo=6000, hi=9000, channels=1024, groups=1, states=16,
             gate=True, shuffled=False, carried=False),
        # 128 streams, one new row each
        dict(name="scan_token", kind="scan", call="token", type="float32", count=128, lo=1, hi=1, channels=1024, groups=1, states=16,
             gate=True, shuffled=False, carried=True),
        # a gradient check in double precision: few short ragged sequences, odd sizes
        dict(name="scan_train_double", kind="scan", call="train", type="float64", count=17, lo=1, hi=77, channels=57, groups=3, states=5,
             gate=True, shuffled=True, carried=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    """One more case of the same ranges: sizes spread over their logarithm, capped so that none costs more than the largest listed."""
    kind = rng.choice(("norm", "conv", "scan", "scan"))
    call = rng.choice(("forward", "train")) if kind == "norm" else rng.choice(("forward", "train", "train", "token"))
    kept = rng.choice(("float32", "float32", "bfloat16", "float64"))
    if kind == "norm":
        models = rng.choice((1, 1, _log(rng, 2, 90)))
        width = _log(rng, 8, 4096) if models == 1 else _log(rng, 8, 64)         # (two values leave a gradient that is all rounding)
        return dict(kind=kind, call=call, type=kept, rows=_log(rng, 1, min(200000, 100000000 // (models * width))), models=models, width=width)
    most = 4000000 if kind == "scan" else 40000000          # rows x channels
    groups = rng.choice((1, 1, _log(rng, 2, 24))) if kind == "scan" else 1
    channels = groups * (_log(rng, 1, 1024) if groups == 1 else _log(rng, 1, 64))
    if call == "token":
        count, lo, hi = _log(rng, 1, 256), 1, 1
    else:
        lo = _log(rng, 1, 12000)
        hi = lo if rng.random() < 0.3 else lo + rng.randint(0, lo)
        count = _log(rng, 1, max(1, min(4096, most // (hi * channels))))
    case = dict(kind=kind, call=call, type=kept, count=count, lo=lo, hi=hi, channels=channels, shuffled=rng.random() < 0.3)
    if kind == "conv":
        return dict(case, taps=rng.randint(2, 4))
    return dict(case, groups=groups, states=rng.choice((16, 16, 8, rng.randint(1, 16))), gate=rng.random() < 0.6,
                carried=call == "token" or (call == "forward" and rng.random() < 0.5))


# ---------------------------------------------------------------------------------------------- inputs
def _plan(case):
    """What belongs to the case and not to its data: the regions' lengths and their order in the table."""
    g = np.random.default_rng([case["count"], case["lo"], case["hi"], case["channels"]])
    lens = g.integers(case["lo"], case["hi"] + 1, size=case["count"])
    edges = np.concatenate([[0], np.cumsum(lens)])
    table = np.stack([edges[:-1], edges[1:]], 1)
    return table[g.permutation(case["count"])] if case["shuffled"] else table


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(int(seed))
    kept = TYPES[case["type"]]
    wide = torch.float64 if kept == torch.float64 else torch.float32            # weights, states and sums
    normal = lambda *shape, dtype=wide: torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)  # noqa: E731
    s = dict(case)
    if case["kind"] == "norm":
        n, m = case["rows"], case["models"] * case["width"]
        s["X"] = (normal(n, m, dtype=torch.float32) * 1.5 + normal(n, 1, dtype=torch.float32)).to(kept)
        s["gamma"], s["beta"] = 1 + 0.2 * normal(1, m), 0.2 * normal(1, m)
        s["out"] = torch.empty_like(s["X"])
        if case["call"] == "train":
            s["dZ"] = normal(n, m, dtype=kept)
            s["dout"] = (torch.empty_like(s["X"]), torch.empty_like(s["gamma"]), torch.empty_like(s["beta"]))
        return s
    D, P = case["channels"], case["count"]
    table = _plan(case)
    tail = 0 if case["call"] == "token" else 23          # the padding after the last sequence, in no region
    n = int(table.max()) + tail
    s["longest"] = int((table[:, 1] - table[:, 0]).max())
    s["R"] = torch.from_numpy(table.astype(np.int32)).to(DEVICE)
    s["out"] = torch.zeros((n, D), dtype=kept, device=DEVICE)
    if case["kind"] == "conv":
        K = case["taps"]
        s["X"] = normal(n, D, dtype=kept)
        s["W"], s["b"] = normal(K, D) / math.sqrt(K), 0.1 * normal(1, D)
        if case["call"] == "token":
            s["state"] = normal(P, K - 1, D, dtype=kept)
            s["next"] = torch.empty_like(s["state"])
        if case["call"] == "train":
            s["dZ"] = normal(n, D, dtype=kept)
            s["dout"] = (torch.zeros_like(s["X"]), torch.empty_like(s["W"]), torch.empty_like(s["b"]))
        return s
    S, G = case["states"], case["groups"]
    s["X"] = normal(n, D, dtype=kept)
    s["dt"] = (0.5 * normal(n, D, dtype=torch.float32)).to(kept)
    steps = torch.exp(torch.rand((1, D), generator=gen, device=DEVICE) * math.log(100) + math.log(1e-3))      # 0.001 to 0.1
    s["bias"] = torch.log(torch.expm1(steps)).to(wide)
    s["A"] = -(torch.arange(1, S + 1, device=DEVICE, dtype=wide)[:, None] * torch.exp(0.1 * normal(S, D))).contiguous()
    both = normal(n, 2 * G * S)                          # one projection's output: input and output weights side by side
    s["B"], s["C"] = both[:, :G * S], both[:, G * S:]
    s["D"] = 1 + 0.1 * normal(1, D)
    # the gate is the second half of the projection whose first half went through the convolution
    s["gate"] = normal(n, 2 * D, dtype=kept)[:, D:] if case["gate"] else None
    s["state"] = normal(P, S, D) if case["carried"] else None
    s["next"] = torch.empty_like(s["state"]) if case["carried"] else None
    if case["call"] == "train":
        s["dY"] = normal(n, D, dtype=kept)
        zero = lambda t: None if t is None else torch.zeros(t.shape, dtype=t.dtype, device=DEVICE)  # noqa: E731
        s["dout"] = tuple(zero(s[k]) for k in ("X", "dt", "A", "B", "C", "D", "gate", "bias"))
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _up(t):
    return t if t is None or t.dtype == torch.float64 else t.float()


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _norm(s):
    X, gamma, beta = _up(s["X"]), s["gamma"], s["beta"]
    n, m, w = X.shape[0], X.shape[1], s["width"]
    V = X.view(n, -1, w)
    c = V - V.mean(2, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(2, keepdim=True) + EPS)
    H = c * r
    Z = (H.view(n, m) * gamma + beta).to(s["X"].dtype)
    if s["call"] == "forward":
        return Z
    dZ = _up(s["dZ"])
    dH = (dZ * gamma).view(n, -1, w)
    dX = r * (dH - dH.mean(2, keepdim=True) - H * (dH * H).mean(2, keepdim=True))
    return Z, dX.view(n, m).to(s["X"].dtype), (dZ * H.view(n, m)).sum(0, keepdim=True), dZ.sum(0, keepdim=True)


def _rows(s):
    """Row numbers (regions, longest) of every region and which of them exist."""
    R = s["R"].long()
    at = torch.arange(s["longest"], device=R.device)
    ok = at[None, :] < (R[:, 1] - R[:, 0])[:, None]
    return torch.where(ok, R[:, :1] + at, 0), ok[:, :, None]


def _padded(t, rows, ok):
    return torch.where(ok, _up(t)[rows], 0)


def _packed(v, rows, ok, like):
    """The rows of v that exist, at their places in a map that is zero elsewhere."""
    out = torch.zeros(like.shape, dtype=like.dtype, device=like.device)
    out[rows[ok[:, :, 0]]] = v[ok[:, :, 0]].to(like.dtype)
    return out


def _conv(s):
    K, W, b = s["taps"], s["W"], s["b"]
    if s["call"] == "token":
        window = torch.cat([s["state"], s["X"][:, None]], 1)
        pre = (_up(window) * W).sum(1) + b
        return (pre * _sigmoid(pre)).to(s["X"].dtype), window[:, 1:]
    rows, ok = _rows(s)
    x = _padded(s["X"], rows, ok)
    x = torch.cat([x.new_zeros(x.shape[0], K - 1, x.shape[2]), x], 1)
    windows = x.unfold(1, K, 1)                          # (regions, longest, channels, taps)
    pre = (windows * W.t()).sum(3) + b
    gate = _sigmoid(pre)
    Z = _packed(pre * gate, rows, ok, s["X"])
    if s["call"] == "forward":
        return Z
    dpre = _padded(s["dZ"], rows, ok) * gate * (1 + pre * (1 - gate))
    ahead = torch.cat([dpre, dpre.new_zeros(dpre.shape[0], K - 1, dpre.shape[2])], 1).unfold(1, K, 1)
    dX = (ahead * W.flip(0).t()).sum(3)
    return Z, _packed(dX, rows, ok, s["X"]), (windows * dpre[..., None]).sum((0, 1)).t(), dpre.sum((0, 1))[None]


def _recur(a, b):
    """h[:, t] = a[:, t] h[:, t-1] + b[:, t] for all t at once: pairs of steps are joined, then pairs of pairs."""
    a, h, k = a.clone(), b.clone(), 1
    while k < h.shape[1]:
        h[:, k:] += a[:, k:] * h[:, :-k]
        a[:, k:] = a[:, k:] * a[:, :-k]
        k *= 2
    return h


def _steps(s):
    """softplus(dt + bias) and its derivative."""
    v = _up(s["dt"]) + s["bias"]
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs())), _sigmoid(v)


def _spread(t, s):
    """(..., groups x states) to (..., channels, states): every channel's own group's values."""
    G, S = s["groups"], s["states"]
    return t.reshape(t.shape[:-1] + (G, 1, S)).expand(t.shape[:-1] + (G, s["channels"] // G, S)).reshape(t.shape[:-1] + (s["channels"], S))


def _gathered(t, s):
    """The gradient's way back: the sum over a group's channels."""
    G, S = s["groups"], s["states"]
    return t.reshape(t.shape[:-2] + (G, s["channels"] // G, S)).sum(-2).reshape(t.shape[:-2] + (G * S,))


def _scan(s):
    A, D, X = s["A"].t(), s["D"], s["X"]
    step, slope = _steps(s)
    if s["call"] == "token":
        x, gate = _up(X), _up(s["gate"])
        h = torch.exp(step[:, :, None] * A) * s["state"].transpose(1, 2) + (step * x)[:, :, None] * _spread(s["B"], s)
        y = (h * _spread(s["C"], s)).sum(2) + D * x
        if gate is not None:
            y = y * gate * _sigmoid(gate)
        return y.to(X.dtype), h.transpose(1, 2).contiguous()
    rows, ok = _rows(s)
    x, d = _padded(X, rows, ok), _padded(step, rows, ok)
    Bs, Cs = _spread(_padded(s["B"], rows, ok), s), _spread(_padded(s["C"], rows, ok), s)
    a = torch.exp(d[..., None] * A)
    inputs = (d * x)[..., None] * Bs
    if s["state"] is not None:
        inputs[:, 0] += a[:, 0] * s["state"].transpose(1, 2)
    h = _recur(a, inputs)
    y = (h * Cs).sum(3) + D * x
    if s["gate"] is not None:
        gate = _padded(s["gate"], rows, ok)
        sig = _sigmoid(gate)
        Y = y * gate * sig
    else:
        Y = y
    Y = _packed(Y, rows, ok, X)
    if s["call"] == "forward":
        # (steps behind a region's end have d = 0: the state stays)
        return (Y, h[:, -1].transpose(1, 2).contiguous()) if s["state"] is not None else Y
    dy = _padded(s["dY"], rows, ok)
    if s["gate"] is not None:
        dgate = dy * y * sig * (1 + gate * (1 - sig))
        dy = dy * gate * sig
    later = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _recur(later.flip(1), (dy[..., None] * Cs).flip(1)).flip(1)
    before = a * torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)          # a[t] h[t-1]
    dC, dB = _gathered(dy[..., None] * h, s), _gathered(g * (d * x)[..., None], s)
    gB, gah = (g * Bs).sum(3), g * before
    dX = d * gB + D * dy
    dd = (x * gB + (gah * A).sum(3)) * _padded(slope, rows, ok)
    return (Y, _packed(dX, rows, ok, X), _packed(dd, rows, ok, X), (gah * d[..., None]).sum((0, 1)).t().contiguous(),
            _packed(dB, rows, ok, s["B"]), _packed(dC, rows, ok, s["C"]), (dy * x).sum((0, 1))[None],
            _packed(dgate, rows, ok, X) if s["gate"] is not None else 0.0, dd.sum((0, 1))[None])


# ---------------------------------------------------------------------------------------------- the package's calls
def _own_norm(s):
    from deepbind_amd import smat as sm
    Z, stats = sm.layernorm(s["X"], s["gamma"], s["beta"], nchunk=s["models"], eps=EPS, want_stats=s["call"] == "train", out=s["out"])
    if s["call"] == "forward":
        return Z
    return (Z,) + tuple(sm.layernorm_bprop(s["X"], s["gamma"], stats, s["dZ"], nchunk=s["models"], out=s["dout"]))


def _own_conv(s):
    from deepbind_amd import kangaroo_smat as ks
    if s["call"] == "token":
        return ks.causalconv_step(s["X"], s["W"], s["b"], s["state"], into=s["next"], out=s["out"]), s["next"]
    Z, _ = ks.causalconv(s["X"], s["W"], s["b"], s["R"], out=s["out"])
    if s["call"] == "forward":
        return Z
    return (Z,) + tuple(ks.causalconv_bprop(s["X"], s["W"], s["b"], s["R"], s["dZ"], out=s["dout"]))


def _own_scan(s):
    from deepbind_amd import kangaroo_smat as ks
    more = dict(D=s["D"], gate=s["gate"], dt_bias=s["bias"], softplus=True)
    if s["call"] == "token":
        return ks.statescan_step(s["X"], s["dt"], s["A"], s["B"], s["C"], s["state"], into=s["next"], out=s["out"], **more), s["next"]
    if s["call"] == "forward":
        Y, last = ks.statescan(s["X"], s["dt"], s["A"], s["B"], s["C"], s["R"], state=s["state"], want_state=s["state"] is not None, out=s["out"], **more)
        return Y if last is None else (Y, last)
    keep = ks.kept_states(s["X"], s["A"])
    Y, _ = ks.statescan(s["X"], s["dt"], s["A"], s["B"], s["C"], s["R"], keep=keep, out=s["out"], **more)
    grads = ks.statescan_bprop(s["X"], s["dt"], s["A"], s["B"], s["C"], s["R"], keep, s["dY"], out=s["dout"], **more)
    return (Y,) + tuple(0.0 if g is None else g for g in grads)


def run(state):
    if own:
        return {"norm": _own_norm, "conv": _own_conv, "scan": _own_scan}[state["kind"]](state)
    return {"norm": _norm, "conv": _conv, "scan": _scan}[state["kind"]](state)


def work(case):
    b = {"float32": 4, "float64": 8, "bfloat16": 2}[case["type"]]
    wb = 8 if b == 8 else 4
    train = case["call"] == "train"
    if case["kind"] == "norm":
        e = case["rows"] * case["models"] * case["width"]
        return {"bytes": e * b * (4 if train else 2), "flops": e * (24 if train else 9)}
    table = _plan(case)
    rows = int((table[:, 1] - table[:, 0]).sum())
    e = rows * case["channels"]
    if case["kind"] == "conv":
        K = case["taps"]
        state = 2 * case["count"] * (K - 1) * case["channels"] * b if case["call"] == "token" else 0
        return {"bytes": e * b * (4 if train else 2) + state, "flops": e * ((6 * K + 20) if train else 2 * K + 6)}
    S, weights = case["states"], 2 * rows * case["groups"] * case["states"] * wb
    gate = 1 if case["gate"] else 0
    state = 2 * case["count"] * S * case["channels"] * wb if case["carried"] else 0
    if train:       # X, dt, gate, dY in; Y, dX, ddt, dgate out; per step and state 7 operations forward, 15 backward
        return {"bytes": e * b * (6 + 2 * gate) + 2 * weights, "flops": e * (22 * S + 40)}
    return {"bytes": e * b * (3 + gate) + weights + state, "flops": e * (7 * S + 20)}


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in prepare(case, seed).items()
         if k not in ("out", "dout", "next")}
    if case["kind"] == "norm":
        X, g, b, w = s["X"], s["gamma"], s["beta"], case["width"]
        blocks, Z, dX, dg = X.split(w, 1), [], [], []
        for i, x in enumerate(blocks):
            gi = g[:, i * w:(i + 1) * w]
            mean = x.sum(1, keepdim=True) / w
            var = ((x - mean) ** 2).sum(1, keepdim=True) / w
            h = (x - mean) * (var + EPS) ** -0.5
            Z.append(h * gi + b[:, i * w:(i + 1) * w])
            if case["call"] == "train":
                d = s["dZ"][:, i * w:(i + 1) * w]
                q = d * gi
                dX.append((var + EPS) ** -0.5 * (q - q.sum(1, keepdim=True) / w - h * (q * h).sum(1, keepdim=True) / w))
                dg.append((d * h).sum(0, keepdim=True))
        return torch.cat(Z, 1) if case["call"] == "forward" else (torch.cat(Z, 1), torch.cat(dX, 1), torch.cat(dg, 1), s["dZ"].sum(0, keepdim=True))
    D, R = case["channels"], _plan(case)
    start, length = torch.from_numpy(R[:, 0]).to(DEVICE), torch.from_numpy(R[:, 1] - R[:, 0]).to(DEVICE)
    longest, n = int(length.max()), s["X"].shape[0]
    silu = lambda v: v / (1 + torch.exp(-v))  # noqa: E731

    def dsilu(v):
        p = 1 / (1 + torch.exp(-v))
        return p + v * p * (1 - p)

    if case["kind"] == "conv":
        K, W, b, X = case["taps"], s["W"], s["b"], s["X"]
        if case["call"] == "token":
            pre = b + W[K - 1] * X
            for j in range(K - 1):
                pre = pre + W[j] * s["state"][:, j]
            return silu(pre), torch.cat([s["state"][:, 1:], X[:, None]], 1)[:, :K - 1]
        # place of every row in its region, -1 outside
        place = torch.full((n,), -1, dtype=torch.long, device=DEVICE)
        for a, z in R.tolist():
            place[a:z] = torch.arange(z - a, device=DEVICE)
        inside = (place >= 0)[:, None]
        back = lambda t, j: torch.where((place >= j)[:, None], torch.roll(t, j, 0), 0)          # row t - j of the same region  # noqa: E731
        pre = b + sum(W[K - 1 - j] * back(X, j) for j in range(K))
        Z = torch.where(inside, silu(pre), 0)
        if case["call"] == "forward":
            return Z
        dpre = torch.where(inside, s["dZ"] * dsilu(pre), 0)
        dX = torch.zeros_like(X)
        for j in range(K):                               # row t sends w[K-1-j] dpre[t] to row t - j
            dX += torch.roll(torch.where((place >= j)[:, None], W[K - 1 - j] * dpre, 0), -j, 0)
        dW = torch.stack([(back(X, K - 1 - j) * dpre).sum(0) for j in range(K)])
        return Z, dX, dW, dpre.sum(0, keepdim=True)
    S, G, P = case["states"], case["groups"], case["count"]
    group = torch.arange(D, device=DEVICE) // (D // G)
    A, skip, gated = s["A"], s["D"], s["gate"] is not None                      # (states, channels)
    soft = lambda v: torch.where(v > 30, v, torch.log1p(torch.exp(torch.clamp(v, max=30))))  # noqa: E731
    if case["call"] == "token":
        d = soft(s["dt"] + s["bias"])
        Bt, Ct = (s[k].view(P, G, S)[:, group].transpose(1, 2) for k in ("B", "C"))             # (regions, states, channels)
        h = torch.exp(d[:, None] * A) * s["state"] + Bt * (d * s["X"])[:, None]
        y = (h * Ct).sum(1) + skip * s["X"]
        return (y * silu(s["gate"]) if gated else y), h
    if longest > 25000 or (case["call"] == "train" and longest * P * D * S > 800000000):       # (every step's states are held)
        return None
    by_length = torch.argsort(length, descending=True)   # so that the regions that still run are the first ones
    start, length = start[by_length], length[by_length]
    alive = (length[None, :] > torch.arange(longest, device=DEVICE)[:, None]).sum(1).tolist()
    train = case["call"] == "train"
    h = s["state"][by_length] if s["state"] is not None else torch.zeros((P, S, D), dtype=torch.float64, device=DEVICE)
    d_all, raw = soft(s["dt"] + s["bias"]), s["dt"] + s["bias"]
    B3, C3 = s["B"].reshape(n, G, S), s["C"].reshape(n, G, S)
    y_all, hs = torch.zeros_like(s["X"]), []
    h = h.clone()
    for t in range(longest):
        k = alive[t]
        at = start[:k] + t
        d, x = d_all[at], s["X"][at]
        hs.append(h[:k].clone() if train else None)
        h[:k] = torch.exp(d[:, None] * A) * h[:k] + B3[at][:, group].transpose(1, 2) * (d * x)[:, None]
        y_all[at] = (h[:k] * C3[at][:, group].transpose(1, 2)).sum(1) + skip * x
    Y = y_all * silu(s["gate"]) if gated else y_all
    if not train:
        last = torch.empty_like(h)
        last[by_length] = h
        return (Y, last) if s["state"] is not None else Y
    inside = torch.zeros((n, 1), dtype=torch.bool, device=DEVICE)
    for a, z in R.tolist():
        inside[a:z] = True
    dy = torch.where(inside, s["dY"] * silu(s["gate"]) if gated else s["dY"], 0)
    dgate = torch.where(inside, s["dY"] * y_all * dsilu(s["gate"]), 0) if gated else 0.0
    dX, dd = skip * dy, torch.zeros_like(dy)
    dA, dB, dC = torch.zeros_like(A), torch.zeros_like(B3), torch.zeros_like(C3)
    g = torch.zeros((P, S, D), dtype=torch.float64, device=DEVICE)              # what the later rows send to the state
    summed = lambda v: v.reshape(v.shape[0], S, G, D // G).sum(3).transpose(1, 2)  # noqa: E731
    for t in range(longest - 1, -1, -1):
        k = alive[t]
        at = start[:k] + t
        d, x, e = d_all[at], s["X"][at], dy[at]
        Bt, Ct = B3[at][:, group].transpose(1, 2), C3[at][:, group].transpose(1, 2)
        a = torch.exp(d[:, None] * A)
        now = g[:k] + Ct * e[:, None]
        kept = a * hs[t]
        dC[at] = summed((kept + Bt * (d * x)[:, None]) * e[:, None])
        dB[at] = summed(now * (d * x)[:, None])
        sent = (now * Bt).sum(1)
        dX[at] += d * sent
        dd[at] = x * sent + (now * kept * A).sum(1)
        dA += (now * kept * d[:, None]).sum(0)
        g[:k] = a * now
        hs[t] = None
    draw_dt = dd / (1 + torch.exp(-raw))
    return (Y, dX, draw_dt, dA, dB.reshape(n, G * S), dC.reshape(n, G * S), (dy * s["X"]).sum(0, keepdim=True), dgate, draw_dt.sum(0, keepdim=True))
