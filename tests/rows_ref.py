"""Plain 64-bit restatement of the row operators (layer norm, causal convolution, state scan), forward and backward, with a
bound on what rounding may do to each result.

Every function returns (values, sizes): `sizes` holds, per output, the same sums over the ABSOLUTE values of their terms. A
result that is computed with unit roundoff u by a chain of at most k roundings per term is off by at most about k u times that
size, whatever cancels; the tests multiply by the k they derive and add the rounding of the stored result."""
import numpy as np


def sigmoid(v):
    return np.where(v >= 0, 1 / (1 + np.exp(-np.abs(v))), np.exp(-np.abs(v)) / (1 + np.exp(-np.abs(v))))


def softplus(v):
    return np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v)))


def rows_of(regions, N):
    out = []
    for s, e in np.asarray(regions).astype(np.int64).tolist():
        s, e = min(s, N), min(e, N)
        out.append((s, max(s, e)))
    return out


def layernorm(X, gamma, beta, nchunk, eps):
    n, m = X.shape
    V = X.reshape(n, nchunk, -1)
    mean = V.mean(2, keepdims=True)
    c = V - mean
    r = 1 / np.sqrt((c * c).mean(2, keepdims=True) + eps)
    h = (c * r).reshape(n, m)
    # what rounding x - mean costs, relative to 1: the values' size over the deviation. The mean's own error is that of a sum of
    # signed terms: fl(sum x) is off by at most (w - 1) u sum |x|, so the mean by (w - 1) u mean |x|, however small it is itself
    size = ((np.abs(V) + np.abs(V).mean(2, keepdims=True)) * r).reshape(n, m)
    return (h * gamma + beta, mean.ravel(), r.ravel()), (size * np.abs(gamma) + np.abs(beta), np.abs(V).mean(2).ravel(), r.ravel() * size.reshape(n, nchunk, -1).max(2).ravel())


def layernorm_bprop(X, gamma, nchunk, eps, dZ):
    n, m = X.shape
    (h, _, r), (hs, _, _) = layernorm(X, np.ones((1, m)), np.zeros((1, m)), nchunk, eps)
    r = r.reshape(n, nchunk, 1)
    q = (dZ * gamma).reshape(n, nchunk, -1)
    H, HS = h.reshape(q.shape), hs.reshape(q.shape)
    dX = (r * (q - q.mean(2, keepdims=True) - H * (q * H).mean(2, keepdims=True))).reshape(n, m)
    a = np.abs(q)
    size = (r * HS.max(2, keepdims=True) * (a + a.mean(2, keepdims=True) + HS * (a * HS).mean(2, keepdims=True))).reshape(n, m)
    return (dX, (dZ * h).sum(0, keepdims=True), dZ.sum(0, keepdims=True)), (size, (np.abs(dZ) * hs).sum(0, keepdims=True), np.abs(dZ).sum(0, keepdims=True))


def _conv_pre(X, W, b, s, e, state):
    K, D = W.shape
    x = np.concatenate([np.zeros((K - 1, D)) if state is None else state, X[s:e]])
    pre = np.zeros((e - s, D)) + b
    for j in range(K):
        pre = pre + W[j] * x[j:j + e - s]
    return x, pre


def causalconv(X, W, b, regions, silu=True, state=None):
    """values: (Z, last); rows in no region are nan."""
    N, D = X.shape
    K = W.shape[0]
    Z, size = np.full((N, D), np.nan), np.full((N, D), np.nan)
    last = np.zeros((len(regions), K - 1, D))
    for r, (s, e) in enumerate(rows_of(regions, N)):
        x, pre = _conv_pre(X, W, b, s, e, None if state is None else state[r])
        _, ps = _conv_pre(np.abs(X), np.abs(W), np.abs(b), s, e, None if state is None else np.abs(state[r]))
        Z[s:e] = pre * sigmoid(pre) if silu else pre
        size[s:e] = ps * (1 + np.abs(pre)) if silu else ps
        last[r] = x[x.shape[0] - (K - 1):]
    return (Z, last), (size, np.abs(last))


def causalconv_bprop(X, W, b, regions, dZ, silu=True):
    N, D = X.shape
    K = W.shape[0]
    out, sizes = [], []
    dX, dXs = np.full((N, D), np.nan), np.full((N, D), np.nan)
    dW, dWs, db, dbs = np.zeros((K, D)), np.zeros((K, D)), np.zeros((1, D)), np.zeros((1, D))
    for s, e in rows_of(regions, N):
        if s == e:
            continue
        x, pre = _conv_pre(X, W, b, s, e, None)
        xs, ps = _conv_pre(np.abs(X), np.abs(W), np.abs(b), s, e, None)
        d, ds = dZ[s:e], np.abs(dZ[s:e])
        if silu:
            g = sigmoid(pre)
            d, ds = d * (g + pre * g * (1 - g)), ds * (1 + ps * (1 + np.abs(pre)))
        gx, gs = np.zeros((e - s + K - 1, D)), np.zeros((e - s + K - 1, D))
        for j in range(K):
            gx[j:j + e - s] += W[j] * d
            gs[j:j + e - s] += np.abs(W[j]) * ds
            dW[j] += (d * x[j:j + e - s]).sum(0)
            dWs[j] += (ds * xs[j:j + e - s]).sum(0)
        dX[s:e], dXs[s:e] = gx[K - 1:], gs[K - 1:]
        db += d.sum(0)
        dbs += ds.sum(0)
    return (dX, dW, db), (dXs, dWs, dbs)


def statescan(X, dt, A, B, C, regions, D, gate, bias, soft=True, state=None, dY=None):
    """values: (Y, last) or, with dY, (Y, last, dX, ddt, dA, dB, dC, dD, dgate, dbias), and their sizes; rows in no region nan."""
    N, n = X.shape
    S = A.shape[0]
    G = B.shape[1] // S
    of = np.arange(n) // (n // G)
    nan = lambda *s: np.full(s, np.nan)  # noqa: E731
    v = {k: nan(N, n) for k in ("Y", "dX", "ddt", "dgate")}
    z = {k: nan(N, n) for k in v}
    for k in ("dB", "dC"):
        v[k], z[k] = nan(N, G * S), nan(N, G * S)
    for k, s in (("dA", (S, n)), ("dD", (1, n)), ("dbias", (1, n)), ("last", (len(regions), S, n))):
        v[k], z[k] = np.zeros(s), np.zeros(s)
    add = lambda t: np.stack([t[:, of == g].sum(1) for g in range(G)]).reshape(-1)              # (S, n) -> (G * S)  # noqa: E731
    for r, (s, e) in enumerate(rows_of(regions, N)):
        h = np.zeros((S, n)) if state is None else state[r].copy()
        hz = np.abs(h)
        hist = []
        raw = dt[s:e] + bias
        d = softplus(raw) if soft else raw
        slope = sigmoid(raw) if soft else np.ones_like(raw)
        # a step's own rounding acts through exp(d A): (|dt| + |bias|) slope beside d itself
        ds = np.abs(d) + (np.abs(dt[s:e]) + np.abs(bias)) * slope
        for t in range(e - s):
            x = X[s + t]
            Bt, Ct = B[s + t].reshape(G, S)[of].T, C[s + t].reshape(G, S)[of].T
            a = np.exp(d[t] * A)
            az = a * (1 + ds[t] * np.abs(A))
            hist.append((h, hz, a, az))
            h = a * h + d[t] * x * Bt
            hz = a * hz * (1 + ds[t] * np.abs(A) / 16) + ds[t] * np.abs(x) * np.abs(Bt)         # (the tests take 16 roundings and more per step)
            y, yz = (Ct * h).sum(0) + D[0] * x, (np.abs(Ct) * hz).sum(0) + np.abs(D[0] * x)
            g = gate[s + t] if gate is not None else None
            v["Y"][s + t] = y if gate is None else y * g * sigmoid(g)
            z["Y"][s + t] = yz if gate is None else yz * np.abs(g) * sigmoid(g) * (1 + np.abs(g))
            if gate is not None and dY is not None:
                p = sigmoid(g)
                v["dgate"][s + t] = dY[s + t] * y * p * (1 + g * (1 - p))
                z["dgate"][s + t] = np.abs(dY[s + t]) * yz * p * (1 + np.abs(g)) ** 2
        v["last"][r], z["last"][r] = h, hz
        if dY is None:
            continue
        G_, Gz = np.zeros((S, n)), np.zeros((S, n))
        after, afterz = h, hz
        for t in range(e - s - 1, -1, -1):
            x, (before, beforez, a, az) = X[s + t], hist[t]
            Bt, Ct = B[s + t].reshape(G, S)[of].T, C[s + t].reshape(G, S)[of].T
            g = gate[s + t] if gate is not None else None
            dy = dY[s + t] if gate is None else dY[s + t] * g * sigmoid(g)
            dyz = np.abs(dy) * (1 if gate is None else 1 + np.abs(g))
            now, nowz = G_ + Ct * dy, Gz + np.abs(Ct) * dyz
            in_, inz = d[t] * x, ds[t] * np.abs(x)
            v["dC"][s + t], z["dC"][s + t] = add(dy * after), add(dyz * afterz)
            v["dB"][s + t], z["dB"][s + t] = add(now * in_), add(nowz * inz)
            gB, gBz = (now * Bt).sum(0), (nowz * np.abs(Bt)).sum(0)
            w, wz = now * a * before, nowz * az * beforez
            v["dX"][s + t], z["dX"][s + t] = d[t] * gB + D[0] * dy, ds[t] * gBz + np.abs(D[0]) * dyz
            dd, ddz = x * gB + (w * A).sum(0), np.abs(x) * gBz + (wz * np.abs(A)).sum(0)
            # (the slope's own relative rounding: as a sigmoid's, |raw| and a few)
            slz = slope[t] * (1 + np.abs(raw[t]))
            v["ddt"][s + t], z["ddt"][s + t] = dd * slope[t], ddz * slz
            v["dbias"] += dd * slope[t]
            z["dbias"] += ddz * slz
            v["dA"] += w * d[t]
            z["dA"] += wz * ds[t]
            v["dD"] += dy * x
            z["dD"] += dyz * np.abs(x)
            G_, Gz = a * now, nowz * a * (1 + ds[t] * np.abs(A) / 16)
            after, afterz = before, beforez
    keys = ("Y", "last") if dY is None else ("Y", "last", "dX", "ddt", "dA", "dB", "dC", "dD", "dgate", "dbias")
    return tuple(v[k] for k in keys), tuple(z[k] for k in keys)
