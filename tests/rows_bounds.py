"""Running error analysis of the state scan: how far each result of a computation in unit roundoff u may be from the definition in 64
bits, row by row, so that a bound follows how long the decays remember and not how long a region is.

Every quantity is a pair: s, the sum of the absolute values of its terms, and k, its error's first-order bound in units of u. A product adds the
factors' relative errors and one rounding, a sum the terms' errors and one rounding of what it may hold. 2^x and reciprocals are within one unit
in the last place (2 u); the argument of an exponential, x log2(e) or d (A log2(e)), carries two roundings, which act through its size."""
import numpy as np

from tests import rows_ref as ref


def mul(a, b):
    s = a[0] * b[0]
    return s, a[1] * b[0] + a[0] * b[1] + s


def add(a, b):
    s = a[0] + b[0]
    return s, a[1] + b[1] + s


def exact(v):
    return np.abs(v), np.zeros_like(v)


def summed(a, axis, n):
    """The sum over an axis of n terms in any order."""
    s = a[0].sum(axis)
    return s, a[1].sum(axis) + n * s


def sigmoid(v):
    # e^-v within 2 |v| + 2, 1 + e one rounding, its reciprocal two, and one for a product on the way
    p = ref.sigmoid(v)
    return p, p * (2 * np.abs(v) + 6)


def steps(dt, bias, soft):
    """d = softplus(dt + bias) and its slope, or dt + bias."""
    raw = dt + bias
    if not soft:
        return raw, (np.abs(raw), np.abs(raw)), (np.ones_like(raw), np.zeros_like(raw))
    d, p = ref.softplus(raw), ref.sigmoid(raw)
    # max(raw, 0) + log(1 + e), e = exp(-|raw|) within 2 |raw| + 2 and a dozen roundings on to the logarithm; raw's own rounding acts through the slope
    k = p * np.abs(raw) + np.log1p(np.exp(-np.abs(raw))) * (2 * np.abs(raw) + 12) + d
    slope = sigmoid(raw)
    return d, (d, k), (slope[0], slope[1] + p * (1 - p) * np.abs(raw))


def statescan(X, dt, A, B, C, regions, D, gate, bias, soft=True, state=None, dY=None, segment=0):
    """Error bounds in units of u of rows_ref.statescan's values, in its order. segment: the rows of the segments that regions may be cut
    into; a state then passes a segment by exp(A * sum of its steps), and a sum of L steps is off by L u times itself."""
    N, n = X.shape
    S = A.shape[0]
    G = B.shape[1] // S
    of = np.arange(n) // (n // G)
    v = {k: np.full((N, n), np.nan) for k in ("Y", "dX", "ddt", "dgate")}
    v["dB"], v["dC"] = np.full((N, G * S), np.nan), np.full((N, G * S), np.nan)
    total = {k: (np.zeros(s), np.zeros(s)) for k, s in (("dA", (S, n)), ("dD", (1, n)), ("dbias", (1, n)))}
    v["last"] = np.zeros((len(regions), S, n))
    channels = lambda t: summed((t[0].reshape(S, G, -1), t[1].reshape(S, G, -1)), 2, n // G + 8)[1].T.reshape(-1)  # noqa: E731
    rows = sum(e - s for s, e in ref.rows_of(regions, N))

    def into(k, t):
        total[k] = (total[k][0] + t[0], total[k][1] + t[1])

    for r, (s, e) in enumerate(ref.rows_of(regions, N)):
        h = exact(np.zeros((S, n)) if state is None else state[r])
        d_, d, slope = steps(dt[s:e], bias, soft)
        hist = []
        for t in range(e - s):
            x, dn = exact(X[s + t]), (d[0][t], d[1][t])
            Bt, Ct = (exact(m[s + t].reshape(G, S)[of].T) for m in (B, C))
            arg = np.abs(d_[t] * A)
            a = np.exp(d_[t] * A)
            a = (a, a * (np.abs(A) * dn[1] + (2 + segment) * arg + 2))
            hist.append((h, a))
            h = add(mul(a, h), mul(mul(dn, x), Bt))
            y = add(summed(mul(Ct, h), 0, S + 4), mul(exact(D[0]), x))
            if gate is not None:
                g = gate[s + t]
                p = sigmoid(g)
                if dY is not None:
                    v["dgate"][s + t] = mul(mul(y, exact(dY[s + t])), mul(p, (1 + np.abs(g) * (1 - p[0]), (4 + 3 * np.abs(g)) * (1 + np.abs(g)))))[1]
                y = mul(y, mul(exact(g), p))
            v["Y"][s + t] = y[1]
        v["last"][r] = h[1]
        if dY is None:
            continue
        back, after = exact(np.zeros((S, n))), h
        for t in range(e - s - 1, -1, -1):
            x, dn = exact(X[s + t]), (d[0][t], d[1][t])
            Bt, Ct = (exact(m[s + t].reshape(G, S)[of].T) for m in (B, C))
            before, a = hist[t]
            dy = exact(dY[s + t])
            if gate is not None:
                dy = mul(dy, mul(exact(gate[s + t]), sigmoid(gate[s + t])))
            now = add(back, mul(Ct, dy))
            v["dC"][s + t] = channels(mul((dy[0] * np.ones_like(after[0]), dy[1] * np.ones_like(after[0])), after))
            v["dB"][s + t] = channels(mul(now, mul(dn, x)))
            gB = summed(mul(now, Bt), 0, S + 4)
            w = mul(now, mul(a, before))
            v["dX"][s + t] = add(mul(dn, gB), mul(exact(D[0]), dy))[1]
            wA = mul(w, (np.abs(A), 3 * np.abs(A)))
            dd = mul(add(mul(x, gB), summed(wA, 0, S + 4)), (slope[0][t], slope[1][t]))
            v["ddt"][s + t] = dd[1]
            into("dbias", (dd[0][None], dd[1][None]))
            into("dA", mul(w, dn))
            dD = mul(dy, x)
            into("dD", (dD[0][None], dD[1][None]))
            back, after = mul(a, now), before
    if dY is None:
        return v["Y"], v["last"]
    for k, (s, e) in total.items():
        v[k] = e + rows * s
    return tuple(v[k] for k in ("Y", "last", "dX", "ddt", "dA", "dB", "dC", "dD", "dgate", "dbias"))
