"""Plain 64-bit restatement of the gated delta rule, of the norms around a block and of gradient clipping, with bounds on what rounding
may do to each result.

Delta rule: `delta` is the definition, row by row, and its gradient by the definition's own chain. `delta_bounds` bounds, in units of the unit
roundoff u, how far a computation of the chunked form may be from it, by a running first-order error analysis: a sum of n products is off by
at most n u times the sum of their sizes (Euclidean norms where vectors meet, so that a product of vectors of norms a and b is at most a b),
a product adds its factors' relative errors and one u. What a chunk of 16 rows adds is added up by sizes; what was wrong in the state before it
passes on as the state itself does, and a row's map I - b k k^T lengthens no vector by more than max(1, |1 - b k.k|)."""
import numpy as np

from tests.rows_ref import rows_of, sigmoid

CHUNK = 16


def _split(t, n):
    return t.reshape(t.shape[0], n, -1)


def delta(Q, K, V, beta, decay, regions, G, scale, state=None, dO=None):
    """(O, last) or, with dO, (O, last, dQ, dK, dV, dbeta, ddecay); rows in no region are nan."""
    N, H = beta.shape
    of = np.arange(H) // (H // G)
    q, k, v = _split(Q, G)[:, of], _split(K, G)[:, of], _split(V, H)
    Kd, Vd = q.shape[2], v.shape[2]
    a = np.exp(decay) if decay is not None else np.ones_like(beta)
    O = np.full((N, H, Vd), np.nan)
    last = np.zeros((len(regions), Kd, H * Vd))
    g = dict(q=np.full((N, H, Kd), np.nan), k=np.full((N, H, Kd), np.nan), v=np.full((N, H, Vd), np.nan), b=np.full((N, H), np.nan), a=np.full((N, H), np.nan))
    for r, (s, e) in enumerate(rows_of(regions, N)):
        S = np.zeros((H, Kd, Vd)) if state is None else state[r].reshape(Kd, H, Vd).transpose(1, 0, 2).copy()
        held = []
        for t in range(s, e):
            old = a[t][:, None, None] * S
            miss = v[t] - np.einsum("hk,hkv->hv", k[t], old)
            held.append((S, old, miss))
            S = old + k[t][:, :, None] * (beta[t][:, None] * miss)[:, None]
            O[t] = scale * np.einsum("hk,hkv->hv", q[t], S)
        last[r] = S.transpose(1, 0, 2).reshape(Kd, H * Vd)
        if dO is None:
            continue
        dS = np.zeros_like(S)
        for t in range(e - 1, s - 1, -1):
            before, old, miss = held[t - s]
            d = scale * dO[t].reshape(H, Vd)
            b = beta[t][:, None]
            g["q"][t] = np.einsum("hkv,hv->hk", old + k[t][:, :, None] * (b * miss)[:, None], d)
            new = dS + q[t][:, :, None] * d[:, None]
            du = np.einsum("hk,hkv->hv", k[t], new)
            g["b"][t] = (du * miss).sum(1)
            g["v"][t] = b * du
            g["k"][t] = np.einsum("hkv,hv->hk", new, b * miss) - np.einsum("hkv,hv->hk", old, b * du)
            dold = new - k[t][:, :, None] * (b * du)[:, None]
            g["a"][t] = a[t] * (dold * before).sum((1, 2))
            dS = a[t][:, None, None] * dold
    O = O.reshape(N, -1)
    if dO is None:
        return O, last
    shared = lambda t: t.reshape(N, G, H // G, Kd).sum(2).reshape(N, G * Kd)  # noqa: E731
    return O, last, shared(g["q"]), shared(g["k"]), g["v"].reshape(N, -1), g["b"], g["a"]


def _row(x):
    return np.sqrt((x * x).sum(-1))


def delta_bounds(Q, K, V, beta, decay, regions, G, scale, state=None, dO=None, segment=0):
    """Bounds in units of u of delta()'s values, in its order: per row and head, so the same for all of a head's columns. segment: rows of the
    segments that long regions may be cut into: what is wrong at their borders is carried by products of transitions of at most
    `key` columns, one for each segment before."""
    N, H = beta.shape
    of = np.arange(H) // (H // G)
    q, k, v = _split(Q, G)[:, of], _split(K, G)[:, of], _split(V, H)
    Kd, Vd = q.shape[2], v.shape[2]
    P = len(regions)
    eO, eS = np.full((N, H), np.nan), np.zeros((P, H))
    eq, ek, ev, eb, eg = (np.full((N, H), np.nan) for _ in range(5))
    fro = lambda x: np.sqrt((x * x).sum())  # noqa: E731
    for h in range(H):
        for r, (s, e) in enumerate(rows_of(regions, N)):
            S = np.zeros((Kd, Vd)) if state is None else state[r].reshape(Kd, H, Vd)[:, h]
            E, chunks = 0.0, []
            for c in range(s, e, CHUNK):
                n = min(CHUNK, e - c)
                kk, qq, vv, b = k[c:c + n, h], q[c:c + n, h], v[c:c + n, h], beta[c:c + n, h]
                gg = decay[c:c + n, h] if decay is not None else np.zeros(n)
                low = np.tril(np.ones((n, n)))
                D = np.array([[np.exp(gg[j + 1:i + 1].sum()) if j <= i else 0.0 for j in range(n)] for i in range(n)])
                first, last = np.exp(np.cumsum(gg)), D[n - 1]
                kn, qn, ab = _row(kk), _row(qq), np.abs(b)
                L = b[:, None] * D * np.tril(kk @ kk.T, -1)
                T = np.linalg.inv(np.eye(n) + L)
                T = np.tril(T)
                aT = np.abs(T)
                l = np.tril(ab[:, None] * D * np.outer(kn, kn), -1)
                eT = aT @ (((Kd + 6) + 18) * l) @ aT
                x = vv - first[:, None] * (kk @ S)
                u = T @ (b[:, None] * x)
                xs, us = _row(vv) + first * kn * fro(S), _row(u)
                ex = (Kd + 6) * xs
                eu = eT @ (ab * xs) + aT @ (ab * ex) + 20 * (aT @ (ab * xs))
                grow = np.array([max(1.0, abs(1 - b[i] * kn[i] ** 2)) for i in range(n)])
                rho = first * np.cumprod(grow)
                # the state's own error reaches row i through the rows up to it
                tu = eu + ab * kn * rho * E
                tx = ex + first * kn * E
                sizeP = D * np.outer(qn, kn) * low
                eO[c:c + n, h] = scale * (qn * rho * E + first * qn * (Kd + 8) * fro(S) + sizeP @ eu + (Kd + 28) * (sizeP @ np.maximum(us, aT @ (ab * xs)))) + 2 * scale * qn * fro(S)
                chunks.append((c, n, kk, qq, b, D, first, last, kn, qn, ab, T, aT, eT, x, xs, tx, u, np.maximum(us, aT @ (ab * xs)), tu, S, E, rho, sizeP, l))
                S1 = first[-1] * S + (kk * last[:, None]).T @ u
                E = rho[-1] * E + 3 * first[-1] * fro(S) + (last * kn) @ (eu + 24 * np.maximum(us, aT @ (ab * xs)))
                if segment and (c - s) // segment != (c + n - s) // segment:
                    E += 4 * (Kd + 8) * (fro(S1) + E * 0) * max(1.0, Kd ** 0.5)
                S = S1
            eS[r, h] = E
            if dO is None:
                continue
            dS, F = np.zeros((Kd, Vd)), 0.0
            for (c, n, kk, qq, b, D, first, last, kn, qn, ab, T, aT, eT, x, xs, tx, u, us, tu, S, E, rho, sizeP, l) in reversed(chunks):
                d = scale * dO[c:c + n].reshape(n, H, Vd)[:, h]
                dn, f, f0 = _row(d), fro(dS), fro(S)
                du = (D * (qq @ kk.T) * np.tril(np.ones((n, n)))).T @ d + last[:, None] * (kk @ dS)
                dy = T.T @ du
                sdu = sizeP.T @ dn + last * kn * f
                sdy = aT.T @ sdu
                edy = aT.T @ ((Kd + 30) * sdu) + eT.T @ sdu + 20 * sdy
                # what is wrong behind the chunk reaches row j through the rows behind it
                back = rho[-1] / np.maximum(rho, 1e-300) * kn * F
                tdy = edy + back
                ev[c:c + n, h] = ab * (tdy + 2 * sdy)
                edP = np.outer(dn, tu) + (Vd + 6) * np.outer(dn, us)                 # of dP and of dL, entry by entry
                sdP = np.outer(dn, us)
                edL = np.outer(tdy, us) + np.outer(sdy, tu) + (Vd + 6) * np.outer(sdy, us)
                sdL = np.outer(sdy, us)
                low = np.tril(np.ones((n, n)))
                A_, Ae = D * low * sdP, D * low * (edP + 24 * sdP)
                strict = np.tril(np.ones((n, n)), -1)
                M_, Me = ab[:, None] * D * strict * sdL, ab[:, None] * D * strict * (edL + 24 * sdL)
                qst, eqst = first * dn * f0, first * dn * (E + (Vd + 8) * f0)
                ker, eker = first * ab * sdy * f0, first * ab * (tdy * f0 + sdy * (E + (Vd + 8) * f0))
                kin, ekin = last * us * f, last * (tu * f + us * (F + (Vd + 8) * f))
                eq[c:c + n, h] = eqst + Ae @ kn + 4 * (qst + A_ @ kn)
                ek[c:c + n, h] = eker + ekin + Ae.T @ qn + Me @ kn + Me.T @ kn + 8 * (ker + kin + A_.T @ qn + M_ @ kn + M_.T @ kn)
                nn = np.outer(kn, kn) * D * strict
                eb[c:c + n, h] = tdy * xs + sdy * tx + (Vd + 8) * sdy * xs + ((edL + (Kd + 28) * sdL) * nn).sum(1) + 6 * (sdy * xs + (sdL * nn).sum(1))
                pe = edP * sizeP + (Kd + 10) * sdP * sizeP + edL * l + (Kd + 12) * sdL * l
                ps = sdP * sizeP + sdL * l
                into_e, into_s = qn * eqst + kn * eker + (Kd + 12) * (qn * qst + kn * ker), qn * qst + kn * ker
                out_e, out_s = kn * ekin + (Kd + 12) * kn * kin, kn * kin
                thr_e, thr_s = first[-1] * (E * f + f0 * F + (Kd * Vd + 8) * f0 * f), first[-1] * f0 * f
                for m in range(n):
                    eg[c + m, h] = (pe[m:, :m].sum() + into_e[m:].sum() + out_e[:m].sum() + thr_e
                                    + 50 * (ps[m:, :m].sum() + into_s[m:].sum() + out_s[:m].sum() + thr_s))
                F = rho[-1] * F + 4 * first[-1] * f + (kn * first * ab) @ (edy + 28 * sdy) + 28 * ((qn * first) @ dn)
                dS1 = first[-1] * dS - kk.T @ ((first * b)[:, None] * dy) + (qq * first[:, None]).T @ d
                if segment and c > s and (c - s) % segment == 0:
                    F += 4 * (Kd + 8) * fro(dS1) * max(1.0, Kd ** 0.5)
                dS = dS1
    spread = lambda t, w: np.repeat(t, w, axis=1)  # noqa: E731
    # a state of the norm E is off by at most E anywhere
    states = np.repeat(eS[:, None, :], Kd, 1).repeat(Vd, 2)
    if dO is None:
        return spread(eO, Vd), states
    keys = lambda t: spread(t.reshape(N, G, H // G).sum(2), Kd)  # noqa: E731
    return spread(eO, Vd), states, keys(eq), keys(ek), spread(ev, Vd), eb, eg


def _chunked(X, w):
    return X.reshape(X.shape[0], -1, w)


def _norm(X, w, rms, eps):
    """h, mean, reciprocal deviation, and the size of h: what rounding x - mean costs, relative to h's one."""
    V = _chunked(X, w)
    mean = np.zeros(V.shape[:2] + (1,)) if rms else V.mean(2, keepdims=True)
    c = V - mean
    r = 1 / np.sqrt((c * c).mean(2, keepdims=True) + eps)
    size = (np.abs(V) if rms else np.abs(V) + np.abs(V).mean(2, keepdims=True)) * r
    return c * r, mean, r, size


def blocknorm(Y, R, gate, gamma, beta, scale, ngamma, nbeta, nchunk, rms, norm, nxt, eps, store=lambda x: x, kept=None):
    """values: (O, Z|None, what the gradient takes); sizes: (O, Z|None). store: the rounding of O as it is kept, which Z is made of; kept: O as a
    computation stored it, in place of store(O)."""
    n, m = Y.shape
    w = m // nchunk
    h, _, r, hs = _norm(Y, w, rms, eps) if norm else (_chunked(Y, w), None, np.ones((n, nchunk, 1)), np.abs(_chunked(Y, w)))
    p, ps = h.reshape(n, m) * gamma + beta, hs.reshape(n, m) * np.abs(gamma) + np.abs(beta)
    act = np.ones_like(p) if gate is None else gate * sigmoid(gate)
    acts = np.abs(act) * (1 if gate is None else 1 + np.abs(gate))
    O = R + scale * p * act
    Os = np.abs(R) + np.abs(scale) * ps * acts
    if not nxt:
        return (O, None, (h, r, p, act)), (Os, None, (hs, ps, acts))
    held = store(O) if kept is None else kept
    h2, _, r2, h2s = _norm(held, w, rms, eps)
    return (O, h2.reshape(n, m) * ngamma + nbeta, (h, r, p, act, h2, r2)), (Os, h2s.reshape(n, m) * np.abs(ngamma) + np.abs(nbeta), (hs, ps, acts, h2s))


def blocknorm_bprop(Y, R, gate, gamma, beta, scale, ngamma, nbeta, nchunk, rms, norm, nxt, eps, dR, dZ, kept):
    """values and sizes of (dY, dR, dgate, dgamma, dbeta, dscale, dnext_gamma, dnext_beta); kept: O as the forward call stored it."""
    n, m = Y.shape
    w = m // nchunk
    f, s = blocknorm(Y, R, gate, gamma, beta, scale, ngamma, nbeta, nchunk, rms, norm, nxt, eps, kept=kept)
    (h, r, p, act), (hs, ps, acts) = f[2][:4], s[2][:3]
    flat = lambda t: t.reshape(n, m)  # noqa: E731

    def back(q, qs, h, hs, r):
        q, qs = _chunked(q, w), _chunked(qs, w)
        d = q - h * (q * h).mean(2, keepdims=True) - (0 if rms else q.mean(2, keepdims=True))
        # (h's own error reaches everything in its chunk by its largest size)
        ds = hs.max(2, keepdims=True) * (qs + hs * (qs * hs).mean(2, keepdims=True) + (0 if rms else qs.mean(2, keepdims=True)))
        return flat(r * d), flat(r * ds)

    t, ts = dR.copy(), np.abs(dR)
    zero = np.zeros((1, m))
    dng = dngs = dnb = dnbs = zero
    if nxt:
        h2, r2, h2s = f[2][4], f[2][5], s[2][3]
        b, bs = back(dZ * ngamma, np.abs(dZ * ngamma), h2, h2s, r2)
        t, ts = t + b, ts + bs
        dng, dngs = (dZ * flat(h2)).sum(0, keepdims=True), (np.abs(dZ) * flat(h2s)).sum(0, keepdims=True)
        dnb, dnbs = dZ.sum(0, keepdims=True), np.abs(dZ).sum(0, keepdims=True)
    dp, dps = t * scale * act, ts * np.abs(scale) * acts
    g = zero if gate is None else gate
    e = sigmoid(g)
    open_, opens = e * (1 + g * (1 - e)), e * (1 + np.abs(g)) ** 2
    dgate, dgates = t * scale * p * open_, ts * np.abs(scale) * ps * opens
    dY, dYs = back(dp * gamma, dps * np.abs(gamma), h, hs, r) if norm else (dp * gamma, dps * np.abs(gamma))
    rows = lambda x: x.sum(0, keepdims=True)  # noqa: E731
    return ((dY, t, dgate, rows(dp * flat(h)), rows(dp), rows(t * p * act), dng, dnb),
            (dYs, ts, dgates, rows(dps * flat(hs)), rows(dps), rows(ts * ps * acts), dngs, dnbs))


def clip(grads, max_norm, nblock, by_rows):
    """norms and scaled gradients"""
    blocks = [np.split(t, nblock, axis=0 if r else t.ndim - 1) for t, r in zip(grads, by_rows)]
    norms = np.array([np.sqrt(sum((b[i] ** 2).sum() for b in blocks)) for i in range(nblock)])
    factor = [max_norm / n if n > max_norm else 1.0 for n in norms]
    return norms, [np.concatenate([b[i] * factor[i] for i in range(nblock)], axis=0 if r else t.ndim - 1) for t, b, r in zip(grads, blocks, by_rows)]
