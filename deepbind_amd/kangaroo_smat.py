"""Sequence operators over device tensors: same names, argument order and in-place conventions
as the reference's operator shim (reference: code/libs/kangaroo/kangaroo/_ext/kangaroo_smat.py:86-146),
plus the fused scan+pool entry points. Arrays are torch tensors on the GPU; all arithmetic happens
in libdeepbind_hip.so on the current HIP stream.
"""
import ctypes

import torch

from . import _lib
from ._lib import DeepbindError, call, dtype_code, ptr, require, str2pooltype, stream

uindex = torch.uint32

_rng_seed = 0
_rng_offset = 0


def set_seed(seed):
    """Seeds the generator behind dropoutord_fp_train (and resets its stream position)."""
    global _rng_seed, _rng_offset
    _rng_seed, _rng_offset = int(seed), 0


def _u8(X):
    require(X.dtype == torch.uint8, "TypeError: X must be uint8, got %s" % X.dtype)
    return X


def _regions(R):
    require(R.dtype in (torch.uint32, torch.int32), "TypeError: regions must be uint32, got %s" % R.dtype)
    require(R.dim() == 2 and R.shape[1] in (2, 3), "ValueError: regions array must have 2 or 3 columns.")
    return R


def set_exact_scan(on):
    """on: corr1ord, corr1ord_bprop_W and corr1ord_bprop_X keep to the kernels that sum in one fixed order at every
    size (corr1ord: the reference's own order, so its bits whatever the batch size). Off (the default) float32 calls
    switch to the faster matrix-core kernels at bulk sizes, whose results equal these to round-off. Process-wide;
    returns the previous setting."""
    from ._lib import dll
    return bool(dll().dbk_set_exact_scan(int(bool(on))))


def corr1ord(W, X, Z, nchannel):
    """Cross-correlates the filter bank W ((M*nchannel) x P) with the ordinal vector X (N uint8,
    values 0..nchannel-1, 255 = all ordinals, 254 = none) into Z (N x P). The final M-1 rows of Z
    are left untouched. reference: kangaroo_smat.py:86-99, kangaroo_smat.cpp:98-124"""
    _u8(X)
    require(W.shape[0] % nchannel == 0, "ValueError: W rows must be a multiple of nchannel")
    require(W.dtype == Z.dtype, "TypeError: W dtype must match Z dtype")
    require(Z.shape[1] == W.shape[1], "ValueError: Z must have one column per filter")
    require(Z.shape[0] == X.numel(), "ValueError: Z must have one row per element of X")
    m = W.shape[0] // nchannel
    n = X.numel() - m + 1
    if n <= 0:
        return
    call("dbk_corr1ord", stream(), dtype_code(Z), ptr(W), m, W.shape[1], ptr(X), n, nchannel, ptr(Z))


def corr1ord_bprop_W(dW, X, dZ, nchannel):
    """Accumulates the filter gradient of corr1ord into dW. reference: kangaroo_smat.py:101-109"""
    _u8(X)
    require(dW.shape[0] % nchannel == 0, "ValueError: dW rows must be a multiple of nchannel")
    require(dW.dtype == dZ.dtype, "TypeError: dW dtype must match dZ dtype")
    require(dZ.shape[1] == dW.shape[1] and dZ.shape[0] == X.numel(), "ValueError: dZ must be N x P")
    m = dW.shape[0] // nchannel
    n = X.numel() - m + 1
    if n <= 0:
        return
    call("dbk_corr1ord_bprop_W", stream(), dtype_code(dZ), ptr(dW), m, dW.shape[1], ptr(X), n, nchannel, ptr(dZ))


def corr1ord_bprop_X(dX, W, dZ, nchannel):
    """Accumulates the input gradient of corr1ord into dX (N x nchannel). reference: kangaroo_smat.py:111-119,
    kangaroo_smat.cpp:141-168"""
    require(W.shape[0] % nchannel == 0, "ValueError: W rows must be a multiple of nchannel")
    require(W.dtype == dZ.dtype and dX.dtype == dZ.dtype, "TypeError: dX, W and dZ must share a dtype")
    require(dX.shape[1] == nchannel, "ValueError: dX must have nchannel columns")
    require(dZ.shape[1] == W.shape[1] and dZ.shape[0] == dX.shape[0], "ValueError: dZ must be N x P")
    m = W.shape[0] // nchannel
    call("dbk_corr1ord_bprop_X", stream(), dtype_code(dZ), ptr(dX), dX.shape[0], nchannel, ptr(W), m, W.shape[1], ptr(dZ))


def poolrgn(unpooledmaps, regions, ptype, want_argmax=False):
    """Pools rows of unpooledmaps (N x M) per region. Returns (pooled, argmax|None); "all" gives
    (P x 2M) with (max, avg) at columns (2j, 2j+1). reference: kangaroo_smat.py:121-132"""
    _regions(regions)
    noutputs = 2 if ptype == "all" else 1
    nregion, nfeaturemap = regions.shape[0], unpooledmaps.shape[1]
    pooledmaps = torch.empty((nregion, nfeaturemap * noutputs), dtype=unpooledmaps.dtype, device=unpooledmaps.device)
    argmax = None
    if ptype in ("max", "all") and want_argmax:
        argmax = torch.empty((nregion, nfeaturemap), dtype=uindex, device=unpooledmaps.device)
    call("dbk_poolrgn", stream(), dtype_code(unpooledmaps), ptr(unpooledmaps), nfeaturemap, ptr(regions), nregion,
         int(regions.shape[1] == 3), ptr(pooledmaps), ptr(argmax), str2pooltype[ptype])
    return pooledmaps, argmax


def poolrgn_bprop(unpooledmaps, regions, pooledmaps, pooledmaps_argmax, ptype):
    """Accumulates the pooling gradient into unpooledmaps. reference: kangaroo_smat.py:134-138"""
    _regions(regions)
    nregion, nfeaturemap = regions.shape[0], unpooledmaps.shape[1]
    noutputs = 2 if ptype == "all" else 1
    require(unpooledmaps.dtype == pooledmaps.dtype, "TypeError: unpooledmaps dtype must match pooledmaps dtype.")
    require(tuple(pooledmaps.shape) == (nregion, nfeaturemap * noutputs),
            "ValueError: pooledmaps must be (regions x feature maps%s)." % (" x 2" if noutputs == 2 else ""))
    amax = pooledmaps_argmax if (pooledmaps_argmax is not None and ptype in ("max", "all")) else None
    if amax is not None:
        require(tuple(amax.shape) == (nregion, nfeaturemap) and amax.dtype in (torch.uint32, torch.int32),
                "ValueError: pooledmaps_argmax must be a (regions x feature maps) uint32 array.")
    call("dbk_poolrgn_bprop", stream(), dtype_code(unpooledmaps), ptr(unpooledmaps), nfeaturemap, ptr(regions), nregion,
         int(regions.shape[1] == 3), ptr(pooledmaps), ptr(amax), str2pooltype[ptype])


def dropoutord_fp_train(X, rate, U=None, regions=None, padding=None, seed=None, offset=None, counter=None):
    """Input-base dropout: returns (Z, M) with dropped bases replaced by 254 (padding always passes and
    reports True in M). U (optional, float32, same shape) supplies the uniforms instead of the
    library's generator; `offset` / `counter` (device int64 tensor) supply the generator position
    instead of the module's host-side one. With `regions` (pairs of fwd/rev rows) and `padding` the reverse
    strand's mask is the forward strand's mirrored, as in reverse-complement training.
    reference: kangaroo_smat.py:140-146, kangaroo/_ext/dropoutord.py:50-70"""
    global _rng_offset
    _u8(X)
    Z = torch.empty_like(X)
    M = torch.empty(X.shape, dtype=torch.bool, device=X.device)
    n = X.numel()
    if U is not None:
        require(U.dtype == torch.float32 and U.numel() == n, "ValueError: U must be float32 with one value per element")
        call("dbk_dropoutord_fp_tr_u", stream(), ptr(X), ptr(Z), ptr(M), n, float(rate), ptr(U))
    elif counter is not None:
        call("dbk_dropoutord_fp_tr", stream(), ptr(X), ptr(Z), ptr(M), n, float(rate), _rng_seed if seed is None else int(seed), 0, ptr(counter))
    elif offset is not None:
        call("dbk_dropoutord_fp_tr", stream(), ptr(X), ptr(Z), ptr(M), n, float(rate), _rng_seed if seed is None else int(seed), int(offset), None)
    else:
        call("dbk_dropoutord_fp_tr", stream(), ptr(X), ptr(Z), ptr(M), n, float(rate), _rng_seed if seed is None else int(seed), _rng_offset, None)
        _rng_offset += (n + 3) // 4
    if regions is not None:
        _regions(regions)
        require(regions.shape[1] == 2 and padding is not None, "ValueError: mirroring needs 2-column regions and the padding length")
        call("dbk_dropoutord_mirror", stream(), ptr(X), ptr(Z), ptr(M), ptr(regions), regions.shape[0], int(padding))
    return Z, M


def corr1ord_enforce_constraints(W, constraint, nchannel=4):
    """Applies the scan filters' constraint to W (4*m, nfilter) in place: "pfm" (each tap's letter weights become
    log-probabilities), "psam" (log of the weights relative to the tap's largest), a (lo, hi) tuple (clip), or
    None (nothing). reference: corr1ord.enforce_constraints, kangaroo/_ext/corr1ord.py:60-77"""
    if constraint is None:
        return
    require(nchannel == 4, "NotImplementedError: only the 4-letter alphabet is supported")
    require(W.dim() == 2 and W.shape[0] % 4 == 0 and W.is_contiguous(), "ValueError: W must be a contiguous (4*m, nfilter) matrix")
    if constraint in ("pfm", "psam"):
        kind, lo, hi = (0 if constraint == "pfm" else 1), 0.0, 0.0
    elif type(constraint) == tuple:
        kind, (lo, hi) = 2, constraint
    else:
        raise NotImplementedError("constraint \"%s\" not implemented" % str(constraint))
    call("dbk_corr1ord_constraint", stream(), dtype_code(W), ptr(W), W.shape[0] // 4, W.shape[1], kind, float(lo), float(hi))


# ------------------------------------------------------------------------------------------------
# fused scan + bias + ReLU + pool
# ------------------------------------------------------------------------------------------------
def activity_words(X, W):
    """Empty buffer for the activity masks of scanpool_fprop: one 64-bit word per row of X and tile of 64 filters."""
    return torch.empty((X.numel(), (W.shape[1] + 63) // 64), dtype=torch.int64, device=W.device)


def scanpool_fprop(W, b, X, regions, ptype, want_argmax=False, path="auto", act=None, out=None):
    """pool(relu(corr1ord(W, X) + b)) per region without storing the (N x P) map.
    Returns (pooled, argmax|None) laid out exactly as poolrgn's. float32; float64 tensors run the operator kernels in
    double precision one after another inside the library (no fused float64 kernel).
    path: "auto" lets the library choose; "general" / "mfma" / "wide" / "kmer" force the general path (which picks its
    kernel by size), its matrix-core kernel for many regions (filters of up to 32 taps; sums in another order than
    the lookup kernels', equal to round-off), the four-filters-per-lane lookup kernel (9-24 taps; the bits of the
    one-filter-per-lane kernel) or the bulk kernel (6-bit digits on the matrix cores, filters of up to 24 taps);
    "kmer_static" is the bulk kernel with the scratch buffer that is built into the library (no allocation inside the
    call; at most 64 MiB of sequence bytes; calls that overlap on one GPU must not use it together).
    out (optional): (pooled, argmax|None) tensors to write into instead of new ones, so that the call allocates nothing.
    act (optional, from activity_words): receives 1 bit per row and filter - rectifier open or not - which
    scanpool_bprop takes in place of recomputing the map (general kernel only).
    Sum pooling and 3-column regions (row step) run the operator kernels one after another inside the library, with
    the map in its scratch: same results as the reference's chain; path must be "auto" and no masks are written."""
    _u8(X)
    _regions(regions)
    f64 = W.dtype == torch.float64
    unfused = regions.shape[1] == 3 or ptype == "sum" or f64
    require(not unfused or (path == "auto" and act is None),
            "ValueError: sum pooling, stepped regions and float64 run the operator chain: no kernel choice, no activity masks")
    require(W.dtype in (torch.float32, torch.float64) and b.dtype == W.dtype, "TypeError: W and b must both be float32 or both float64")
    require(W.shape[0] % 4 == 0 and b.numel() == W.shape[1], "ValueError: W must be (4m x P) and b must have P entries")
    m, F, P = W.shape[0] // 4, W.shape[1], regions.shape[0]
    want_argmax = want_argmax and ptype in ("max", "all")
    if out is not None:
        pooled, argmax = out
        require(pooled.dtype == W.dtype and tuple(pooled.shape) == (P, F * (2 if ptype == "all" else 1)),
                "ValueError: out[0] must be (regions x pooled features) of W's dtype")
        require((argmax is not None) == bool(want_argmax), "ValueError: out[1] must be given exactly when argmax is wanted")
        require(argmax is None or (argmax.dtype == uindex and tuple(argmax.shape) == (P, F)), "ValueError: out[1] must be (regions x filters) indices")
    else:
        pooled = torch.empty((P, F * (2 if ptype == "all" else 1)), dtype=W.dtype, device=W.device)
        argmax = torch.empty((P, F), dtype=uindex, device=W.device) if want_argmax else None
    if unfused:
        # (float64: the operator kernels in double precision, as the reference compiles every operator for both types)
        call("dbk_scanpool_fprop_f64" if f64 else "dbk_scanpool_fprop_unfused", stream(), ptr(W), ptr(b), m, F, ptr(X), X.numel(),
             ptr(regions), P, regions.shape[1], str2pooltype[ptype], ptr(pooled), ptr(argmax))
        return pooled, argmax
    entry = {"auto": "dbk_scanpool_fprop", "general": "dbk_scanpool_fprop_general", "wide": "dbk_scanpool_fprop_wide", "mfma": "dbk_scanpool_fprop_mfma",
             "kmer": "dbk_scanpool_fprop_kmer", "kmer_static": "dbk_scanpool_fprop_kmer_static"}[path]
    args = [stream(), ptr(W), ptr(b), m, F, ptr(X), X.numel(), ptr(regions), P, str2pooltype[ptype], ptr(pooled), ptr(argmax)]
    if path not in ("kmer", "kmer_static"):
        args.append(_act(act, X, F))
    else:
        require(act is None, "ValueError: the bulk kernel does not write activity masks")
    call(entry, *args)
    return pooled, argmax


def _act(act, X, F):
    if act is None:
        return None
    require(act.dtype == torch.int64 and act.numel() == X.numel() * ((F + 63) // 64),
            "ValueError: act must hold one 64-bit word per row of X and tile of 64 filters")
    return ptr(act)


def scanpool_bprop(W, b, X, regions, ptype, pooled, argmax, dpooled, dW, db, overwrite=False, act=None):
    """Backward of scanpool_fprop: dW += filter gradient (dW[:] = with overwrite), db[:] = bias gradient.
    act: the activity masks the forward call filled (same W, b, X, regions), if it was given any."""
    _u8(X)
    _regions(regions)
    f64 = W.dtype == torch.float64
    require(W.dtype in (torch.float32, torch.float64) and all(t.dtype == W.dtype for t in (b, dpooled, dW, db)),
            "TypeError: W, b, dpooled, dW and db must all be float32 or all float64")
    require(dW.shape == W.shape and db.numel() == W.shape[1], "ValueError: dW / db shapes must match W / b")
    require(dpooled.shape == pooled.shape, "ValueError: dpooled must have pooled's shape")
    m, F, P = W.shape[0] // 4, W.shape[1], regions.shape[0]
    if regions.shape[1] == 3 or ptype == "sum" or f64:
        require(act is None, "ValueError: sum pooling, stepped regions and float64 take no activity masks")
        call("dbk_scanpool_bprop_f64" if f64 else "dbk_scanpool_bprop_unfused", stream(), ptr(W), ptr(b), m, F, ptr(X), X.numel(),
             ptr(regions), P, regions.shape[1], str2pooltype[ptype], ptr(argmax), ptr(dpooled), ptr(dW), ptr(db), int(bool(overwrite)))
        return
    call("dbk_scanpool_bprop", stream(), ptr(W), ptr(b), m, F, ptr(X), X.numel(), ptr(regions), P, str2pooltype[ptype],
         ptr(pooled), ptr(argmax), ptr(dpooled), ptr(dW), ptr(db), int(bool(overwrite)), _act(act, X, F))


# ------------------------------------------------------------------------------------------------
# layers along the rows of every region, between the motif scan and the pooling
# ------------------------------------------------------------------------------------------------
def _row_regions(a, R):
    _regions(R)
    if R.shape[1] != 2 or not R.is_contiguous():
        raise DeepbindError("ValueError: regions must be a contiguous (P x 2) array")
    return R.shape[0], a.dense("regions", R, R.shape, R.dtype)


def _map(X):
    if not isinstance(X, torch.Tensor) or X.dim() != 2:
        raise DeepbindError("ValueError: X must be a matrix")
    return _lib.row_dtype_code(X), _lib.wide_dtype(X), X.shape[0], X.shape[1]


def _rows_out(t, shape, dtype, device):
    """A matrix of rows that the caller gave, or a new one: zeros, as rows in no region are not written."""
    return torch.zeros(shape, dtype=dtype, device=device) if t is None else t


def _dense_out(t, shape, dtype, device):
    return torch.empty(shape, dtype=dtype, device=device) if t is None else t


def _conv_args(X, W, b):
    code, wide, N, D = _map(X)
    require(isinstance(W, torch.Tensor) and W.dim() == 2 and W.shape[1] == D, "ValueError: W must be (taps x channels)")
    K = W.shape[0]
    if not 1 <= K <= 4:
        raise DeepbindError("NotImplementedError: filters of 1 to 4 taps, got %d" % K)
    a = _lib.Arguments()
    return (a, code, wide, N, D, K) + a.rows("X", X, (N, D), X.dtype) + (a.dense("W", W, (K, D), wide), a.dense("b", b, (1, D), wide))


def causalconv(X, W, b, regions, silu=True, state=None, want_state=False, out=None):
    """Causal convolution along the rows of every region of the map X (N x D), a filter of 1 to 4 taps per channel: p[t] = b +
    sum_j W[j] X[t - taps + 1 + j] (W: taps x D, b: 1 x D or None), returned as p * sigmoid(p), or as p without silu.
    X: float32, float64 or bfloat16, row stride of its own; weights float32 (float64 beside float64). Regions (P x 2) may come in any
    order and must not overlap; rows in no region are zeros in a new output, and stay as they are in `out`.
    Rows before a region's first are those of state (P x taps-1 x D, X's type) or zeros.
    Returns (Z, last|None): with want_state, last is what the next piece of each sequence takes as its state."""
    a, code, wide, N, D, K, x, ldx, w, bp = _conv_args(X, W, b)
    P, rp = _row_regions(a, regions)
    sp = a.dense("state", state, (P, K - 1, D), X.dtype)
    if out is not None:
        a.rows("out", out, (N, D), X.dtype, out=True)
    a.check()
    Z = _rows_out(out, (N, D), X.dtype, X.device)
    last = torch.empty((P, K - 1, D), dtype=X.dtype, device=X.device) if want_state else None
    need = ctypes.c_size_t(0)
    call("dbk_causalconv_workspace", code, K, N, D, P, 0, ctypes.addressof(need))
    work, wp = _lib.workspace(need.value, X)
    call("dbk_causalconv", stream(), code, x, ldx, w, bp, K, N, D, rp, P, int(bool(silu)), sp, Z.data_ptr(), _lib.row_stride(Z),
         None if last is None else last.data_ptr(), wp, need.value)
    return Z, last


def causalconv_bprop(X, W, b, regions, dZ, silu=True, out=None):
    """Gradients (dX, dW, db|None) of causalconv at X, for sequences that start from zeros. out (optional): a tuple like the returned
    one of tensors to write into, None where one is to be made; rows of dX in no region are zeros, or stay as they are in out's."""
    a, code, wide, N, D, K, x, ldx, w, bp = _conv_args(X, W, b)
    P, rp = _row_regions(a, regions)
    dz, lddz = a.rows("dZ", dZ, (N, D), X.dtype)
    dX, dW, db = (None, None, None) if out is None else out
    require(b is not None or db is None, "ValueError: no bias, no gradient of it")
    if dX is not None:
        a.rows("dX", dX, (N, D), X.dtype, out=True)
    a.dense("dW", dW, (K, D), wide, out=True)
    a.dense("db", db, (1, D), wide, out=True)
    a.check()
    dX = _rows_out(dX, (N, D), X.dtype, X.device)
    dW = _dense_out(dW, (K, D), wide, X.device)
    db = None if b is None else _dense_out(db, (1, D), wide, X.device)
    need = ctypes.c_size_t(0)
    call("dbk_causalconv_workspace", code, K, N, D, P, 1, ctypes.addressof(need))
    work, wp = _lib.workspace(need.value, X)
    call("dbk_causalconv_bprop", stream(), code, x, ldx, w, bp, K, N, D, rp, P, int(bool(silu)), dz, lddz, dX.data_ptr(), _lib.row_stride(dX),
         dW.data_ptr(), None if db is None else db.data_ptr(), wp, need.value)
    return dX, dW, db


def causalconv_step(X, W, b, state, silu=True, into=None, out=None):
    """One new row for each of n sequences: X (n x D) and state (n x taps-1 x D) give Z (n x D). The state moves on in place, or
    its successor goes to `into`, which leaves it as it is."""
    a, code, wide, n, D, K, x, ldx, w, bp = _conv_args(X, W, b)
    require(state is not None, "ValueError: state is needed")
    into = None if into is state else into
    sp = a.dense("state", state, (n, K - 1, D), X.dtype, out=into is None)
    ip = sp if into is None else a.dense("into", into, (n, K - 1, D), X.dtype, out=True)
    if out is not None:
        a.rows("out", out, (n, D), X.dtype, out=True)
    a.check()
    Z = _dense_out(out, (n, D), X.dtype, X.device)
    call("dbk_causalconv_step", stream(), code, x, ldx, w, bp, K, n, D, int(bool(silu)), sp, ip, Z.data_ptr(), _lib.row_stride(Z))
    return Z


def kept_states(X, A):
    """Empty buffer for the states that statescan keeps for statescan_bprop: one (S x D) block per 8 rows of X."""
    return torch.empty(((X.shape[0] + 7) // 8, A.shape[0], A.shape[1]), dtype=A.dtype, device=A.device)


def _scan_args(X, dt, A, B, C, D, gate, dt_bias, softplus):
    code, wide, N, D_ = _map(X)
    require(isinstance(A, torch.Tensor) and A.dim() == 2 and A.shape[1] == D_ and A.shape[0] >= 1, "ValueError: A must be (states x channels)")
    S = A.shape[0]
    if S > 64:
        raise DeepbindError("NotImplementedError: 1 to 64 states per channel, got %d" % S)
    require(isinstance(B, torch.Tensor) and B.dim() == 2 and B.shape[1] % S == 0 and B.shape[1] >= S, "ValueError: B must be (rows x groups * states)")
    G = B.shape[1] // S
    require(D_ % G == 0, "ValueError: the number of channels must be divisible by the number of groups")
    g = _lib.Arguments()
    kept, shape, weights = X.dtype, (N, D_), (N, G * S)
    x, ldx = g.rows("X", X, shape, kept)
    t, ldt = g.rows("dt", dt, shape, kept)
    ap = g.dense("A", A, (S, D_), wide)
    b, ldb = g.rows("B", B, weights, wide)
    c, ldc = g.rows("C", C, weights, wide)
    sk, bi = g.dense("D", D, (1, D_), wide), g.dense("dt_bias", dt_bias, (1, D_), wide)
    gp, ldg = (None, 0) if gate is None else g.rows("gate", gate, shape, kept)
    return g, _lib.StateScanArgs(code, int(bool(softplus)), N, D_, S, G, None, 0, x, ldx, t, ldt, ap, b, ldb, c, ldc, sk, bi, gp, ldg), wide, N, D_, S, G


def statescan(X, dt, A, B, C, regions, D=None, gate=None, dt_bias=None, softplus=True, state=None, want_state=False, keep=None, out=None):
    """Selective state space scan along the rows of every region of the map X (N x D): with d = softplus(dt + dt_bias) (dt + dt_bias
    without softplus), h = exp(d * A) * h + d * X * B and Y = sum over states of C * h + D * X, times gate * sigmoid(gate) where
    there is a gate. dt, gate (N x D, X's type); A (S x D), D, dt_bias (1 x D); B, C (N x G*S): the channels form G equal groups, each
    with its own S columns; up to 64 states per channel.
    X: float32, float64 or bfloat16; weights, B, C and states float32 (float64 beside float64); matrices of rows have row strides of
    their own. Regions (P x 2) may come in any order and must not overlap; rows in no region are zeros in a new output, and stay as
    they are in `out`. States start from state (P x S x D), or zeros.
    keep (optional, from kept_states): receives the states that statescan_bprop starts from (without `state` only).
    Returns (Y, last|None): with want_state, last (P x S x D) holds the states behind the regions' last rows."""
    g, a, wide, N, D_, S, G = _scan_args(X, dt, A, B, C, D, gate, dt_bias, softplus)
    P, a.regions = _row_regions(g, regions)
    a.nregion = P
    a.state = g.dense("state", state, (P, S, D_), wide)
    a.keep = g.dense("keep", keep, ((N + 7) // 8, S, D_), wide, out=True)
    require(keep is None or state is None, "ValueError: states are kept for the backward pass of whole sequences, which starts from zeros: no initial state")
    if out is not None:
        g.rows("out", out, (N, D_), X.dtype, out=True)
    g.check()
    Y = _rows_out(out, (N, D_), X.dtype, X.device)
    a.Y, a.ldy = Y.data_ptr(), _lib.row_stride(Y)
    last = None
    if want_state:
        last = torch.empty((P, S, D_), dtype=wide, device=X.device)
        a.last = last.data_ptr()
    at, need = ctypes.addressof(a), ctypes.c_size_t(0)
    call("dbk_statescan_workspace", at, 0, ctypes.addressof(need))
    work, wp = _lib.workspace(need.value, X)
    call("dbk_statescan", stream(), at, wp, need.value)
    return Y, last


def statescan_bprop(X, dt, A, B, C, regions, keep, dY, D=None, gate=None, dt_bias=None, softplus=True, out=None):
    """Gradients (dX, ddt, dA, dB, dC, dD|None, dgate|None, ddt_bias|None) of statescan for sequences that start from zero states,
    from the states that the forward call kept. out (optional): a tuple like the returned one of tensors to write into, None where
    one is to be made; rows in no region are zeros, or stay as they are in out's."""
    g, a, wide, N, D_, S, G = _scan_args(X, dt, A, B, C, D, gate, dt_bias, softplus)
    P, a.regions = _row_regions(g, regions)
    a.nregion = P
    require(keep is not None, "ValueError: the states that the forward call kept are needed")
    a.keep = g.dense("keep", keep, ((N + 7) // 8, S, D_), wide)
    kept, dev, shape, weights = X.dtype, X.device, (N, D_), (N, G * S)
    a.dY, a.lddy = g.rows("dY", dY, shape, kept)
    dX, ddt, dA, dB, dC, dD, dgate, dbias = (None,) * 8 if out is None else out
    for given, grad, name in ((D, dD, "D"), (gate, dgate, "gate"), (dt_bias, dbias, "dt_bias")):
        if given is None and grad is not None:
            raise DeepbindError("ValueError: no %s, no gradient of it" % name)
    for name, t, s, dtype in (("dX", dX, shape, kept), ("ddt", ddt, shape, kept), ("dgate", dgate, shape, kept), ("dB", dB, weights, wide), ("dC", dC, weights, wide)):
        if t is not None:
            g.rows(name, t, s, dtype, out=True)
    for name, t, s in (("dA", dA, (S, D_)), ("dD", dD, (1, D_)), ("ddt_bias", dbias, (1, D_))):
        g.dense(name, t, s, wide, out=True)
    g.check()
    dX, ddt = _rows_out(dX, shape, kept, dev), _rows_out(ddt, shape, kept, dev)
    dA = _dense_out(dA, (S, D_), wide, dev)
    dB, dC = _rows_out(dB, weights, wide, dev), _rows_out(dC, weights, wide, dev)
    dD = None if D is None else _dense_out(dD, (1, D_), wide, dev)
    dgate = None if gate is None else _rows_out(dgate, shape, kept, dev)
    dbias = None if dt_bias is None else _dense_out(dbias, (1, D_), wide, dev)
    ld = _lib.row_stride
    a.dX, a.lddx, a.ddt, a.ldddt, a.dB, a.lddb, a.dC, a.lddc = dX.data_ptr(), ld(dX), ddt.data_ptr(), ld(ddt), dB.data_ptr(), ld(dB), dC.data_ptr(), ld(dC)
    a.dA = dA.data_ptr()
    if dgate is not None:
        a.dgate, a.lddgate = dgate.data_ptr(), ld(dgate)
    if dD is not None:
        a.dskip = dD.data_ptr()
    if dbias is not None:
        a.ddt_bias = dbias.data_ptr()
    at, need = ctypes.addressof(a), ctypes.c_size_t(0)
    call("dbk_statescan_workspace", at, 1, ctypes.addressof(need))
    work, wp = _lib.workspace(need.value, X)
    call("dbk_statescan_bprop", stream(), at, wp, need.value)
    return dX, ddt, dA, dB, dC, dD, dgate, dbias


def statescan_step(X, dt, A, B, C, state, D=None, gate=None, dt_bias=None, softplus=True, into=None, out=None):
    """One new row for each of n sequences: Y (n x D) from X, dt, gate (n x D), B, C (n x G*S) and state (n x S x D), arguments
    otherwise as in statescan. The state moves on in place, or its successor goes to `into`, which leaves it as it is."""
    g, a, wide, n, D_, S, G = _scan_args(X, dt, A, B, C, D, gate, dt_bias, softplus)
    require(state is not None, "ValueError: state is needed")
    into = None if into is state else into
    a.state = g.dense("state", state, (n, S, D_), wide, out=into is None)
    a.last = a.state if into is None else g.dense("into", into, (n, S, D_), wide, out=True)
    if out is not None:
        g.rows("out", out, (n, D_), X.dtype, out=True)
    g.check()
    Y = _dense_out(out, (n, D_), X.dtype, X.device)
    a.Y, a.ldy = Y.data_ptr(), _lib.row_stride(Y)
    call("dbk_statescan_step", stream(), ctypes.addressof(a))
    return Y


def _delta_shape(K, V, beta, groups):
    """(heads, key heads, columns of a key, columns of a value) of the delta rule's maps."""
    for name, t in (("K", K), ("V", V), ("beta", beta)):
        if not isinstance(t, torch.Tensor) or t.dim() != 2:
            raise DeepbindError("ValueError: %s must be a matrix" % name)
    H = beta.shape[1]
    G = H if groups is None else int(groups)
    require(H >= 1 and G >= 1 and H % G == 0, "ValueError: the number of heads must be divisible by the number of key heads")
    require(K.shape[1] >= G and K.shape[1] % G == 0, "ValueError: K must be (rows x key heads * columns of a key)")
    require(V.shape[1] >= H and V.shape[1] % H == 0, "ValueError: V must be (rows x heads * columns of a value)")
    if K.shape[1] // G > 128:
        raise DeepbindError("NotImplementedError: keys of 1 to 128 columns, got %d" % (K.shape[1] // G))
    return H, G, K.shape[1] // G, V.shape[1] // H


def _kept_values(code, N, H, G, key, value):
    a, need = _lib.DeltaRuleArgs(code, N, H, G, key, value), ctypes.c_size_t(0)
    call("dbk_deltarule_kept", ctypes.addressof(a), ctypes.addressof(need))
    return need.value


def kept_delta(K, V, beta, groups=None):
    """Empty buffer (1 x values) for what deltarule keeps for deltarule_bprop, for maps of these shapes: the states at every 64th row of a
    region, and what takes them over the segments that long regions are cut into."""
    H, G, key, value = _delta_shape(K, V, beta, groups)
    return torch.empty((1, _kept_values(_lib.row_dtype_code(V), V.shape[0], H, G, key, value)), dtype=_lib.wide_dtype(V), device=V.device)


def _delta_args(Q, K, V, beta, decay, groups, scale):
    H, G, key, value = _delta_shape(K, V, beta, groups)
    code, wide, N, D = _map(V)
    g = _lib.Arguments()
    kept, keys, rates = V.dtype, (N, G * key), (N, H)
    q, ldq = g.rows("Q", Q, keys, kept)
    k, ldk = g.rows("K", K, keys, kept)
    v, ldv = g.rows("V", V, (N, D), kept)
    b, ldb = g.rows("beta", beta, rates, wide)
    d, ldd = (None, 0) if decay is None else g.rows("decay", decay, rates, wide)
    scale = key ** -0.5 if scale is None else float(scale)
    return g, _lib.DeltaRuleArgs(code, N, H, G, key, value, None, 0, q, ldq, k, ldk, v, ldv, b, ldb, d, ldd, scale), wide, N, key, D


def _delta_keep(g, a, keep, wide, out):
    """The pointer of a buffer from kept_delta for a call's shapes."""
    return None if keep is None else g.dense("keep", keep, (1, _kept_values(a.dtype, a.N, a.H, a.G, a.K, a.V)), wide, out=out)


def deltarule(Q, K, V, beta, regions, decay=None, groups=None, scale=None, state=None, want_state=False, keep=None, out=None):
    """Gated delta rule along the rows of every region. Every head has a state S (key x value), which a row first multiplies by
    exp(decay), then corrects by what its key finds in it, u = beta * (v - S^T k) and S = S + k u^T, and its query reads: O = scale * S^T q.
    V (N x heads*value); beta, decay (N x heads; decay None: nothing decays); Q, K (N x groups*key, up to 128 columns a key): the heads
    form `groups` equal groups (None: as many as heads), each with its own query and key. scale: key ** -0.5 if None.
    Keys of length 1 (blocknorm with rms and gamma = key ** -0.5) keep the state bounded for beta up to 2.
    Rows: float32, float64 or bfloat16; beta, decay and states float32 (float64 beside float64); matrices of rows have row strides of
    their own. Regions (P x 2) may come in any order and must not overlap; rows in no region are zeros in a new output, and stay as
    they are in `out`. States start from state (P x key x heads*value), or zeros.
    keep (optional, from kept_delta): receives the states that deltarule_bprop starts from (without `state` only).
    Returns (O, last|None): with want_state, last (P x key x heads*value) holds the states behind the regions' last rows."""
    g, a, wide, N, key, D = _delta_args(Q, K, V, beta, decay, groups, scale)
    P, a.regions = _row_regions(g, regions)
    a.nregion = P
    a.state = g.dense("state", state, (P, key, D), wide)
    a.keep = _delta_keep(g, a, keep, wide, True)
    require(keep is None or state is None, "ValueError: states are kept for the backward pass of whole sequences, which starts from zeros: no initial state")
    if out is not None:
        g.rows("out", out, (N, D), V.dtype, out=True)
    g.check()
    O = _rows_out(out, (N, D), V.dtype, V.device)
    a.O, a.ldo = O.data_ptr(), _lib.row_stride(O)
    last = None
    if want_state:
        last = torch.empty((P, key, D), dtype=wide, device=V.device)
        a.last = last.data_ptr()
    at, need = ctypes.addressof(a), ctypes.c_size_t(0)
    call("dbk_deltarule_workspace", at, 0, ctypes.addressof(need))
    work, wp = _lib.workspace(need.value, V)
    call("dbk_deltarule", stream(), at, wp, need.value)
    return O, last


def deltarule_bprop(Q, K, V, beta, regions, keep, dO, decay=None, groups=None, scale=None, out=None):
    """Gradients (dQ, dK, dV, dbeta, ddecay|None) of deltarule for sequences that start from zero states, from the states that the
    forward call kept. out (optional): a tuple like the returned one of tensors to write into, None where one is to be made; rows in
    no region are zeros, or stay as they are in out's."""
    g, a, wide, N, key, D = _delta_args(Q, K, V, beta, decay, groups, scale)
    P, a.regions = _row_regions(g, regions)
    a.nregion = P
    require(keep is not None, "ValueError: the states that the forward call kept are needed")
    a.keep = _delta_keep(g, a, keep, wide, False)
    a.dO, a.lddo = g.rows("dO", dO, (N, D), V.dtype)
    given = (None,) * 5 if out is None else tuple(out)
    require(len(given) == 5, "ValueError: out must be (dQ, dK, dV, dbeta, ddecay)")
    require(decay is not None or given[4] is None, "ValueError: no decay, no gradient of it")
    likes = (("dQ", Q), ("dK", K), ("dV", V), ("dbeta", beta), ("ddecay", decay))
    for (name, like), t in zip(likes, given):
        if t is not None:
            g.rows(name, t, tuple(like.shape), like.dtype, out=True)
    g.check()
    grads = tuple(None if like is None else _rows_out(t, like.shape, like.dtype, V.device) for (_, like), t in zip(likes, given))
    ld = _lib.row_stride
    a.dQ, a.lddq, a.dK, a.lddk, a.dV, a.lddv = grads[0].data_ptr(), ld(grads[0]), grads[1].data_ptr(), ld(grads[1]), grads[2].data_ptr(), ld(grads[2])
    a.dbeta, a.lddbeta = grads[3].data_ptr(), ld(grads[3])
    if grads[4] is not None:
        a.ddecay, a.ldddecay = grads[4].data_ptr(), ld(grads[4])
    at, need = ctypes.addressof(a), ctypes.c_size_t(0)
    call("dbk_deltarule_workspace", at, 1, ctypes.addressof(need))
    work, wp = _lib.workspace(need.value, V)
    call("dbk_deltarule_bprop", stream(), at, wp, need.value)
    return grads


def deltarule_step(Q, K, V, beta, state, decay=None, groups=None, scale=None, into=None, out=None):
    """One new row for each of n sequences: O (n x heads*value) from Q, K, V, beta, decay (n rows) and state (n x key x heads*value),
    arguments otherwise as in deltarule. The state moves on in place, or its successor goes to `into`, which leaves it as it is."""
    g, a, wide, n, key, D = _delta_args(Q, K, V, beta, decay, groups, scale)
    require(state is not None, "ValueError: state is needed")
    into = None if into is state else into
    a.state = g.dense("state", state, (n, key, D), wide, out=into is None)
    a.last = a.state if into is None else g.dense("into", into, (n, key, D), wide, out=True)
    if out is not None:
        g.rows("out", out, (n, D), V.dtype, out=True)
    g.check()
    O = _dense_out(out, (n, D), V.dtype, V.device)
    a.O, a.ldo = O.data_ptr(), _lib.row_stride(O)
    call("dbk_deltarule_step", stream(), ctypes.addressof(a))
    return O
