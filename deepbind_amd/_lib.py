"""ctypes binding of libdeepbind_hip.so.

The library is the only compute path: if it cannot be loaded, importing an operator module
raises. After every call the thread's last-error text is polled and turned into an exception,
the convention of the reference's Python shim (reference: code/libs/smat/py/smat/smat_dll.py:166-183).
"""
import ctypes
import os
from ctypes import c_char_p, c_double, c_float, c_int, c_size_t, c_uint64, c_void_p

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libdeepbind_hip.so")


class DeepbindError(RuntimeError):
    """Raised when a library call reports a failure (counterpart of the reference's SmatException)."""


DBK_F32, DBK_F64, DBK_BF16 = 0, 1, 2
PT_MAX, PT_AVG, PT_SUM, PT_ALL = 0, 1, 2, 3
str2pooltype = {"max": PT_MAX, "avg": PT_AVG, "sum": PT_SUM, "all": PT_ALL}
# loss_kind of dbk_head_train / dbk_train_step*: output non-linearity + loss (reference: deepity/std/loss.py:131-174)
LOSS_KIND = {"nll": 0, "mse": 1, "hinge": 2}

_P, _Z, _I, _U64, _F, _D = c_void_p, c_size_t, c_int, c_uint64, c_float, c_double

# name -> argument types; every function returns int except the two noted below
_SIGNATURES = {
    "dbk_version": [],
    "dbk_device_count": [],
    "dbk_set_exact_scan": [_I],
    "dbk_sync": [_P],
    "dbk_corr1ord": [_P, _I, _P, _Z, _Z, _P, _Z, _Z, _P],
    "dbk_corr1ord_bprop_W": [_P, _I, _P, _Z, _Z, _P, _Z, _Z, _P],
    "dbk_corr1ord_bprop_X": [_P, _I, _P, _Z, _Z, _P, _Z, _Z, _P],
    "dbk_poolrgn": [_P, _I, _P, _Z, _P, _Z, _I, _P, _P, _I],
    "dbk_poolrgn_bprop": [_P, _I, _P, _Z, _P, _Z, _I, _P, _P, _I],
    "dbk_dropoutord_fp_tr": [_P, _P, _P, _P, _Z, _F, _U64, _U64, _P],
    "dbk_corr1ord_constraint": [_P, _I, _P, _Z, _Z, _I, _D, _D],
    "dbk_dropoutord_mirror": [_P, _P, _P, _P, _P, _Z, _Z],
    "dbk_dropoutord_fp_tr_u": [_P, _P, _P, _P, _Z, _F, _P],
    "dbk_scanpool_fprop": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _P, _P, _P],
    "dbk_scanpool_fprop_general": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _P, _P, _P],
    "dbk_scanpool_fprop_wide": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _P, _P, _P],
    "dbk_scanpool_fprop_mfma": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _P, _P, _P],
    "dbk_scanpool_fprop_kmer": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _P, _P],
    "dbk_scanpool_fprop_kmer_static": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _P, _P],
    "dbk_scanpool_bprop": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _P, _P, _P, _P, _P, _I, _P],
    "dbk_scanpool_fprop_unfused": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _I, _P, _P],
    "dbk_scanpool_bprop_unfused": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _I, _P, _P, _P, _P, _I],
    "dbk_scanpool_fprop_f64": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _I, _P, _P],
    "dbk_scanpool_bprop_f64": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _I, _I, _P, _P, _P, _P, _I],
    "dbk_blockwise_dot": [_P, _I, _I, _I, _I, _I, _I, _P, _P, _P],
    "dbk_blockwise_dot_nt": [_P, _I, _I, _I, _I, _I, _P, _P, _P],
    "dbk_blockwise_dot_tn": [_P, _I, _I, _I, _I, _I, _I, _P, _P, _P],
    "dbk_blockwise_dot_combined": [_P, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P],
    "dbk_blockwise_dot_nt_combined": [_P, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P],
    "dbk_blockwise_dot_tn_combined": [_P, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P],
    "dbk_gradstep": [_P, _I, _Z, _P, _P, _P, _P, _P],
    "dbk_gradstep_nesterov1": [_P, _I, _Z, _P, _P, _P],
    "dbk_gradstep_nesterov2": [_P, _I, _Z, _P, _P, _P, _P, _P],
    "dbk_gradstep_lookahead": [_P, _I, _Z, _P, _P, _P, _P],
    "dbk_gradstep_nesterov2_lookahead": [_P, _I, _Z, _P, _P, _P, _P, _P, _P],
    "dbk_madd_bcast": [_P, _I, _P, _P, _P, _Z, _Z, _Z],
    "dbk_maskout": [_P, _I, _P, _P, _Z],
    "dbk_calc_zmask": [_P, _I, _P, _P, _Z, _Z],
    "dbk_pair_max": [_P, _I, _P, _P, _Z, _Z],
    "dbk_dropout_fp_tr": [_P, _I, _P, _P, _P, _P, _Z, _Z, _Z, _I, _U64, _U64],
    "dbk_dropout_fp_tr_u": [_P, _I, _P, _P, _P, _P, _Z, _Z, _Z, _I, _P],
    "dbk_dropout_fp_te": [_P, _I, _P, _P, _P, _Z, _Z, _Z],
    "dbk_dropout_bp_tr": [_P, _I, _P, _P, _P, _Z],
    "dbk_dropout_bp_te": [_P, _I, _P, _P, _P, _Z, _Z, _Z],
    "dbk_uniform_fill": [_P, _P, _Z, _U64, _U64],
    "dbk_normal_fill": [_P, _I, _P, _Z, _U64, _U64],
    "dbk_philox4x32_10": [_P, _P, _P],
    "dbk_add_rowvec": [_P, _I, _P, _P, _P, _Z, _Z],
    "dbk_colsum": [_P, _I, _P, _P, _Z, _Z],
    "dbk_relu": [_P, _I, _P, _P, _Z],
    "dbk_mul_sign": [_P, _I, _P, _P, _P, _Z],
    "dbk_sign": [_P, _I, _P, _P, _Z],
    "dbk_logistic": [_P, _I, _P, _P, _Z],
    "dbk_loss_terms": [_P, _I, _I, _P, _P, _P, _Z],
    "dbk_sub_scale": [_P, _I, _P, _P, _D, _P, _Z],
    "dbk_hinge_grad": [_P, _I, _P, _P, _D, _P, _Z],
    "dbk_head_train": [_P, _Z, _I, _I, _I, _I, _I, _P, _I, _P, _P, _P, _U64, _U64, _P, _U64, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P],
    "dbk_softmax": [_P, _I, _P, _P, _Z, _Z],
    "dbk_counter_add": [_P, _P, _U64],
    "dbk_l1_decay": [_P, _I, _P, _P, _P, _Z],
    "dbk_head_fprop": [_P, _Z, _I, _I, _I, _P, _I, _P, _P, _P, _P, _P, _P, _I, _P],
    "dbk_pack_text": [_P, _P, _P, _Z, _Z, _I, _P, _P],
    "dbk_pack_windows": [_P, _P, _P, _P, _Z, _Z, _Z, _Z, _Z, _I, _P, _P],
    "dbk_predict_small_takes": [_Z, _Z, _Z, _Z, _Z, _I, _Z],
    "dbk_predict_small": [_P, _P, _P, _Z, _Z, _Z, _P, _Z, _P, _Z, _I, _Z, _P, _P, _P, _P, _P, _I, _P],
    "dbk_mutation_map_takes": [_Z, _Z, _I, _Z],
    "dbk_mutation_map": [_P, _P, _P, _Z, _Z, _P, _Z, _P, _Z, _Z, _I, _Z, _P, _P, _P, _P, _P, _I, _I, _P, _P],
    "dbk_gradient_map_takes": [_Z, _Z, _Z, _Z, _I, _Z],
    "dbk_gradient_map": [_P, _P, _P, _Z, _Z, _P, _P, _Z, _Z, _Z, _I, _Z, _P, _P, _P, _P, _P, _I, _I, _P, _P, _P],
    "dbk_gather_maps": [_P, _I, _P, _Z, _Z, _I, _P, _P, _P],
    "dbk_layernorm": [_P, _I, _P, _Z, _P, _P, _Z, _Z, _Z, _D, _P, _Z, _P],
    "dbk_layernorm_bprop_workspace": [_I, _Z, _Z, _Z, _P],
    "dbk_layernorm_bprop": [_P, _I, _P, _Z, _P, _P, _P, _Z, _Z, _Z, _Z, _P, _Z, _P, _P, _P, _Z],
    "dbk_blocknorm_args_size": [],
    "dbk_blocknorm": [_P, _P],
    "dbk_blocknorm_bprop_workspace": [_P, _P],
    "dbk_blocknorm_bprop": [_P, _P, _P, _Z],
    "dbk_causalconv_workspace": [_I, _Z, _Z, _Z, _Z, _I, _P],
    "dbk_causalconv": [_P, _I, _P, _Z, _P, _P, _Z, _Z, _Z, _P, _Z, _I, _P, _P, _Z, _P, _P, _Z],
    "dbk_causalconv_bprop": [_P, _I, _P, _Z, _P, _P, _Z, _Z, _Z, _P, _Z, _I, _P, _Z, _P, _Z, _P, _P, _P, _Z],
    "dbk_causalconv_step": [_P, _I, _P, _Z, _P, _P, _Z, _Z, _Z, _I, _P, _P, _P, _Z],
    "dbk_statescan_args_size": [],
    "dbk_statescan_workspace": [_P, _I, _P],
    "dbk_statescan": [_P, _P, _P, _Z],
    "dbk_statescan_bprop": [_P, _P, _P, _Z],
    "dbk_statescan_step": [_P, _P],
    "dbk_deltarule_args_size": [],
    "dbk_deltarule_kept": [_P, _P],
    "dbk_deltarule_workspace": [_P, _I, _P],
    "dbk_deltarule": [_P, _P, _P, _Z],
    "dbk_deltarule_bprop": [_P, _P, _P, _Z],
    "dbk_deltarule_step": [_P, _P],
    "dbk_clip_gradients_workspace": [_Z, _P, _Z, _P],
    "dbk_clip_gradients": [_P, _Z, _P, _Z, _D, _P, _P, _Z],
    "dbk_train_step": [_P, _P],
    "dbk_train_steps": [_P, _Z, _P],
    "dbk_train_step_single_workspace": [_P, _P],
    "dbk_train_step_single_pays": [_P],
    "dbk_longest_region": [_P, _P, _Z, _P],
    "dbk_train_step_single": [_P, _P, _P, _Z],
    "dbk_train_step_args_size": [],
}


class TrainStepArgs(ctypes.Structure):
    """dbk_train_step_args of the public header, field for field."""
    _fields_ = [
        ("nmodel", _Z), ("nfilter", _Z), ("m", _Z), ("hidden", _Z),
        ("ptype", _I), ("loss_kind", _I), ("reverse_complement", _I), ("nesterov", _I),
        ("nparam", _Z),
        ("P", _P), ("dP", _P), ("mP", _P), ("drate", _P), ("mrate", _P),
        ("off_Wc", _Z), ("off_bc", _Z), ("off_W1", _Z), ("off_b1", _Z), ("off_W2", _Z), ("off_b2", _Z),
        ("X", _P), ("N", _Z), ("regions", _P), ("nregion", _Z), ("Y", _P), ("Ymask", _P),
        ("input_rate", _F), ("Xdrop", _P), ("Mdrop", _P),
        ("rate", _P), ("seed", _U64), ("counter", _P),
        ("decay", _P), ("freeze_scan", _I),
        ("pooled", _P), ("argmax", _P), ("Z", _P), ("dpooled", _P), ("loss", _P), ("act", _P),
        ("L", _P), ("L_ready", _I),
        ("nfeat", _Z), ("feats", _P),
        ("ycol", _P), ("ldY", _Z),
    ]


class ClipTensor(ctypes.Structure):
    """dbk_clip_tensor of the public header, field for field."""
    _fields_ = [("in_", _P), ("out", _P), ("rows", _Z), ("cols", _Z), ("ld_in", _Z), ("ld_out", _Z), ("dtype", _I), ("by_rows", _I)]


class BlockNormArgs(ctypes.Structure):
    """dbk_blocknorm_args of the public header, field for field."""
    _fields_ = [
        ("dtype", _I), ("rms", _I), ("norm", _I), ("next", _I), ("n", _Z), ("m", _Z), ("group", _Z), ("eps", _D),
        ("Y", _P), ("ldy", _Z), ("R", _P), ("ldr", _Z), ("gate", _P), ("ldgate", _Z),
        ("gamma", _P), ("beta", _P), ("scale", _P), ("next_gamma", _P), ("next_beta", _P),
        ("O", _P), ("ldo", _Z), ("Z", _P), ("ldz", _Z), ("stats", _P), ("dR", _P), ("lddr", _Z), ("dZ", _P), ("lddz", _Z),
        ("dY", _P), ("lddy", _Z), ("dR_in", _P), ("lddr_in", _Z), ("dgate", _P), ("lddgate", _Z),
        ("dgamma", _P), ("dbeta", _P), ("dscale", _P), ("dnext_gamma", _P), ("dnext_beta", _P),
    ]


class StateScanArgs(ctypes.Structure):
    """dbk_statescan_args of the public header, field for field."""
    _fields_ = [
        ("dtype", _I), ("softplus", _I), ("N", _Z), ("D", _Z), ("S", _Z), ("G", _Z), ("regions", _P), ("nregion", _Z),
        ("X", _P), ("ldx", _Z), ("dt", _P), ("lddt", _Z), ("A", _P), ("B", _P), ("ldb", _Z), ("C", _P), ("ldc", _Z),
        ("skip", _P), ("dt_bias", _P), ("gate", _P), ("ldgate", _Z), ("state", _P), ("Y", _P), ("ldy", _Z), ("last", _P), ("keep", _P),
        ("dY", _P), ("lddy", _Z), ("dX", _P), ("lddx", _Z), ("ddt", _P), ("ldddt", _Z), ("dgate", _P), ("lddgate", _Z),
        ("dB", _P), ("lddb", _Z), ("dC", _P), ("lddc", _Z), ("dA", _P), ("dskip", _P), ("ddt_bias", _P),
    ]


class DeltaRuleArgs(ctypes.Structure):
    """dbk_deltarule_args of the public header, field for field."""
    _fields_ = [
        ("dtype", _I), ("N", _Z), ("H", _Z), ("G", _Z), ("K", _Z), ("V", _Z), ("regions", _P), ("nregion", _Z),
        ("Q", _P), ("ldq", _Z), ("Kk", _P), ("ldk", _Z), ("Vv", _P), ("ldv", _Z), ("beta", _P), ("ldbeta", _Z), ("decay", _P), ("lddecay", _Z),
        ("scale", _D), ("state", _P), ("O", _P), ("ldo", _Z), ("last", _P), ("keep", _P),
        ("dO", _P), ("lddo", _Z), ("dQ", _P), ("lddq", _Z), ("dK", _P), ("lddk", _Z), ("dV", _P), ("lddv", _Z),
        ("dbeta", _P), ("lddbeta", _Z), ("ddecay", _P), ("ldddecay", _Z),
    ]


_dll = None


def dll():
    """The loaded shared library; raises if it has not been built."""
    global _dll
    if _dll is None:
        if not os.path.exists(LIB_PATH):
            raise DeepbindError("libdeepbind_hip.so is missing (%s): build it with `python -m deepbind_amd.build`; "
                                "there is no fallback path" % LIB_PATH)
        lib = ctypes.CDLL(LIB_PATH)
        lib.dbk_last_error.restype = c_char_p
        lib.dbk_last_error.argtypes = []
        for name, argtypes in _SIGNATURES.items():
            fn = getattr(lib, name)
            fn.restype = c_int
            fn.argtypes = argtypes
        _dll = lib
    return _dll


def exported_names():
    return ["dbk_last_error"] + sorted(_SIGNATURES)


def call(name, *args):
    """Calls lib.<name>(*args) and raises DeepbindError with the library's message on failure."""
    lib = _dll or dll()
    rc = getattr(lib, name)(*args)
    if rc != 0:
        msg = lib.dbk_last_error()
        raise DeepbindError("%s: %s" % (name, msg.decode("utf-8", "replace") if msg else "error %d" % rc))
    return rc


def stream():
    """The current HIP stream of the current device, as the void* the library expects."""
    # (the raw handle: building torch's stream object costs as much as a whole call of the library)
    if not torch.cuda.is_initialized():
        torch.cuda.init()
    return c_void_p(torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice()))


def ptr(t):
    """Device pointer of a contiguous tensor (None -> NULL)."""
    if t is None:
        return None
    if not t.is_cuda:
        raise DeepbindError("TypeError: expected a device tensor, got a host tensor")
    if not t.is_contiguous():
        raise DeepbindError("ValueError: tensors passed to the library must be contiguous (full stride)")
    return c_void_p(t.data_ptr())


def dtype_code(t):
    if t.dtype == torch.float32:
        return DBK_F32
    if t.dtype == torch.float64:
        return DBK_F64
    raise DeepbindError("TypeError: expected a float32 or float64 tensor, got %s" % t.dtype)


ROW_DTYPES = {torch.float32: DBK_F32, torch.float64: DBK_F64, torch.bfloat16: DBK_BF16}


def row_dtype_code(t):
    """Type code of a matrix of rows of the row operators."""
    code = ROW_DTYPES.get(t.dtype)
    if code is None:
        raise DeepbindError("TypeError: expected float32, float64 or bfloat16 rows, got %s" % t.dtype)
    return code


def wide_dtype(t):
    """The type of the weights, statistics and states that go with rows of t's type."""
    return torch.float64 if t.dtype is torch.float64 else torch.float32


# (the checks below build their messages only where they fail: a call on a few rows costs the host no more than the device)
def _shape_or_type(name, t, shape, dtype, what):
    if not isinstance(t, torch.Tensor) or t.shape != shape:
        raise DeepbindError("ValueError: %s must be %s, got %s" % (name, what % (tuple(shape),), tuple(t.shape) if isinstance(t, torch.Tensor) else type(t).__name__))
    raise DeepbindError("TypeError: %s must be %s, got %s" % (name, dtype, t.dtype))


_ITEM = {torch.float32: 4, torch.float64: 8, torch.bfloat16: 2, torch.uint32: 4, torch.int32: 4}


class Arguments(object):
    """The tensors of one call of a row operator: each is checked as it is added, for shape, type and layout, and all of them in check()."""
    __slots__ = ("ins", "outs")

    def __init__(self):
        self.ins, self.outs = [], []

    def rows(self, name, t, shape, dtype, out=False):
        """A matrix of rows, its own row stride, elements of a row next to each other: (pointer, row stride)."""
        if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype is not dtype:
            _shape_or_type(name, t, shape, dtype, "a %s matrix")
        p = t.data_ptr()
        n, ld = shape
        if t.is_contiguous():
            hi = p + n * ld * _ITEM[dtype]
        else:
            step, one = t.stride()
            if ld > 1 and one != 1:
                raise DeepbindError("ValueError: the elements of a row of %s must lie next to each other" % name)
            if n > 1:
                if step < ld:
                    raise DeepbindError("ValueError: the rows of %s must not overlap" % name)
                hi = p + ((n - 1) * step + ld) * _ITEM[dtype]
                ld = step
            else:
                hi = p + ld * _ITEM[dtype]
        (self.outs if out else self.ins).append((p, hi, t.get_device(), t))
        return p, ld

    def dense(self, name, t, shape, dtype, out=False):
        """The pointer of a contiguous array of weights or states; None passes."""
        if t is None:
            return None
        if not isinstance(t, torch.Tensor) or t.shape != shape or t.dtype is not dtype:
            _shape_or_type(name, t, shape, dtype, "%s")
        if not t.is_contiguous():
            raise DeepbindError("ValueError: %s must be contiguous" % name)
        p = t.data_ptr()
        (self.outs if out else self.ins).append((p, p + t.numel() * _ITEM[dtype], t.get_device(), t))
        return p

    def check(self):
        """Everything on the current device, whose stream the call runs on, and no output on an input's memory or another output's."""
        current = None
        for _, _, at, _ in self.ins + self.outs:
            if at != current:
                if at < 0:
                    raise DeepbindError("TypeError: expected a device tensor, got a host tensor")
                current = torch.cuda.current_device()
                if at != current:
                    raise DeepbindError("ValueError: a tensor lies on device %d, the current device is %d" % (at, current))
        known = self.ins
        for out in self.outs:
            lo, hi, _, t = out
            if lo == hi:
                continue
            for lo2, hi2, _, t2 in known:
                # (blocks of columns of one wider matrix: their spans overlap, their elements need not)
                if lo < hi2 and lo2 < hi and lo2 != hi2 and not _column_blocks(*((t, t2) if lo <= lo2 else (t2, t))):
                    raise DeepbindError("ValueError: an output shares memory with another argument")
            known = known + [out]


def check_many(a):
    """Arguments.check for long lists: pairs are compared one by one only where memory of some tensors overlaps at all."""
    every = a.ins + a.outs
    current = every[0][2]
    if current < 0 or any(t[2] != current for t in every) or current != torch.cuda.current_device():
        return a.check()
    end = 0
    for lo, hi in sorted([(t[0], t[1]) for t in every if t[0] != t[1]]):
        if lo < end:
            return a.check()
        end = hi


def _column_blocks(a, b):
    """Whether b, which starts no earlier than a, is another block of columns of the same matrix."""
    if a.dim() != 2 or b.dim() != 2 or a.stride(0) != b.stride(0) or a.element_size() != b.element_size():
        return False
    ld = a.stride(0)
    if ld < a.shape[1]:                          # (one row, whose stride says nothing)
        return False
    off = (b.data_ptr() - a.data_ptr()) // a.element_size()
    return off % ld >= a.shape[1] and off % ld + b.shape[1] <= ld


def row_stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def workspace(nbytes, like):
    """Scratch of one call, from torch's allocator: its own under capture, returned to the stream's pool afterwards. (tensor, pointer)"""
    if not nbytes:
        return None, None
    t = torch.empty(nbytes, dtype=torch.uint8, device=like.device)
    return t, t.data_ptr()


def require(cond, msg):
    if not cond:
        raise DeepbindError(msg)
