"""ctypes binding of libvc3d.so (include/vc3d.h).

The library is the product's compute path.  There is no fallback: if the shared object
is missing or a symbol does not resolve, importing fails loudly.
"""
import ctypes as C
import os

# torch must be imported BEFORE libvc3d.so is loaded: the library has to bind to the HIP runtime
# that torch ships (one runtime per process, shared streams and device memory).  Loading
# /opt/rocm's runtime first leaves the process with two half-initialised runtimes
# ("no ROCm-capable device is detected").
import torch  # noqa: F401

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("VC3D_LIB") or os.path.join(_HERE, "libvc3d.so")  # VC3D_LIB: experiment builds

VC_STAT_REPLICAS = 32
VC_TICKET_WORDS = 64  # int32 words behind a ticket pointer (bn_fin.h)
STEM_K = 1344


class Vc3dError(RuntimeError):
    pass


class ConvDesc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in
                ("N", "Ci", "Ti", "Hi", "Wi", "Co", "kt", "kh", "kw", "st", "sh", "sw", "pt", "ph", "pw")]

    def out_dims(self):
        return ((self.Ti + 2 * self.pt - self.kt) // self.st + 1,
                (self.Hi + 2 * self.ph - self.kh) // self.sh + 1,
                (self.Wi + 2 * self.pw - self.kw) // self.sw + 1)


class PoolDesc(C.Structure):
    _fields_ = [(n, C.c_int32) for n in
                ("N", "C", "T", "H", "W", "kt", "kh", "kw", "st", "sh", "sw", "pt", "ph", "pw")]

    def out_dims(self):
        return ((self.T + 2 * self.pt - self.kt) // self.st + 1,
                (self.H + 2 * self.ph - self.kh) // self.sh + 1,
                (self.W + 2 * self.pw - self.kw) // self.sw + 1)


class BnFin(C.Structure):
    """vc_bn_fin: BatchNorm finalize folded into the launch that produces the sums (include/vc3d.h)."""
    _fields_ = [("ticket", C.c_void_p), ("gamma", C.c_void_p), ("beta", C.c_void_p), ("running_mean", C.c_void_p),
                ("running_var", C.c_void_p), ("params", C.c_void_p), ("count", C.c_float), ("momentum", C.c_float),
                ("eps", C.c_float), ("shift", C.c_void_p), ("shift_next", C.c_void_p)]


_P = C.c_void_p
_I = C.c_int32
_L = C.c_int64
_F = C.c_float
class BnBwdRed(C.Structure):
    """vc_bn_bwd_red: the BatchNorm backward reduction that rides along with vc_conv3d_dgrad_fused (include/vc3d.h)."""
    _fields_ = [(n, C.c_void_p) for n in ("y", "params", "relu_bits", "sums", "ticket", "coef", "dgamma", "dbeta")]


class Cmd(C.Structure):
    """vc_cmd: one recorded call / cross-stream dependency of a command list (include/vc3d.h, vc_replay)."""
    _fields_ = [("fn", C.c_void_p), ("kind", C.c_int32), ("nint", C.c_int32), ("nflt", C.c_int32), ("pad_", C.c_int32),
                ("iarg", C.c_int64 * 16), ("farg", C.c_float * 8)]


CMD_CALL, CMD_EVENT_RECORD, CMD_STREAM_WAIT = 0, 1, 2


class AdamwHyper(C.Structure):
    """vc_adamw_hyper (include/vc3d.h)"""
    _fields_ = [(n, C.c_double) for n in ("lr", "beta1", "beta2", "eps", "weight_decay", "grad_scale")] + [("step", C.c_int64)]


class ScanDesc(C.Structure):
    """vc_scan_desc (include/vc3d.h)"""
    _fields_ = [(n, C.c_int32) for n in ("B", "T", "H", "is_bf16", "reverse", "pad_")] + [("stride_b", C.c_int64), ("stride_t", C.c_int64)]


class LinearCeDesc(C.Structure):
    """vc_linear_ce_desc (include/vc3d.h)"""
    _fields_ = [(n, C.c_int32) for n in ("N", "D", "V", "is_bf16", "reduction", "w_align")] + \
               [(n, C.c_int64) for n in ("ldx", "ldw", "ignore_index", "keep_bytes")]

_CD = C.POINTER(ConvDesc)
_PD = C.POINTER(PoolDesc)
_IP = C.POINTER(C.c_int32)
_BF = C.POINTER(BnFin)
_SD = C.POINTER(ScanDesc)
_LD = C.POINTER(LinearCeDesc)

# name -> argtypes (every function returns int unless listed in _RESTYPE)
PROTOTYPES = {
    "vc_last_error": [],
    "vc_abi_version": [],
    "vc_set_deterministic": [_I],
    "vc_get_deterministic": [],
    "vc_conv3d_out_dims": [_CD, _IP, _IP, _IP],
    "vc_conv3d_workspace_bytes": [_CD, _I],
    "vc_conv3d_fwd": [_CD, _P, _P, _P, _P, _P, C.c_size_t, _P],
    "vc_conv3d_fwd_bn": [_CD, _P, _P, _P, _P, _BF, _P, C.c_size_t, _P],
    "vc_conv3d_fwd_act": [_CD, _P, _P, _P, _P, _P, _I, _P, C.c_size_t, _P],
    "vc_static_scratch_bytes": [],
    "vc_conv3d_fwd_noalloc": [_CD, _P, _P, _P, _P, _P],
    "vc_conv3d_dgrad": [_CD, _P, _P, _P, _I, _P, C.c_size_t, _P],
    "vc_conv3d_dgrad_fused": [_CD, _P, _P, _P, _I, _P, C.POINTER(BnBwdRed), _P, C.c_size_t, _P],
    "vc_conv3d_wgrad": [_CD, _P, _P, _P, _P, C.c_size_t, _P],
    "vc_pack_weight": [_P, _P, _P, _I, _I, _I, _P],
    "vc_sgd_step": [_P, _P, _P, _P, _L, _F, _F, _F, _I, _P],
    "vc_adam_step": [_P, _P, _P, _P, _P, _L, _F, _F, _F, _F, _F, _L, _P],
    "vc_shadow_bf16": [_P, _P, _L, _P],
    "vc_pack_dgrad_batched": [_P, _P, _P, _P, _I, _P],
    "vc_stem_packed_input_elems": [_I, _I, _I, _I],
    "vc_stem_pack_input": [_P, _I, _P, _I, _I, _I, _I, _P],
    "vc_clip_pack_u8": [_P, _P, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, C.POINTER(C.c_float), C.POINTER(C.c_float), _P],
    "vc_stem_pack_weight": [_P, _P, _I, _P],
    "vc_stem_fwd": [_P, _P, _P, _P, _I, _I, _I, _I, _I, _P],
    "vc_stem_fwd_bn": [_P, _P, _P, _P, _BF, _I, _I, _I, _I, _I, _P],
    "vc_stem_wgrad_workspace_bytes": [_I, _I, _I, _I, _I],
    "vc_stem_wgrad": [_P, _P, _P, _I, _I, _I, _I, _I, _P, C.c_size_t, _P],
    "vc_stem_unpack_wgrad": [_P, _P, _I, _P],
    "vc_bn_stats": [_P, _P, _P, _L, _I, _P],
    "vc_bn_finalize": [_P, _I, _F, _P, _P, _P, _P, _F, _F, _P, _P, _P, _P],
    "vc_bn_eval_params": [_I, _P, _P, _P, _P, _F, _P, _P],
    "vc_bn_apply": [_P, _P, _P, _P, _L, _I, _I, _P],
    "vc_bn_apply_mask": [_P, _P, _P, _P, _P, _L, _I, _P],
    "vc_bn_bwd_reduce": [_P, _P, _P, _P, _P, _L, _I, _I, _P],
    "vc_bn_bwd_reduce_fin": [_P, _P, _P, _P, _P, _L, _I, _I, _P, _P, _P, _P, _P],
    "vc_bn_bwd_finalize": [_P, _I, _F, _P, _P, _P, _P],
    "vc_bn_bwd_apply": [_P, _P, _P, _P, _P, _P, _P, _L, _I, _I, _P],
    "vc_add": [_P, _P, _P, _L, _P],
    "vc_pool3d_out_dims": [_PD, _IP, _IP, _IP],
    "vc_maxpool3d_fwd": [_PD, _P, _P, _P, _P, _P],
    "vc_maxpool3d_bwd": [_PD, _P, _P, _P, _P],
    "vc_bn_bwd_reduce_pooled": [_PD, _P, _P, _P, _P, _P, _P, _P],
    "vc_bn_bwd_reduce_pooled_fin": [_PD, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P],
    "vc_bn_bwd_apply_pooled": [_PD, _P, _P, _P, _P, _P, _P, _P],
    "vc_gavgpool_fwd": [_P, _P, _I, _I, _I, _P],
    "vc_gavgpool_bwd": [_P, _P, _I, _I, _I, _P],
    "vc_softmax_ce": [_P, _P, _P, _P, _I, _I, _P],
    "vc_linear_fwd": [_P, _P, _P, _P, _I, _I, _I, _P],
    "vc_linear_bwd": [_P, _P, _P, _P, _P, _P, _I, _I, _I, _P],
    "vc_lstm_pointwise_fwd": [_P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _P],
    "vc_lstm_pointwise_bwd": [_P, _P, _P, _P, _P, _P, _P, _P, _I, _I, _P],
    "vc_adamw_step": [_P, _I, _I, _I, C.POINTER(AdamwHyper), _P, _P],
    "vc_gated_scan_workspace_bytes": [_SD, _I],
    "vc_gated_scan_fwd": [_SD, _P, _P, _P, _P, _P, _P, _P, C.c_size_t, _P],
    "vc_gated_scan_bwd": [_SD, _P, _P, _P, _P, _P, _P, _P, _P, C.c_size_t, _P],
    "vc_gated_scan_step": [_P, _L, _I, _P, _P, _I, _I, _P],
    "vc_bias_columns": [_P, _P, _P, _I, _L, _I, _P],
    "vc_linear_ce_workspace_bytes": [_LD, _I],
    "vc_linear_ce_saved_bytes": [_LD],
    "vc_linear_ce_fwd": [_LD] + [_P] * 7 + [C.c_size_t, _P],
    "vc_linear_ce_bwd": [_LD] + [_P] * 10 + [C.c_size_t, _P],
    "vc_ncthw_to_nthwc": [_P, _I, _P, _I, _I, _L, _P],
    "vc_nthwc_to_ncthw": [_P, _P, _I, _I, _I, _L, _P],
    "vc_replay": [C.POINTER(Cmd), _I, C.POINTER(C.c_void_p), _I, _I, _P, _P, _IP],
    "vc_replay_events_create": [_I, _I, C.POINTER(C.c_void_p)],
    "vc_replay_events_destroy": [_I, C.POINTER(C.c_void_p)],
    "vc_replay_event_elapsed_ms": [_P, _P, C.POINTER(C.c_float)],
    "vc_memset_async": [_P, _I, C.c_size_t, _P],
    "vc_incr_i64": [_P, _I, _P],
}
_RESTYPE = {"vc_last_error": C.c_char_p, "vc_stem_packed_input_elems": C.c_size_t, "vc_static_scratch_bytes": C.c_size_t,
            "vc_conv3d_workspace_bytes": C.c_size_t, "vc_stem_wgrad_workspace_bytes": C.c_size_t,
            "vc_gated_scan_workspace_bytes": C.c_size_t, "vc_linear_ce_workspace_bytes": C.c_size_t,
            "vc_linear_ce_saved_bytes": C.c_size_t}


def _load():
    if not os.path.isfile(LIB_PATH):
        raise Vc3dError(
            "libvc3d.so not found at %s: build it with `make -C video-classification_amd/csrc` "
            "(or __graft_entry__.build()); there is no fallback path" % LIB_PATH)
    lib = C.CDLL(LIB_PATH)
    for name, argtypes in PROTOTYPES.items():
        fn = getattr(lib, name)  # AttributeError if the symbol is missing
        fn.argtypes = argtypes
        fn.restype = _RESTYPE.get(name, C.c_int)
    if lib.vc_abi_version() != 2:
        raise Vc3dError("libvc3d.so ABI version mismatch")
    return lib


_raw = _load()

# The recorder of a command list (vc3d/replay.py) while a step is being recorded, else None.  Every call of an entry
# point goes through _Lib below: the call is made, and -- while recording -- appended to the list with its arguments.
RECORDER = None
_HOST_ONLY = {"vc_abi_version", "vc_conv3d_out_dims", "vc_pool3d_out_dims", "vc_set_deterministic", "vc_get_deterministic",
              "vc_replay", "vc_replay_events_create", "vc_replay_events_destroy", "vc_replay_event_elapsed_ms"}


class _Lib:
    """libvc3d.so's entry points; `lib.vc_xxx(...)` as with the plain CDLL.  A wrapper per entry point is made on first
    use and kept in the instance dict, so later attribute lookups do not come back to __getattr__."""

    def __getattr__(self, name):
        fn = getattr(_raw, name)
        argtypes = fn.argtypes
        recordable = fn.restype is C.c_int and name in PROTOTYPES and name not in _HOST_ONLY

        def call(*args):
            rc = fn(*args)
            if RECORDER is not None and recordable:
                RECORDER.add(name, fn, argtypes, args, rc)
            return rc

        call.__name__ = name
        call.raw = fn
        setattr(self, name, call)
        return call


lib = _Lib()


def check(rc, what=""):
    if rc != 0:
        raise Vc3dError("%s failed (%d): %s" % (what or "vc3d call", rc, lib.vc_last_error().decode()))


def ptr(t):
    """device pointer of a tensor (None -> NULL)."""
    return None if t is None else t.data_ptr()


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_raw_device = getattr(torch._C, "_cuda_getDevice", None)


def cur_stream():
    """raw hipStream_t of torch's current stream on the current device.  The private C accessors are ~20x
    cheaper than torch.cuda.current_stream() (8 us per call, ~150 calls per training step)."""
    if _raw_stream is not None and _raw_device is not None:
        return _raw_stream(_raw_device())
    return torch.cuda.current_stream().cuda_stream
