"""ctypes binding of the C-ABI in include/attn_bwd_b200.h.

The shared library is built in-tree (``__graft_entry__.build()``) next to this
file.  There is no fallback: if the library is missing, every entry point
raises.
"""
import ctypes
import os

LIB_NAME = "libattn_bwd_b200.so"
# ATTN_BWD_B200_LIB may point at another build of the same library (e.g. a tuning variant).
LIB_PATH = os.environ.get("ATTN_BWD_B200_LIB") or os.path.join(os.path.dirname(os.path.abspath(__file__)), LIB_NAME)

# C-ABI error codes (enum in include/attn_bwd_b200.h)
OK, EINVAL, EALIGN, EUNSUPPORTED, ETMAP, ECUDA, EDEVICE, EKERNEL = range(8)

_VP, _I, _F, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_int64
_L3 = ctypes.c_int64 * 3

DT_BF16, DT_FP16, DT_FP32 = range(3)   # ATTN_BWD_DT_*


class RopeArgs(ctypes.Structure):
    """attn_bwd_rope_t"""
    _fields_ = [(n, _I) for n in ("bs", "seq", "q_heads", "k_heads", "head_dim", "rotary_dim", "dtype", "interleaved",
                                  "inverse")] + [
        ("factor", _F), ("position_stride", _L), ("q_in", _L3), ("k_in", _L3), ("q_out", _L3), ("k_out", _L3)]


class FusedArgs(ctypes.Structure):
    """attn_bwd_fused_t"""
    _fields_ = [(n, _I) for n in ("bs", "seq_q", "seq_kv", "heads", "kv_heads", "head_dim", "dtype", "causal")] + [
        ("scale", _F), ("softcap", _F)] + [
        (n, _VP) for n in ("slopes", "prefix_lens", "q_documents", "kv_documents")] + [
        (n, _L3) for n in ("q_stride", "k_stride", "v_stride", "dq_stride", "dk_stride", "dv_stride")]


_ROPE_P, _FUSED_P = ctypes.POINTER(RopeArgs), ctypes.POINTER(FusedArgs)

# Every symbol the header declares, with its ctypes signature.
SIGNATURES = {
    "attn_bwd_b200": (_I, [_VP, _VP, _VP, _VP, _VP, _F, _I, _I, _I, _VP, _VP, _VP]),
    "attn_bwd_b200_shard": (_I, [_VP, _VP, _VP, _VP, _VP, _F, _I, _I, _I, _I, _I, _VP, _VP, _VP]),
    "attn_bwd_b200_ds_shard": (_I, [_VP, _VP, _VP, _VP, _F, _I, _I, _I, _I, _I, _VP, _VP]),
    "attn_bwd_b200_dv_shard": (_I, [_VP, _VP, _I, _I, _I, _I, _I, _VP, _VP]),
    "attn_bwd_b200_shard_from_mask": (_I, [_VP, _VP, _VP, _VP, _F, _I, _I, _I, _I, _I, _VP, _VP, _VP]),
    "attn_bwd_b200_host_shard": (_I, [_VP] * 5 + [_F, _I, _I, _I, _I, _I] + [_VP] * 9 + [_I, _VP]),
    "attn_bwd_b200_host": (_I, [_VP] * 5 + [_F, _I, _I, _I] + [_VP] * 9 + [_I, _VP]),
    "attn_bwd_b200_rope": (_I, [_ROPE_P] + [_VP] * 7),
    "attn_bwd_b200_fused_workspace": (_L, [_FUSED_P, _I]),
    "attn_bwd_b200_fused_fwd": (_I, [_FUSED_P] + [_VP] * 6 + [_L, _VP]),
    "attn_bwd_b200_fused_bwd": (_I, [_FUSED_P] + [_VP] * 10 + [_L, _VP]),
    "attn_bwd_b200_poll_error": (_I, []),
    "attn_bwd_b200_selftest_wait_timeout": (_I, [_I, _VP]),
    "attn_bwd_b200_strerror": (ctypes.c_char_p, [_I]),
    "attn_bwd_b200_version": (_I, []),
    "attn_bwd_b200_release": (_I, []),
    "attn_bwd_b200_set_option": (_I, [_I, _I]),
    "attn_bwd_b200_get_option": (_I, [_I]),
}

# Measurement / test options (ATTN_BWD_OPT_* in include/attn_bwd_b200.h); -1 = automatic.
OPTIONS = {"ds_mode": 0, "row_kind": 1, "ds_cluster": 2, "l2_prefetch": 3, "l2_hint": 4, "split": 5,
           "dv_sms": 6, "side_stream": 7, "graph": 8, "map_cache": 9}

_lib = None


class AttnBwdError(RuntimeError):
    """A C-ABI call returned a non-zero ATTN_BWD_E* code."""

    def __init__(self, fn, code):
        self.code = code
        super().__init__(f"{fn} failed: {code} ({strerror(code)})")


def load():
    """Load the in-tree library (once).  Raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"attn_bwd_b200 CUDA library not built: {LIB_PATH} is missing "
                "(run __graft_entry__.build()); there is no CPU fallback")
        lib = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            f = getattr(lib, name)
            f.restype = res
            f.argtypes = args
        _lib = lib
    return _lib


def fast_fn():
    """The bound attn_bwd_b200 entry point (loads the library on first use)."""
    return load().attn_bwd_b200


def strerror(code):
    return load().attn_bwd_b200_strerror(int(code)).decode()


def set_option(name, value):
    """Sets one measurement / test option (process-wide; -1 restores the automatic choice)."""
    call("attn_bwd_b200_set_option", OPTIONS[name], int(value))


def get_option(name):
    return load().attn_bwd_b200_get_option(OPTIONS[name])


def call(name, *args):
    rc = getattr(load(), name)(*args)
    if rc != OK:
        raise AttnBwdError(name, rc)


_binding = []


def binding():
    """The C++ host binding (csrc/torch_fast.cpp), or None when it is not built or when
    ATTN_BWD_B200_LIB selects another build of the library (the binding links the in-tree
    one) or ATTN_BWD_NO_TORCH_BINDING is set."""
    if not _binding:
        mod = None
        if not (os.environ.get("ATTN_BWD_B200_LIB") or os.environ.get("ATTN_BWD_NO_TORCH_BINDING")):
            try:
                from . import _torch_fast as mod
            except ImportError:
                mod = None
        _binding.append(mod)
    return _binding[0]


def bound(name, *args):
    """Calls a function of the C++ binding; None where it declines (the general path then looks
    at the arguments), AttnBwdError where the library refuses the call."""
    mod = binding()
    if mod is None:
        return None
    try:
        r = getattr(mod, name)(*args)
    except TypeError:   # not what it takes: the general path reports it
        return None
    if isinstance(r, int):
        raise AttnBwdError("attn_bwd_b200_" + name.removesuffix("_into"), r)
    return r
