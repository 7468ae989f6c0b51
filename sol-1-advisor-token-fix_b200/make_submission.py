"""Writes a single-file ``submission.py`` for the reference harness.

The reference evaluator takes a submission as source TEXT: it writes the text to a fresh
temporary ``submission.py``, imports it with importlib and calls its module-level
``custom_kernel`` (eval_modal_attn_bwd.py:238-247, 273).  Nothing next to that file is
available, so the generated module carries everything itself:

- the CUDA sources of the library (``csrc/*.cu*`` and ``include/attn_bwd_b200.h``) as string
  literals;
- a build step that, on first import on a machine, writes them to a cache directory
  (``$ATTN_BWD_B200_CACHE``, default ``~/.cache/attn_bwd_b200/<source hash>``) and compiles
  ``libattn_bwd_b200.so`` with nvcc for sm_100a (about a minute; later imports reuse it;
  concurrent first imports are serialised by a file lock);
- ``custom_kernel(data)`` over the library's C-ABI through ctypes, with the reference's
  6-tuple in and the fresh ``(dS, dV)`` out, ordered on the current stream.

Usage: ``python make_submission.py [out_path]`` (default: ``submission.py`` next to this
file).  ``build_text()`` returns the text without writing it.
"""
import hashlib
import os
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
HEADER = os.path.join(ROOT, "include", "attn_bwd_b200.h")
# what attn_bwd_b200.cu includes; the library's other translation units (rope, fused attention)
# serve calls that a submission does not make
KERNEL_SOURCES = ("attn_bwd_b200.cu", "host_shared.h", "ds_kernel.cuh", "dv_kernel.cuh", "sm100.cuh")

_TEMPLATE = r'''"""Single-file submission: GQA attention backward on hand-written sm_100a (B200) kernels.

Generated by make_submission.py from the library's CUDA sources (source hash {digest});
edit those, not this file.  Drop-in for the reference's custom_kernel
(starting_point.py:27-70): same 6-tuple in, fresh (grad_attn_scores, grad_value_states)
out, ordered on torch.cuda.current_stream().  On first import the embedded sources are
compiled with nvcc into a cached shared library (see _build); there is no CPU fallback.
"""
import ctypes
import fcntl
import os
import subprocess

import torch

_DIGEST = "{digest}"
_SOURCES = {sources}
_KERNEL_SOURCES = {kernel_sources!r}
_NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17", "-shared",
               "-Xcompiler", "-fPIC,-O2", "-Xlinker", "-soname=libattn_bwd_b200.so"]


def _cache_dir():
    base = os.environ.get("ATTN_BWD_B200_CACHE") or os.path.join(os.path.expanduser("~"), ".cache", "attn_bwd_b200")
    return os.path.join(base, _DIGEST)


def _build():
    """Path of the compiled library, compiling it first if this machine has no copy."""
    d = _cache_dir()
    lib = os.path.join(d, "libattn_bwd_b200.so")
    if os.path.exists(lib):
        return lib
    os.makedirs(os.path.join(d, "src", "csrc"), exist_ok=True)
    os.makedirs(os.path.join(d, "include"), exist_ok=True)
    with open(os.path.join(d, ".lock"), "w") as lk:
        fcntl.flock(lk, fcntl.LOCK_EX)
        if os.path.exists(lib):
            return lib
        for name, text in _SOURCES.items():
            sub = "include" if name == "attn_bwd_b200.h" else os.path.join("src", "csrc")
            with open(os.path.join(d, sub, name), "w") as f:
                f.write(text)
        nvcc = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "bin", "nvcc")
        if not os.path.exists(nvcc):
            nvcc = "nvcc"
        tmp = lib + ".tmp"
        r = subprocess.run([nvcc] + _NVCC_FLAGS + ["-o", tmp, os.path.join(d, "src", "csrc", "attn_bwd_b200.cu")],
                           capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError("nvcc failed building the attention-backward library:\n" + r.stderr[-4000:])
        os.replace(tmp, lib)
    return lib


_lib = ctypes.CDLL(_build())
_vp, _i = ctypes.c_void_p, ctypes.c_int
_lib.attn_bwd_b200.restype = _i
_lib.attn_bwd_b200.argtypes = [_vp, _vp, _vp, _vp, _vp, ctypes.c_float, _i, _i, _i, _vp, _vp, _vp]
_lib.attn_bwd_b200_strerror.restype = ctypes.c_char_p
_lib.attn_bwd_b200_strerror.argtypes = [_i]


def _ready(t, dtype, name):
    if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
        raise ValueError(f"{{name}}: expected a CUDA tensor (no CPU path)")
    if t.dtype != dtype:
        raise TypeError(f"{{name}}: expected {{dtype}}, got {{t.dtype}}")
    if not t.is_contiguous() or t.data_ptr() % 16:
        t = t.contiguous() if not t.is_contiguous() else t.clone()
    return t


def custom_kernel(data):
    """(grad_attn_output [bs,sq,80,128], attn_weights [bs,80,sq,skv], attn_weights_dropped,
    value_states [bs,8,skv,128], dropout_mask [bs,80,sq,skv] bool, attention_dropout)
    -> (grad_attn_scores [bs,80,sq,skv], grad_value_states [bs,8,skv,128]), bf16."""
    dO, P, Pd, V, M, p = data
    dO = _ready(dO, torch.bfloat16, "grad_attn_output")
    P = _ready(P, torch.bfloat16, "attn_weights")
    Pd = _ready(Pd, torch.bfloat16, "attn_weights_dropped")
    V = _ready(V, torch.bfloat16, "value_states")
    M = _ready(M, torch.bool, "dropout_mask")
    bs, sq, h, d = dO.shape
    skv = V.shape[2]
    if h != 80 or d != 128 or tuple(V.shape) != (bs, 8, skv, 128):
        raise ValueError(f"expected grad_attn_output [bs,sq,80,128] and value_states [bs,8,skv,128], "
                         f"got {{tuple(dO.shape)}} and {{tuple(V.shape)}}")
    for t, name in ((P, "attn_weights"), (Pd, "attn_weights_dropped"), (M, "dropout_mask")):
        if tuple(t.shape) != (bs, 80, sq, skv):
            raise ValueError(f"{{name}}: expected {{(bs, 80, sq, skv)}}, got {{tuple(t.shape)}}")
    with torch.cuda.device(dO.device):
        dS = torch.empty_like(P)
        dV = torch.empty_like(V)
        rc = _lib.attn_bwd_b200(dO.data_ptr(), P.data_ptr(), Pd.data_ptr(), V.data_ptr(), M.data_ptr(), float(p),
                                bs, sq, skv, dS.data_ptr(), dV.data_ptr(), torch.cuda.current_stream().cuda_stream)
    if rc:
        raise RuntimeError(f"attn_bwd_b200 failed: {{rc}} ({{_lib.attn_bwd_b200_strerror(rc).decode()}})")
    return dS, dV
'''


def _sources():
    out = {}
    for name in KERNEL_SOURCES:
        with open(os.path.join(CSRC, name)) as f:
            out[name] = f.read()
    with open(HEADER) as f:
        out["attn_bwd_b200.h"] = f.read()
    return out


def build_text():
    """The submission's source text."""
    src = _sources()
    for name, text in src.items():
        if "'''" in text or text.endswith("\\"):   # would end the raw literal early
            raise ValueError(f"{name} cannot be embedded as a raw triple-quoted literal")
    digest = hashlib.sha256("".join(k + v for k, v in sorted(src.items())).encode()).hexdigest()[:16]
    lits = "{\n" + "".join(f"    {k!r}: r'''{v}''',\n" for k, v in src.items()) + "}"
    return _TEMPLATE.format(digest=digest, sources=lits, kernel_sources=KERNEL_SOURCES)


def main(argv):
    out = argv[1] if len(argv) > 1 else os.path.join(HERE, "submission.py")
    text = build_text()
    with open(out, "w") as f:
        f.write(text)
    print(f"wrote {out} ({len(text)} bytes)")


if __name__ == "__main__":
    main(sys.argv)
