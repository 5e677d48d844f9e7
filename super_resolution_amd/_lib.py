"""ctypes binding of libgpsr.so (the C ABI declared in include/gpsr.h).

The HIP library is the product path: there is NO CPU fallback.  If the shared
object is missing or cannot be loaded, every compute entry point raises.
"""
import ctypes
import glob
import os
import subprocess

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("GPSR_LIB", os.path.join(_HERE, "libgpsr.so"))   # override: instrumented debug builds (tools/upd_trace.py)
_CSRC = os.path.join(_HERE, "csrc")
SRC = os.path.join(_CSRC, "gpsr_api.hip")
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
# no packed float32 arithmetic: some of its forms have given wrong results on this hardware
HIPCC_FLAGS = ["-O3", "--offload-arch=gfx950", "-shared", "-fPIC", "-ffp-contract=off",
               "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]

_lib = None

c_void_p, c_int, c_float, c_size_t = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t


class Bank(ctypes.Structure):
    """gpsr_bank of include/gpsr.h."""
    _fields_ = [(n, c_void_p) for n in ("k_codes", "k_scales", "v_codes", "v_scales", "offset", "centroid")] + [
        ("pages", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("heads", "page_rows", "dim", "bits", "kernel_id")]


# name -> (restype, argtypes); must list every symbol include/gpsr.h declares
SIGNATURES = {
    "gpsr_version": (ctypes.c_char_p, []),
    "gpsr_last_error": (ctypes.c_char_p, []),
    "gpsr_padded_n": (c_int, [c_int]),
    "gpsr_create": (c_void_p, [c_int, c_int, c_int, c_int]),
    "gpsr_destroy": (None, [c_void_p]),
    "gpsr_ctx_workspace": (c_void_p, [c_void_p]),
    "gpsr_ctx_workspace_bytes": (c_size_t, [c_void_p]),
    "gpsr_flag_count": (c_int, [c_void_p, c_int, c_void_p]),
    "gpsr_gather": (c_int, [c_void_p] * 3 + [c_int] * 4 + [c_void_p, c_int, c_void_p, c_int] + [c_void_p] * 4),
    "gpsr_init_hypers": (c_int, [c_void_p, c_int, c_int, c_int, c_float, c_float, c_void_p, c_int, c_void_p, c_void_p]),
    "gpsr_covariance": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "gpsr_covariance_grad": (c_int, [c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p]),
    "gpsr_invert_workspace_bytes": (c_size_t, [c_int, c_int]),
    "gpsr_invert": (c_int, [c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "gpsr_fit_workspace_bytes": (c_size_t, [c_int, c_int, c_int]),
    "gpsr_fit": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_float,
                         c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "gpsr_noalloc_scratch_bytes": (c_size_t, []),
    "gpsr_fit_noalloc": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_float,
                                 c_void_p, c_void_p, c_void_p, c_void_p]),
    "gpsr_set_dual_stream": (c_int, [c_int]),
    "gpsr_set_split_small": (c_int, [c_int]),
    "gpsr_set_fused": (c_int, [c_int]),
    "gpsr_loss_grad": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p,
                               c_void_p, c_void_p, c_size_t, c_void_p]),
    "gpsr_predict": (c_int, [c_void_p] * 4 + [c_int] * 4 + [c_void_p, c_void_p]),
    "gpsr_combine": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_int, c_void_p, c_int,
                             c_int, c_int, c_void_p, c_void_p]),
    "gpsr_predict_pixels_workspace_bytes": (c_size_t, [c_int] * 5),
    "gpsr_predict_pixels": (c_int, [c_void_p] * 3 + [c_int] * 4 + [c_void_p, c_int, c_void_p, c_int, c_void_p, c_int]
                            + [c_int, c_float, c_float, c_int, c_float, c_int, c_int]
                            + [c_void_p, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "gpsr_agpr_weights": (c_int, [c_void_p, c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p]),
    "gpsr_agpr_filter": (c_int, [c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p]),
    "gpsr_selftest_mfma": (c_int, [c_void_p, c_void_p, c_void_p, c_void_p]),
    "gpsr_profile_select": (c_int, [ctypes.c_uint]),
    "gpsr_profile_begin": (c_int, [c_int]),
    "gpsr_profile_end": (c_int, [c_void_p, c_void_p]),
    "gpsr_u8_to_unit": (c_int, [c_void_p, c_void_p, c_size_t, c_void_p]),
    "gpsr_unit_to_u8": (c_int, [c_void_p, c_void_p, c_size_t, ctypes.c_double, c_void_p]),
    "gpsr_resample": (c_int, [c_void_p, c_int, c_int, c_void_p, c_int, c_int] + [c_void_p] * 4 + [c_int, c_void_p]),
    "gpsr_decimate2": (c_int, [c_void_p, c_int, c_int, c_void_p, c_void_p]),
    "gpsr_sepfilter_sym": (c_int, [c_void_p, c_int, c_int, c_void_p, c_void_p, c_int, c_void_p]),
    "gpsr_filter3x3": (c_int, [c_void_p, c_int, c_int, c_void_p, c_void_p, c_void_p]),
    "gpsr_axpy": (c_int, [c_void_p, c_void_p, ctypes.c_double, c_void_p, c_size_t, c_void_p]),
    "gpsr_bgr2gray": (c_int, [c_void_p, c_void_p, c_size_t, c_void_p]),
    "gpsr_bgr2yuv": (c_int, [c_void_p] * 4 + [c_size_t, c_void_p]),
    "gpsr_yuv2bgr": (c_int, [c_void_p] * 4 + [c_size_t, c_void_p]),
    "gpsr_bgr2ycrcb": (c_int, [c_void_p] * 4 + [c_size_t, c_void_p]),
    "gpsr_ycrcb2bgr": (c_int, [c_void_p] * 4 + [c_size_t, c_void_p]),
    "gpsr_resample_u8": (c_int, [c_void_p, c_int, c_int, c_void_p, c_int, c_int] + [c_void_p] * 5),
    "gpsr_active_sample_workspace_bytes": (c_size_t, [c_int]),
    "gpsr_active_sample": (c_int, [c_void_p, c_int, c_int, c_int, c_int, ctypes.c_double, ctypes.c_double,
                                   ctypes.c_double, c_void_p, c_void_p, c_void_p, c_size_t, c_void_p]),
    "gpsr_bank_write": (c_int, [c_void_p, c_void_p, c_int, c_int] + [c_void_p] * 4 + [c_int, c_int] + [c_void_p] * 3),
    "gpsr_bank_read": (c_int, [c_void_p, c_void_p, c_int, c_int] + [c_void_p] * 4 + [c_int, c_int, c_void_p]),
    "gpsr_bank_attend_workspace_bytes": (c_size_t, [c_void_p] + [c_int] * 5),
    "gpsr_bank_attend": (c_int, [c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p,
                                 c_float] + [c_void_p] * 4 + [c_size_t, c_void_p]),
    "gpsr_bank_select_workspace_bytes": (c_size_t, [c_void_p] + [c_int] * 6),
    "gpsr_bank_select": (c_int, [c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p, c_int, c_int, c_int, c_void_p,
                                 c_int] + [c_void_p] * 3 + [c_size_t, c_void_p]),
    "gpsr_bank_attend_pages_workspace_bytes": (c_size_t, [c_void_p] + [c_int] * 6),
    "gpsr_bank_attend_pages": (c_int, [c_void_p, c_void_p, c_int, c_int, c_void_p, c_void_p, c_int, c_int, c_int,
                                       c_void_p, c_void_p, c_int, c_float] + [c_void_p] * 4 + [c_size_t, c_void_p]),
    "gpsr_bank_windows": (c_int, [c_void_p] + [c_int] * 4 + [c_void_p, c_int, c_int, c_void_p]),
    "gpsr_bank_blend": (c_int, [c_void_p] + [c_int] * 3 + [c_void_p, c_int, c_int, c_void_p, c_void_p]),
    "gpsr_sepfilter_u8": (c_int, [c_void_p, c_int, c_int, c_void_p, c_void_p, c_int, c_void_p]),
    "gpsr_metrics_workspace_bytes": (c_size_t, [c_int, c_int, c_int]),
    "gpsr_metrics": (c_int, [c_void_p, c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_size_t, c_void_p]),
}


def build(force=False):
    """Compile csrc/*.hip for gfx950 (one object per file, side by side) into libgpsr.so (in-tree); what was built by another
    compiler or with other flags (build/command) is built again."""
    from concurrent.futures import ThreadPoolExecutor
    heads = glob.glob(os.path.join(_CSRC, "*.hpp")) + [os.path.join(os.path.dirname(_HERE), "include", "gpsr.h")]
    srcs = sorted(glob.glob(os.path.join(_CSRC, "*.hip")))
    newer = lambda path, than: os.path.exists(path) and all(os.path.getmtime(path) >= os.path.getmtime(t) for t in than)
    objdir = os.path.join(_HERE, "build")
    stamp, command = os.path.join(objdir, "command"), " ".join([HIPCC] + HIPCC_FLAGS)
    if not os.path.exists(stamp) or open(stamp).read() != command:
        force = True
    if not force and newer(LIB_PATH, srcs + heads):
        return LIB_PATH
    os.makedirs(objdir, exist_ok=True)
    if os.path.exists(stamp):
        os.remove(stamp)            # until everything is built by it
    flags = [f for f in HIPCC_FLAGS if f != "-shared"]

    def compile_one(src):
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        if force or not newer(obj, [src] + heads):
            subprocess.run([HIPCC] + flags + ["-c", "-o", obj, src], check=True, cwd=_HERE)
        return obj

    with ThreadPoolExecutor(max_workers=min(8, len(srcs))) as pool:
        objs = list(pool.map(compile_one, srcs))
    subprocess.run([HIPCC, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB_PATH] + objs, check=True, cwd=_HERE)
    with open(stamp, "w") as f:
        f.write(command)
    return LIB_PATH


def load():
    """Load libgpsr.so; raises if it is absent (no fallback)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(
            f"{LIB_PATH} not found: the HIP extension is the only compute path "
            "(run `python -c 'import __graft_entry__ as g; g.build()'`)")
    # torch first: the process must hold ONE HIP runtime, the copy torch ships (it owns the device memory and the streams
    # this library is handed).  Loaded before torch, libgpsr.so would bring /opt/rocm's libamdhip64 with it, torch its
    # own afterwards, and the launches of whichever runtime comes second fail with "no ROCm-capable device is detected".
    import torch  # noqa: F401
    lib = ctypes.CDLL(LIB_PATH)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)  # AttributeError if the symbol is not exported
        fn.restype, fn.argtypes = res, args
    _lib = lib
    return lib


class GpsrError(RuntimeError):
    pass


def check(rc, what):
    """Negative status -> exception; positive = number of flagged GPs (returned)."""
    if rc < 0:
        raise GpsrError(f"{what} failed ({rc}): {load().gpsr_last_error().decode()}")
    return rc
