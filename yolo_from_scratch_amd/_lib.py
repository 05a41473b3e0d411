"""ctypes binding of libyfs.so (include/yfs.h).  No fallback: if the HIP library is missing the
import of any op raises, loudly."""
import ctypes
import os

import torch  # noqa: F401  (must be imported first: libyfs.so binds to the HIP runtime torch loaded)

_HERE = os.path.dirname(os.path.abspath(__file__))
# YFS_LIB_PATH: load another build of the same ABI (A/B measurements of two builds on one GPU box)
LIB_PATH = os.environ.get("YFS_LIB_PATH") or os.path.join(_HERE, "libyfs.so")
_lib = None


class YfsError(RuntimeError):
    pass


def lib():
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise YfsError(
                f"{LIB_PATH} is missing: build it with `make -C {os.path.join(_HERE, 'csrc')}` "
                "(or `python -c 'import __graft_entry__ as g; g.build()'`). There is no CPU fallback.")
        _lib = ctypes.CDLL(LIB_PATH)
        for name in ("yfs_iou_xywh_workspace_bytes", "yfs_yolov1_loss_workspace_bytes", "yfs_mse_workspace_bytes",
                     "yfs_conv2d_wgrad_workspace_bytes", "yfs_sumsq_workspace_bytes",
                     "yfs_conv2d_fwd_workspace_bytes", "yfs_conv2d_dgrad_workspace_bytes",
                     "yfs_conv2d_stem_wgrad_workspace_bytes", "yfs_single_box_loss_workspace_bytes",
                     "yfs_mask_to_boxes_workspace_bytes", "yfs_layer_norm_bwd_workspace_bytes",
                     "yfs_fp8_packed_scale_bytes", "yfs_fp8_gemm_workspace_bytes", "yfs_fp8_matmul_workspace_bytes",
                     "yfs_fp8_linear_saved_bytes", "yfs_fp8_linear_fwd_workspace_bytes", "yfs_fp8_linear_bwd_workspace_bytes"):
            if hasattr(_lib, name):
                getattr(_lib, name).restype = ctypes.c_size_t
        _declare(_lib)
    return _lib


# Entry points whose calls are short enough that ctypes' per-argument objects would show: their argument types are declared
# once, so plain integers (data_ptr(), sizes, the raw stream) are passed as they are.  p pointer, l int64, z size_t, i int,
# f float, d double, u uint64.
_SIGNATURES = {
    "yfs_layer_norm_fwd": "plppppp" "ll" "fi" "p",
    "yfs_layer_norm_bwd": "plpl" "ppp" "ppp" "ll" "i" "pz" "p",
    "yfs_layer_norm_bwd_workspace_bytes": "lli",
    "yfs_fp8_quantize_weight": "pil" "ll" "pppp" "p",
    "yfs_fp8_packed_scale_bytes": "ll",
    "yfs_fp8_quantize_rows": "pil" "ll" "pppp" "p" "p",
    "yfs_fp8_gemm_workspace_bytes": "lll",
    "yfs_fp8_gemm": "pppp" "i" "p" "pi" "lll" "fi" "pz" "p",
    "yfs_fp8_gemm_plan": "llli" "p",
    "yfs_fp8_matmul_workspace_bytes": "lll",
    "yfs_fp8_matmul": "pil" "pp" "p" "pi" "lll" "f" "pz" "p",
    "yfs_fp8_linear_saved_bytes": "llli",
    "yfs_fp8_linear_fwd_workspace_bytes": "lll",
    "yfs_fp8_linear_bwd_workspace_bytes": "llli",
    "yfs_fp8_linear_fwd": "pil" "pil" "p" "pi" "lll" "i" "pz" "pz" "p",
    "yfs_fp8_linear_bwd": "pil" "pi" "pi" "pi" "lll" "i" "pz" "pz" "p",
    "yfs_fp8_colsum": "pllp" "i" "p",
    "yfs_dropout_fwd": "ppl" "df" "u" "p" "i" "p",
    "yfs_dropout_bwd": "pppl" "df" "u" "p" "i" "p",
}
_TYPES = {"p": ctypes.c_void_p, "l": ctypes.c_int64, "z": ctypes.c_size_t, "i": ctypes.c_int, "f": ctypes.c_float,
          "d": ctypes.c_double, "u": ctypes.c_uint64}


def _declare(handle):
    for name, sig in _SIGNATURES.items():
        if hasattr(handle, name):
            getattr(handle, name).argtypes = [_TYPES[c] for c in sig]


KNOBS = {"igemm_tile": 0, "wgrad_tile": 1, "wgrad_splits": 2, "nms_fused": 3, "stem_kernel": 4, "igemm_persist": 5}     # include/yfs.h: yfs_knob_id


_binding = None


def binding():
    """The extension module with the tensor side of the head operators (csrc/torch_binding.cpp), given the addresses of the
    entry points of the library that is loaded (LIB_PATH)."""
    global _binding
    if _binding is None:
        try:
            from . import _binding as module
        except ImportError as e:
            raise YfsError(f"yolo_from_scratch_amd/_binding.so cannot be loaded ({e}): build it with "
                           f"`make -C {os.path.join(_HERE, 'csrc')}`. There is no CPU fallback.") from e
        if lib().yfs_version() < 301:      # (dropout's p was a float before)
            raise YfsError(f"{LIB_PATH} is version {lib().yfs_version()}, _binding.so calls version 301: build both")
        names = ("yfs_last_error", "yfs_layer_norm_fwd", "yfs_layer_norm_bwd", "yfs_layer_norm_bwd_workspace_bytes",
                 "yfs_dropout_fwd", "yfs_dropout_bwd", "yfs_fp8_matmul", "yfs_fp8_matmul_workspace_bytes", "yfs_fp8_linear_saved_bytes",
                 "yfs_fp8_linear_fwd_workspace_bytes", "yfs_fp8_linear_bwd_workspace_bytes", "yfs_fp8_linear_fwd",
                 "yfs_fp8_linear_bwd")
        module.init({n: ctypes.cast(getattr(lib(), n), ctypes.c_void_p).value for n in names}, YfsError)
        _binding = module
    return _binding


def set_knob(name, value):
    """Measurement aid (include/yfs.h, tuning knobs): force a kernel variant; 0 restores the library's own choice."""
    check(lib().yfs_set_knob(ctypes.c_int(KNOBS[name]), ctypes.c_int(int(value))), "yfs_set_knob")


def get_knob(name):
    return lib().yfs_get_knob(ctypes.c_int(KNOBS[name]))


def last_error():
    buf = ctypes.create_string_buffer(512)
    lib().yfs_last_error(buf, ctypes.c_size_t(512))
    return buf.value.decode("utf-8", "replace")


def last_kernel():
    """Kernel variant the calling thread's last conv entry point launched (include/yfs.h: yfs_last_kernel)."""
    buf = ctypes.create_string_buffer(128)
    lib().yfs_last_kernel(buf, ctypes.c_size_t(128))
    return buf.value.decode("utf-8", "replace")


def check(status, what):
    if status != 0:
        raise YfsError(f"{what} failed with status {status}: {last_error()}")


def ptr(t):
    """Device pointer of a tensor (None -> NULL)."""
    return ctypes.c_void_p(t.data_ptr()) if t is not None else ctypes.c_void_p(0)


def stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}      # include/yfs.h: yfs_dtype


class on_device:
    """Context of a call on the tensors' own device, whichever device is current: gives the raw handle of that device's
    current stream.  The tensors (None allowed) have to be on one GPU."""
    __slots__ = ("index", "before")

    def __init__(self, what, *tensors):
        self.index = -1
        for t in tensors:
            if t is None:
                continue
            index = t.get_device()
            if index < 0:
                require_cuda(t)
            if self.index >= 0 and index != self.index:
                raise YfsError(f"{what}: tensors on devices {self.index} and {index}")
            self.index = index

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.index:
            torch.cuda.set_device(self.index)
        return torch._C._cuda_getCurrentRawStream(self.index)

    def __exit__(self, *exc):
        if self.before != self.index:
            torch.cuda.set_device(self.before)
        return False


def require_cuda(*tensors):
    for t in tensors:
        if t is not None and not t.is_cuda:
            raise YfsError("yolo_from_scratch_amd ops run on the MI355X only: got a CPU tensor "
                           "(there is no CPU fallback; the CPU oracle lives in oracle/ and is test-only)")


i64 = ctypes.c_int64
c_int = ctypes.c_int
c_float = ctypes.c_float
c_size = ctypes.c_size_t
