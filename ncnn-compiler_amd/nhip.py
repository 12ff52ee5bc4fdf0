"""ctypes binding of libnhip.so, the gfx950 runtime for the ncnn Convolution /
ConvolutionDepthWise / InnerProduct / int8 Convolution hot path.

Every compute call goes through the C ABI declared in include/nhip.h; torch is
used only as the device allocator and for the current HIP stream.  There is
no CPU fallback: if libnhip.so is missing or no GPU is visible, the calls
raise.

Layer objects mirror the reference's ncnn layer parameters
(include/ncnn-mlir/Graph/graph.hpp:73-150) and its lowering semantics
(lib/Conversion/NCNNToTosa/NCNNToTosa.cpp); batches are [N,C,H,W] stacks of the
reference's single-image [C,H,W] blobs.

Behind the layers stand the token operators, for a decoder that reads a
network's features: GroupNorm, Rotary, cross_attention and KvCache8 (float32,
float16 and bfloat16).  The reference lowers ncnn's attention layers for the CPU
(lib/Conversion/NCNNToTosa/NCNNToTosa.cpp:3859-4668); these are calls, not layers
of a graph, and the other three have no counterpart there.
"""
from __future__ import annotations

import ctypes
import functools
import os

import numpy as np

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libnhip.so")

STATUS_NAMES = {
    0: "SUCCESS", 1: "NULL_POINTER", 2: "INVALID_SHAPE",
    3: "CONSTRAINT_VIOLATION", 4: "SHAPE_ARITHMETIC_OVERFLOW",
    5: "OUTPUT_CAPACITY_INSUFFICIENT", 6: "DEVICE_ERROR", 7: "UNSUPPORTED",
}

ALGO_AUTO, ALGO_IMPLICIT_GEMM, ALGO_WINOGRAD = 0, 1, 2
ACT_NONE, ACT_RELU, ACT_SIGMOID = 0, 1, 4
ACT_SILU = 64  # group norm only

# Every symbol include/nhip.h declares (checked by the CPU test suite).
EXPORTS = (
    "nhip_init", "nhip_device_count", "nhip_last_error", "nhip_malloc",
    "nhip_free", "nhip_memcpy_h2d", "nhip_memcpy_d2h", "nhip_memcpy_d2d",
    "nhip_stream_sync", "nhip_reload_settings", "nhip_timer_start", "nhip_timer_stop",
    "nhip_conv_output_shape", "nhip_conv2d_f32_create",
    "nhip_conv2d_workspace_size", "nhip_conv2d_f32_forward", "nhip_conv2d_f32_forward_noalloc",
    "nhip_conv2d_int8_create", "nhip_conv2d_int8_forward",
    "nhip_dwconv2d_f32_create", "nhip_dwconv2d_f32_forward",
    "nhip_dwconv2d_pw_f32_supported", "nhip_dwconv2d_pw_f32_forward",
    "nhip_conv1x1_dw_f32_supported", "nhip_conv1x1_dw_f32_forward",
    "nhip_dwconv2d_int8_create", "nhip_dwconv2d_int8_forward",
    "nhip_conv_destroy", "nhip_innerproduct_f32_create",
    "nhip_innerproduct_int8_create", "nhip_innerproduct_int8_forward",
    "nhip_innerproduct_workspace_size", "nhip_innerproduct_f32_forward",
    "nhip_innerproduct_destroy", "nhip_global_avgpool_innerproduct_f32_workspace_size",
    "nhip_global_avgpool_innerproduct_f32_forward", "nhip_relu_f32", "nhip_relu_i8",
    "nhip_add_f32", "nhip_global_avgpool_f32", "nhip_quantize_f32_i8",
    "nhip_requantize_i32_i8", "nhip_dequantize_i32_f32",
    "nhip_group_norm_create", "nhip_group_norm_workspace_size", "nhip_group_norm_forward", "nhip_norm_destroy",
    "nhip_rotary_create", "nhip_rotary_forward", "nhip_rotary_destroy",
    "nhip_cross_attention_workspace_size", "nhip_cross_attention_forward",
    "nhip_kv8_append", "nhip_kv8_read", "nhip_kv8_attention_workspace_size", "nhip_kv8_attention_forward",
)

# Every symbol include/nhip_graph.h declares.
GRAPH_EXPORTS = (
    "nhip_graph_load", "nhip_graph_describe", "nhip_graph_num_io",
    "nhip_graph_io_info", "nhip_graph_infer_shapes", "nhip_graph_run",
    "nhip_graph_run_host", "nhip_graph_destroy",
)
DTYPE_F32, DTYPE_I8, DTYPE_I32, DTYPE_F16, DTYPE_BF16 = 0, 1, 2, 3, 4
LAYOUT_TOKENS, LAYOUT_BLOBS = 0, 1
_NP_DTYPE = {DTYPE_F32: np.float32, DTYPE_I8: np.int8, DTYPE_I32: np.int32}


class NhipError(RuntimeError):
    def __init__(self, status: int, message: str):
        super().__init__(f"nhip status {status} ({STATUS_NAMES.get(status, '?')}): {message}")
        self.status = status


class ConvDesc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in (
        "input_channels", "num_output", "kernel_w", "kernel_h", "dilation_w",
        "dilation_h", "stride_w", "stride_h", "pad_left", "pad_right",
        "pad_top", "pad_bottom", "bias_term", "int8_scale_term",
        "activation_type", "group", "algorithm")]


class AttentionDesc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in (
        "dtype", "batch", "queries", "keys", "heads", "kv_heads", "head_dim")] + [("scale", ctypes.c_float)]


class Kv8Desc(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k", "v", "k_scale", "v_scale")] + [
        ("pages", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("kv_heads", "head_dim", "block_tokens")]


_lib = None
_settings = 0  # reloads: workspace sizes held from before one are asked for again
_P = ctypes.c_void_p
_Strides = ctypes.c_int64 * 3


def load():
    """Load libnhip.so (raises if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} is not built: run __graft_entry__.build()")
    # torch ships its own libamdhip64.so.7; load it first so that torch and
    # libnhip share that one HIP runtime (same SONAME, resolved once).
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    L = ctypes.CDLL(LIB_PATH)
    i32, i64, u64, f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_uint64, ctypes.c_float
    D = ctypes.POINTER(ConvDesc)
    sig = {
        "nhip_init": [i32],
        "nhip_device_count": [ctypes.POINTER(i32)],
        "nhip_malloc": [ctypes.POINTER(_P), u64],
        "nhip_free": [_P],
        "nhip_memcpy_h2d": [_P, _P, u64, _P],
        "nhip_memcpy_d2h": [_P, _P, u64, _P],
        "nhip_memcpy_d2d": [_P, _P, u64, _P],
        "nhip_stream_sync": [_P],
        "nhip_reload_settings": [],
        "nhip_timer_start": [ctypes.c_char_p],
        "nhip_timer_stop": [ctypes.POINTER(u64), ctypes.POINTER(ctypes.c_double)],
        "nhip_conv_output_shape": [D, i32, i32, ctypes.POINTER(i32), ctypes.POINTER(i32)],
        "nhip_conv2d_f32_create": [D, _P, _P, ctypes.POINTER(_P)],
        "nhip_conv2d_workspace_size": [_P, i32, i32, i32, ctypes.POINTER(u64)],
        "nhip_conv2d_f32_forward": [_P, _P, _P, _P, i32, i32, i32, _P, u64, _P],
        "nhip_conv2d_f32_forward_noalloc": [_P, _P, _P, _P, i32, i32, i32, _P],
        "nhip_conv2d_int8_create": [D, _P, i32, _P, _P, i32, f32, f32, ctypes.POINTER(_P)],
        "nhip_conv2d_int8_forward": [_P, _P, i32, _P, i32, i32, i32, _P, u64, _P],
        "nhip_dwconv2d_f32_create": [D, _P, _P, ctypes.POINTER(_P)],
        "nhip_dwconv2d_f32_forward": [_P, _P, _P, i32, i32, i32, _P],
        "nhip_dwconv2d_pw_f32_supported": [_P, _P, i32, i32, i32, ctypes.POINTER(i32)],
        "nhip_dwconv2d_pw_f32_forward": [_P, _P, _P, _P, _P, i32, i32, i32, _P],
        "nhip_conv1x1_dw_f32_supported": [_P, _P, i32, i32, i32, ctypes.POINTER(i32)],
        "nhip_conv1x1_dw_f32_forward": [_P, _P, _P, _P, i32, i32, i32, _P],
        "nhip_dwconv2d_int8_create": [D, _P, i32, _P, _P, i32, f32, f32, ctypes.POINTER(_P)],
        "nhip_dwconv2d_int8_forward": [_P, _P, i32, _P, i32, i32, i32, _P],
        "nhip_innerproduct_int8_create": [i32, i32, _P, i32, _P, _P, f32, i32, ctypes.POINTER(_P)],
        "nhip_innerproduct_int8_forward": [_P, _P, i32, _P, i32, _P, u64, _P],
        "nhip_conv_destroy": [_P],
        "nhip_innerproduct_f32_create": [i32, i32, _P, _P, i32, ctypes.POINTER(_P)],
        "nhip_innerproduct_workspace_size": [_P, i32, ctypes.POINTER(u64)],
        "nhip_innerproduct_f32_forward": [_P, _P, _P, i32, _P, u64, _P],
        "nhip_innerproduct_destroy": [_P],
        "nhip_global_avgpool_innerproduct_f32_workspace_size": [_P, i32, i32, i32, ctypes.POINTER(u64)],
        "nhip_global_avgpool_innerproduct_f32_forward": [_P, _P, _P, i32, i32, i32, i32, _P, u64, _P],
        "nhip_relu_f32": [_P, _P, i64, _P],
        "nhip_relu_i8": [_P, _P, i64, _P],
        "nhip_add_f32": [_P, _P, _P, i64, i32, _P],
        "nhip_global_avgpool_f32": [_P, _P, i32, i32, i32, i32, _P],
        "nhip_quantize_f32_i8": [_P, _P, i32, i32, i64, _P, i32, _P],
        "nhip_requantize_i32_i8": [_P, _P, i32, i32, i64, _P, i32, _P, i32, _P, i32, i32, _P],
        "nhip_dequantize_i32_f32": [_P, _P, i32, i32, i64, _P, i32, _P, i32, _P],
    }
    A, K8, S, U = (ctypes.POINTER(x) for x in (AttentionDesc, Kv8Desc, i64, u64))
    sig.update({
        "nhip_group_norm_create": [i32, i32, _P, _P, f32, i32, ctypes.POINTER(_P)],
        "nhip_group_norm_workspace_size": [_P, i32, i32, i32, i64, U],
        "nhip_group_norm_forward": [_P, _P, i32, i32, i32, i64, i64, i64, _P, _P, u64, _P],
        "nhip_norm_destroy": [_P],
        "nhip_rotary_create": [i32, i32, _P, _P, i32, ctypes.POINTER(_P)],
        "nhip_rotary_forward": [_P, _P, i32, i32, i32, i32, S, _P, i64, i32, _P, S, _P],
        "nhip_rotary_destroy": [_P],
        "nhip_cross_attention_workspace_size": [A, U],
        "nhip_cross_attention_forward": [A, _P, S, _P, S, _P, S, _P, _P, i64, _P, _P, u64, _P],
        "nhip_kv8_append": [K8, i32, _P, S, _P, S, i32, i32, _P, i64, _P, _P, _P],
        "nhip_kv8_read": [K8, i32, i32, i32, _P, i64, _P, _P, _P, _P],
        "nhip_kv8_attention_workspace_size": [A, K8, U],
        "nhip_kv8_attention_forward": [A, K8, _P, S, _P, i64, _P, i32, _P, _P, u64, _P],
    })
    i64p, i32p, vpp = ctypes.POINTER(i64), ctypes.POINTER(i32), ctypes.POINTER(_P)
    sig.update({
        "nhip_graph_load": [ctypes.c_char_p, u64, _P, u64, i64p, i32, vpp],
        "nhip_graph_describe": [ctypes.c_char_p, u64, _P, u64, i64p, i32, vpp],
        "nhip_graph_num_io": [_P, i32p, i32p],
        "nhip_graph_io_info": [_P, i32, i32, i32p, i64p, i32p, ctypes.POINTER(ctypes.c_char_p)],
        "nhip_graph_infer_shapes": [_P, i64p, i64p, i32p],
        "nhip_graph_run": [_P, i32, i64p, vpp, vpp, _P],
        "nhip_graph_run_host": [_P, i64p, vpp, vpp, ctypes.POINTER(u64)],
        "nhip_graph_destroy": [_P],
    })
    for name, args in sig.items():
        fn = getattr(L, name)
        fn.argtypes = args
        fn.restype = ctypes.c_int
    L.nhip_last_error.argtypes = []
    L.nhip_last_error.restype = ctypes.c_char_p
    _lib = L
    return L


def check(status: int) -> None:
    if status != 0:
        raise NhipError(status, load().nhip_last_error().decode(errors="replace"))


# ---------------------------------------------------------------- device glue
def _torch():
    import torch
    return torch


def init(device: int = 0) -> None:
    check(load().nhip_init(device))


def reload_settings() -> None:
    """Re-read the NHIP_* tuning / test switches from the environment (the
    library reads them once, at first use)."""
    global _settings
    check(load().nhip_reload_settings())
    _settings += 1


def timer_start(kernel_filter: str = "") -> None:
    """Bracket every matching kernel launch with HIP events on its stream."""
    check(load().nhip_timer_start(kernel_filter.encode()))


def timer_stop():
    """-> (launches, total_ms) of the launches timed since timer_start."""
    n, ms = ctypes.c_uint64(), ctypes.c_double()
    check(load().nhip_timer_stop(ctypes.byref(n), ctypes.byref(ms)))
    return n.value, ms.value


def _ptr(t):
    return None if t is None else _P(t.data_ptr())


def _torch_dtype(np_dtype):
    torch = _torch()
    return {np.int8: torch.int8, np.int32: torch.int32}.get(np_dtype, torch.float32)


def _stream(stream=None):
    """The given stream's handle, or the current device's current stream's
    (its handle alone: building torch's Stream object took 3 of a call's 8
    us)."""
    if stream is not None:
        return _P(stream.cuda_stream)
    C = _torch()._C
    return _P(C._cuda_getCurrentRawStream(C._cuda_getDevice()))


def _dev(t, dtype):
    """Device tensor check (no host fallback)."""
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("nhip expects a CUDA (HIP) device tensor")
    if t.dtype != dtype:
        raise TypeError(f"expected {dtype}, got {t.dtype}")
    return t.contiguous()


def _workspace(nbytes: int, device):
    torch = _torch()
    if nbytes == 0:
        return None, 0
    return torch.empty(int(nbytes), dtype=torch.uint8, device=device), int(nbytes)


def conv_desc(c, k, kernel=(3, 3), stride=(1, 1), dilation=(1, 1),
              pad=(1, 1, 1, 1), bias=True, act=ACT_NONE, int8_scale_term=0,
              group=1, algorithm=ALGO_AUTO) -> ConvDesc:
    """kernel/stride/dilation are (h, w); pad is (top, bottom, left, right)."""
    d = ConvDesc()
    d.input_channels, d.num_output = c, k
    d.kernel_h, d.kernel_w = kernel
    d.stride_h, d.stride_w = stride
    d.dilation_h, d.dilation_w = dilation
    d.pad_top, d.pad_bottom, d.pad_left, d.pad_right = pad
    d.bias_term = 1 if bias else 0
    d.int8_scale_term = int8_scale_term
    d.activation_type = act
    d.group = group
    d.algorithm = algorithm
    return d


def output_shape(desc: ConvDesc, h: int, w: int):
    oh, ow = ctypes.c_int32(), ctypes.c_int32()
    check(load().nhip_conv_output_shape(ctypes.byref(desc), h, w, ctypes.byref(oh), ctypes.byref(ow)))
    return oh.value, ow.value


def _np_ptr(a):
    return None if a is None else a.ctypes.data_as(_P)


class _Plan:
    _destroy = "nhip_conv_destroy"

    def __init__(self):
        self.handle = _P()

    def close(self):
        if self.handle:
            getattr(load(), self._destroy)(self.handle)
            self.handle = _P()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass


class Conv2dF32(_Plan):
    """ncnn Convolution, fp32 (reference ConvertConvolution fp32 path)."""

    def __init__(self, desc: ConvDesc, weight, bias=None):
        super().__init__()
        self.desc = desc
        self._w = np.ascontiguousarray(weight, dtype=np.float32)
        self._b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        expect = desc.num_output * desc.input_channels * desc.kernel_h * desc.kernel_w
        if self._w.size != expect:
            raise ValueError(f"weight has {self._w.size} elements, expected {expect}")
        check(load().nhip_conv2d_f32_create(ctypes.byref(desc), _np_ptr(self._w), _np_ptr(self._b),
                                            ctypes.byref(self.handle)))

    def workspace_size(self, n, h, w) -> int:
        b = ctypes.c_uint64()
        check(load().nhip_conv2d_workspace_size(self.handle, n, h, w, ctypes.byref(b)))
        return b.value

    def forward(self, x, residual=None, out=None, workspace=None, stream=None):
        torch = _torch()
        x = _dev(x, torch.float32)
        n, c, h, w = x.shape
        if out is None:
            oh, ow = output_shape(self.desc, h, w)
            out = torch.empty((n, self.desc.num_output, oh, ow), dtype=torch.float32, device=x.device)
        if residual is not None:
            residual = _dev(residual, torch.float32)
        if workspace is None:
            workspace, nbytes = _workspace(self.workspace_size(n, h, w), x.device)
        else:
            nbytes = workspace.numel()
        check(load().nhip_conv2d_f32_forward(self.handle, _ptr(x), _ptr(residual), _ptr(out), n, h, w,
                                             _ptr(workspace), nbytes, _stream(stream)))
        return out


class Conv2dInt8(_Plan):
    """ncnn Convolution with int8_scale_term (reference int8 path)."""

    def __init__(self, desc: ConvDesc, weight, bias, weight_scale, input_scale, output_scale=1.0):
        super().__init__()
        self.desc = desc
        w = np.ascontiguousarray(weight)
        self._w = w if w.dtype == np.int8 else np.ascontiguousarray(w, dtype=np.float32)
        self._b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        self._ws = np.ascontiguousarray(np.atleast_1d(weight_scale), dtype=np.float32)
        check(load().nhip_conv2d_int8_create(
            ctypes.byref(desc), _np_ptr(self._w), 1 if self._w.dtype == np.int8 else 0,
            _np_ptr(self._b), _np_ptr(self._ws), self._ws.size, ctypes.c_float(input_scale),
            ctypes.c_float(output_scale), ctypes.byref(self.handle)))

    def workspace_size(self, n, h, w) -> int:
        b = ctypes.c_uint64()
        check(load().nhip_conv2d_workspace_size(self.handle, n, h, w, ctypes.byref(b)))
        return b.value

    def forward(self, x, out=None, workspace=None, stream=None):
        torch = _torch()
        if not x.is_cuda or x.dtype not in (torch.float32, torch.int8):
            raise TypeError("int8 conv input must be a float32 or int8 device tensor")
        x = x.contiguous()
        n, c, h, w = x.shape
        if out is None:
            oh, ow = output_shape(self.desc, h, w)
            odt = torch.int8 if self.desc.int8_scale_term > 100 else torch.float32
            out = torch.empty((n, self.desc.num_output, oh, ow), dtype=odt, device=x.device)
        if workspace is None:
            workspace, nbytes = _workspace(self.workspace_size(n, h, w), x.device)
        else:
            nbytes = workspace.numel()
        check(load().nhip_conv2d_int8_forward(self.handle, _ptr(x), 1 if x.dtype == torch.int8 else 0,
                                              _ptr(out), n, h, w, _ptr(workspace), nbytes,
                                              _stream(stream)))
        return out


class DwConv2dF32(_Plan):
    """ncnn ConvolutionDepthWise, fp32."""

    def __init__(self, desc: ConvDesc, weight, bias=None):
        super().__init__()
        self.desc = desc
        self._w = np.ascontiguousarray(weight, dtype=np.float32)
        self._b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        check(load().nhip_dwconv2d_f32_create(ctypes.byref(desc), _np_ptr(self._w), _np_ptr(self._b),
                                              ctypes.byref(self.handle)))

    def forward(self, x, out=None, stream=None):
        torch = _torch()
        x = _dev(x, torch.float32)
        n, c, h, w = x.shape
        if out is None:
            oh, ow = output_shape(self.desc, h, w)
            out = torch.empty((n, self.desc.num_output, oh, ow), dtype=torch.float32, device=x.device)
        check(load().nhip_dwconv2d_f32_forward(self.handle, _ptr(x), _ptr(out), n, h, w, _stream(stream)))
        return out


def dwconv_pw_supported(dw: "DwConv2dF32", pw: "Conv2dF32", n: int, h: int, w: int) -> bool:
    """Whether a depthwise plan feeding a 1x1 convolution plan has the fused
    kernel for n images of h x w (nhip_dwconv2d_pw_f32_supported)."""
    sup = ctypes.c_int32()
    check(load().nhip_dwconv2d_pw_f32_supported(dw.handle, pw.handle, n, h, w, ctypes.byref(sup)))
    return bool(sup.value)


def dwconv_pw_forward(dw: "DwConv2dF32", pw: "Conv2dF32", x, residual=None, out=None, stream=None):
    """pw(dw(x)) (+ residual) in one pass without the depthwise output in
    memory (nhip_dwconv2d_pw_f32_forward; the graph executor's fusion)."""
    torch = _torch()
    x = _dev(x, torch.float32)
    n, c, h, w = x.shape
    oh, ow = output_shape(dw.desc, h, w)
    if out is None:
        out = torch.empty((n, pw.desc.num_output, oh, ow), dtype=torch.float32, device=x.device)
    res = None if residual is None else _dev(residual, torch.float32)
    check(load().nhip_dwconv2d_pw_f32_forward(dw.handle, pw.handle, _ptr(x), _ptr(res), _ptr(out), n, h, w,
                                               _stream(stream)))
    return out


def conv1x1_dw_supported(pw: "Conv2dF32", dw: "DwConv2dF32", n: int, h: int, w: int) -> bool:
    """Whether a 1x1 convolution plan feeding a depthwise plan has the fused
    kernel for n images of h x w (nhip_conv1x1_dw_f32_supported)."""
    sup = ctypes.c_int32()
    check(load().nhip_conv1x1_dw_f32_supported(pw.handle, dw.handle, n, h, w, ctypes.byref(sup)))
    return bool(sup.value)


def conv1x1_dw_forward(pw: "Conv2dF32", dw: "DwConv2dF32", x, out=None, stream=None):
    """dw(pw(x)) in one pass without the 1x1 output in memory
    (nhip_conv1x1_dw_f32_forward; the graph executor's fusion)."""
    torch = _torch()
    x = _dev(x, torch.float32)
    n, c, h, w = x.shape
    oh, ow = output_shape(dw.desc, h, w)
    if out is None:
        out = torch.empty((n, dw.desc.num_output, oh, ow), dtype=torch.float32, device=x.device)
    check(load().nhip_conv1x1_dw_f32_forward(pw.handle, dw.handle, _ptr(x), _ptr(out), n, h, w, _stream(stream)))
    return out


class DwConv2dInt8(_Plan):
    """ncnn ConvolutionDepthWise with int8_scale_term."""

    def __init__(self, desc: ConvDesc, weight, bias, weight_scale, input_scale, output_scale=1.0):
        super().__init__()
        self.desc = desc
        w = np.ascontiguousarray(weight)
        self._w = w if w.dtype == np.int8 else np.ascontiguousarray(w, dtype=np.float32)
        self._b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        self._ws = np.ascontiguousarray(np.atleast_1d(weight_scale), dtype=np.float32)
        check(load().nhip_dwconv2d_int8_create(
            ctypes.byref(desc), _np_ptr(self._w), 1 if self._w.dtype == np.int8 else 0, _np_ptr(self._b),
            _np_ptr(self._ws), self._ws.size, ctypes.c_float(input_scale), ctypes.c_float(output_scale),
            ctypes.byref(self.handle)))

    def forward(self, x, out=None, stream=None):
        torch = _torch()
        if not x.is_cuda or x.dtype not in (torch.float32, torch.int8):
            raise TypeError("int8 depthwise input must be a float32 or int8 device tensor")
        x = x.contiguous()
        n, c, h, w = x.shape
        if out is None:
            oh, ow = output_shape(self.desc, h, w)
            odt = torch.int8 if self.desc.int8_scale_term > 100 else torch.float32
            out = torch.empty((n, c, oh, ow), dtype=odt, device=x.device)
        check(load().nhip_dwconv2d_int8_forward(self.handle, _ptr(x), 1 if x.dtype == torch.int8 else 0, _ptr(out),
                                                n, h, w, _stream(stream)))
        return out


class InnerProductInt8(_Plan):
    """ncnn InnerProduct with int8_scale_term (fp32 output)."""
    _destroy = "nhip_innerproduct_destroy"

    def __init__(self, weight, bias, weight_scale, input_scale, activation=ACT_NONE):
        super().__init__()
        w = np.ascontiguousarray(weight)
        self._w = w if w.dtype == np.int8 else np.ascontiguousarray(w, dtype=np.float32)
        self.num_output, self.num_input = self._w.shape
        self._b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        self._ws = np.ascontiguousarray(np.broadcast_to(np.atleast_1d(weight_scale), (self.num_output,)),
                                        dtype=np.float32)
        check(load().nhip_innerproduct_int8_create(
            self.num_output, self.num_input, _np_ptr(self._w), 1 if self._w.dtype == np.int8 else 0,
            _np_ptr(self._b), _np_ptr(self._ws), ctypes.c_float(input_scale), activation,
            ctypes.byref(self.handle)))

    def workspace_size(self, m) -> int:
        b = ctypes.c_uint64()
        check(load().nhip_innerproduct_workspace_size(self.handle, m, ctypes.byref(b)))
        return b.value

    def forward(self, x, out=None, workspace=None, stream=None):
        torch = _torch()
        if not x.is_cuda or x.dtype not in (torch.float32, torch.int8):
            raise TypeError("int8 InnerProduct input must be a float32 or int8 device tensor")
        x = x.contiguous()
        m = x.shape[0]
        if out is None:
            out = torch.empty((m, self.num_output), dtype=torch.float32, device=x.device)
        if workspace is None:
            workspace, nbytes = _workspace(self.workspace_size(m), x.device)
        else:
            nbytes = workspace.numel()
        check(load().nhip_innerproduct_int8_forward(self.handle, _ptr(x), 1 if x.dtype == torch.int8 else 0,
                                                    _ptr(out), m, _ptr(workspace), nbytes, _stream(stream)))
        return out


class InnerProductF32(_Plan):
    """ncnn InnerProduct, fp32 packed matmul."""
    _destroy = "nhip_innerproduct_destroy"

    def __init__(self, weight, bias=None, activation=ACT_NONE):
        super().__init__()
        self._w = np.ascontiguousarray(weight, dtype=np.float32)
        self.num_output, self.num_input = self._w.shape
        self._b = None if bias is None else np.ascontiguousarray(bias, dtype=np.float32)
        check(load().nhip_innerproduct_f32_create(self.num_output, self.num_input, _np_ptr(self._w),
                                                  _np_ptr(self._b), activation, ctypes.byref(self.handle)))

    def workspace_size(self, m) -> int:
        b = ctypes.c_uint64()
        check(load().nhip_innerproduct_workspace_size(self.handle, m, ctypes.byref(b)))
        return b.value

    def forward(self, x, out=None, workspace=None, stream=None):
        torch = _torch()
        x = _dev(x, torch.float32)
        m = x.shape[0]
        if out is None:
            out = torch.empty((m, self.num_output), dtype=torch.float32, device=x.device)
        if workspace is None:
            workspace, nbytes = _workspace(self.workspace_size(m), x.device)
        else:
            nbytes = workspace.numel()
        check(load().nhip_innerproduct_f32_forward(self.handle, _ptr(x), _ptr(out), m, _ptr(workspace),
                                                   nbytes, _stream(stream)))
        return out

    def gap_workspace_size(self, n, h, w) -> int:
        b = ctypes.c_uint64()
        check(load().nhip_global_avgpool_innerproduct_f32_workspace_size(self.handle, n, h, w, ctypes.byref(b)))
        return b.value

    def forward_pooled(self, x, out=None, workspace=None, stream=None):
        """Global average pooling of x [n, C, H, W] fused with this
        InnerProduct (C = num_input) -> [n, num_output]."""
        torch = _torch()
        x = _dev(x, torch.float32)
        n, c, h, w = x.shape
        if out is None:
            out = torch.empty((n, self.num_output), dtype=torch.float32, device=x.device)
        if workspace is None:
            workspace, nbytes = _workspace(self.gap_workspace_size(n, h, w), x.device)
        else:
            nbytes = workspace.numel()
        check(load().nhip_global_avgpool_innerproduct_f32_forward(self.handle, _ptr(x), _ptr(out), n, c, h, w,
                                                                  _ptr(workspace), nbytes, _stream(stream)))
        return out


# ---------------------------------------------------------------- elementwise
def relu(x, out=None, stream=None):
    torch = _torch()
    if out is None:
        out = torch.empty_like(x)
    if x.dtype == torch.int8:
        check(load().nhip_relu_i8(_ptr(x), _ptr(out), x.numel(), _stream(stream)))
    else:
        x = _dev(x, torch.float32)
        check(load().nhip_relu_f32(_ptr(x), _ptr(out), x.numel(), _stream(stream)))
    return out


def add(a, b, relu_after=False, out=None, stream=None):
    torch = _torch()
    a, b = _dev(a, torch.float32), _dev(b, torch.float32)
    if a.shape != b.shape:
        raise ValueError("add: shapes differ")
    if out is None:
        out = torch.empty_like(a)
    check(load().nhip_add_f32(_ptr(a), _ptr(b), _ptr(out), a.numel(), 1 if relu_after else 0, _stream(stream)))
    return out


def global_avgpool(x, stream=None):
    torch = _torch()
    x = _dev(x, torch.float32)
    n, c, h, w = x.shape
    out = torch.empty((n, c), dtype=torch.float32, device=x.device)
    check(load().nhip_global_avgpool_f32(_ptr(x), _ptr(out), n, c, h, w, _stream(stream)))
    return out


def _params(device, stream, *values):
    """fp32 device arrays of per-channel (or single) parameters; None stays
    None.  On the current stream they go up in one asynchronous copy from
    pinned memory (torch's host allocator keeps that until the copy is done),
    so the call does not wait for the work queued before it as a copy from
    pageable memory does; on another stream or device, or inside a capture,
    each goes up synchronously."""
    torch = _torch()
    arrays = [None if v is None else np.atleast_1d(np.asarray(v, np.float32)) for v in values]
    if stream is not None or device.index != torch._C._cuda_getDevice() or torch.cuda.is_current_stream_capturing():
        return [None if a is None else torch.as_tensor(a, device=device) for a in arrays]
    host = torch.empty(sum(a.size for a in arrays if a is not None), dtype=torch.float32, pin_memory=True)
    flat, at, spans = host.numpy(), 0, []
    for a in arrays:
        size = 0 if a is None else a.size
        flat[at:at + size] = 0 if a is None else a.ravel()
        spans.append(None if a is None else (at, at + size))
        at += size
    dev = host.to(device, non_blocking=True)
    return [None if sp is None else dev[sp[0]:sp[1]] for sp in spans]


def quantize(x, scale, stream=None):
    """x [N,C,...] fp32 -> int8; scale: 1 or C values (per channel dim 1)."""
    torch = _torch()
    x = _dev(x, torch.float32)
    n, c = x.shape[0], x.shape[1]
    plane = x[0, 0].numel()
    s, = _params(x.device, stream, scale)
    out = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    check(load().nhip_quantize_f32_i8(_ptr(x), _ptr(out), n, c, plane, _ptr(s), s.numel(), _stream(stream)))
    return out


def requantize(x, in_scale, out_scale, bias=None, activation=ACT_NONE, stream=None):
    torch = _torch()
    x = _dev(x, torch.int32)
    n, c = x.shape[0], x.shape[1]
    plane = x[0, 0].numel()
    isc, osc, b = _params(x.device, stream, in_scale, out_scale, bias)
    out = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    check(load().nhip_requantize_i32_i8(_ptr(x), _ptr(out), n, c, plane, _ptr(isc), isc.numel(), _ptr(osc),
                                        osc.numel(), _ptr(b), 0 if b is None else b.numel(), activation,
                                        _stream(stream)))
    return out


def dequantize(x, scale, bias=None, stream=None):
    torch = _torch()
    x = _dev(x, torch.int32)
    n, c = x.shape[0], x.shape[1]
    plane = x[0, 0].numel()
    s, b = _params(x.device, stream, scale, bias)
    out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    check(load().nhip_dequantize_i32_f32(_ptr(x), _ptr(out), n, c, plane, _ptr(s), s.numel(), _ptr(b),
                                         0 if b is None else b.numel(), _stream(stream)))
    return out


# ------------------------------------------------------------ token operators
# Small calls are bound by the host: what torch gives for good is kept, and the
# checks are the cheap forms of themselves.
# stream: the caller has it wait for the inputs and keeps those until it is done;
# new results are of its memory, and may be read by the stream that was current
# at the call once that one waits for it.
_ELEM = {}  # element types, filled with the first call, as are the next
_int32 = _current_device = _current_stream = _empty_like = None


def _begin():
    global _int32, _current_device, _current_stream, _empty_like
    torch = _torch()
    _int32, _empty_like = torch.int32, torch.empty_like
    _current_device, _current_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
    _ELEM.update({torch.float32: DTYPE_F32, torch.float16: DTYPE_F16, torch.bfloat16: DTYPE_BF16})


def _elem(t, *like):
    """(element type code, device index) of a device tensor whose channels
    are contiguous; `like`: tensors that have to have its type and device."""
    if not _ELEM:
        _begin()
    dev, dtype = t.get_device(), t.dtype
    if dev < 0:
        raise TypeError("nhip expects a CUDA (HIP) device tensor")
    code = _ELEM.get(dtype)
    if code is None:
        raise TypeError(f"expected float32, float16 or bfloat16, got {dtype}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError("channels have to be contiguous")
    for x in like:
        if x.dtype != dtype or x.get_device() != dev:
            raise TypeError(f"expected {dtype} on {t.device}, got {x.dtype} on {x.device}")
        if x.stride(-1) != 1 and x.shape[-1] > 1:
            raise ValueError("channels have to be contiguous")
    if dev != _current_device():
        raise ValueError(f"{t.device} is not the current device")
    return code, dev


def _ints(t, dev, shape, what):
    """Pointer of a contiguous int32 tensor of that shape on device `dev`."""
    if t.shape != shape or t.dtype != _int32 or t.get_device() != dev or not t.is_contiguous():
        raise ValueError(f"{what} has to be a contiguous int32 tensor of shape {tuple(shape)} on device {dev}")
    return t.data_ptr()


def _new(like, shape, dtype, stream):
    """A new tensor that `stream` may write at once: of that stream's own
    memory, since what the current one has freed its kernels may still use."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with _torch().cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _output(out, like, shape, stream, dtype=None):
    """`out`, checked, or a new tensor that `stream` may write and the current
    one read."""
    if out is None:
        if stream is not None:
            out = _new(like, shape, dtype, stream)
            out.record_stream(_torch().cuda.current_stream(like.device))
        elif dtype is None and like.is_contiguous() and shape == like.shape:
            out = _empty_like(like)  # the cheapest of torch's allocations
        else:
            out = _new(like, shape, dtype, None)
    elif out.dtype != (dtype or like.dtype) or out.device != like.device or not out.is_contiguous() or out.shape != shape:
        raise ValueError(f"out has to be a contiguous {dtype or like.dtype} tensor of shape {tuple(shape)} on {like.device}")
    return out


def _scratch(workspace, nbytes, like, stream):
    """(tensor, pointer, bytes) of the caller's workspace or a new one, which
    stays allocated until the stream is done with it."""
    if workspace is None:
        if not nbytes:
            return None, None, 0
        workspace = _new(like, nbytes, _torch().uint8, stream)
    elif workspace.device != like.device or not workspace.is_contiguous():
        raise ValueError(f"workspace has to be a contiguous tensor on {like.device}")
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def _on(stream, dev):
    """Handle of the given stream or of the device's current one."""
    return _current_stream(dev) if stream is None else stream.cuda_stream


@functools.lru_cache(4096)
def _strides(strides):
    """The first three of four."""
    return _Strides(*strides[:3])


class GroupNorm(_Plan):
    """Group norm with an activation (ACT_NONE, ACT_RELU, ACT_SILU), channels
    last.  gamma, beta: [channels] or both None."""
    _destroy = "nhip_norm_destroy"

    def __init__(self, groups, channels, gamma=None, beta=None, eps=1e-5, act=ACT_NONE, blobs=False):
        super().__init__()
        self.channels, self.layout = channels, LAYOUT_BLOBS if blobs else LAYOUT_TOKENS
        self._g, self._b = (None if v is None else np.ascontiguousarray(v, dtype=np.float32) for v in (gamma, beta))
        for v in (self._g, self._b):
            if v is not None and v.shape != (channels,):
                raise ValueError(f"gamma and beta have to have {channels} elements")
        check(load().nhip_group_norm_create(channels, groups, _np_ptr(self._g), _np_ptr(self._b), eps, act,
                                            ctypes.byref(self.handle)))
        self._sizes = {}

    def workspace_size(self, dtype_code, n, pixels) -> int:
        key = (_settings, dtype_code, n, pixels)
        if key not in self._sizes:
            b = ctypes.c_uint64()
            check(load().nhip_group_norm_workspace_size(self.handle, dtype_code, self.layout, n, pixels, ctypes.byref(b)))
            if len(self._sizes) > 4096:
                self._sizes.clear()
            self._sizes[key] = b.value
        return self._sizes[key]

    def forward(self, x, out=None, workspace=None, stream=None):
        """x [n, pixels, channels] (any image and pixel strides) or
        [n, h, w, channels] -> the same shape; with blobs=True x
        [n, channels, h, w] or [n, channels, pixels] -> [n, pixels, channels]."""
        shape = x.shape
        if len(shape) == 4 and x.is_contiguous():  # without the view: 0.6 us of a small call's 8
            n, a, b, row = shape
            rows, row = (a, b * row) if self.layout == LAYOUT_BLOBS else (a * b, row)
            image, line = rows * row, row
        else:
            if len(shape) == 4:
                x = x.view(shape[0], shape[1], -1) if self.layout == LAYOUT_BLOBS else x.view(shape[0], -1, shape[3])
            n, rows, row = x.shape
            image, line, _ = x.stride()
            if rows == 1:
                line = max(line, row)
        if self.layout == LAYOUT_BLOBS:
            pixels, c = row, rows
            shape = (n, pixels, c)
        else:
            pixels, c = rows, row
        code, dev = _elem(x)
        if c != self.channels:
            raise ValueError(f"x has {c} channels, expected {self.channels}")
        out = _output(out, x, shape, stream)
        ws, ptr, nbytes = _scratch(workspace, self.workspace_size(code, n, pixels), x, stream)
        check(load().nhip_group_norm_forward(self.handle, x.data_ptr(), code, self.layout, n, pixels, image, line,
                                             out.data_ptr(), ptr, nbytes, _on(stream, dev)))
        return out


class Rotary(_Plan):
    """Rotary positions over the axes that `sections` counts pairs for.
    inv_freq: [sum(sections)]; default theta^(-i / sections[a]) for pair i of
    axis a.  neighbours: pairs (2i, 2i + 1) instead of (i, i + pairs)."""
    _destroy = "nhip_rotary_destroy"

    def __init__(self, head_dim, sections, inv_freq=None, theta=10000.0, neighbours=False):
        super().__init__()
        self.head_dim, self.axes = head_dim, len(sections)
        if inv_freq is None:
            inv_freq = [float(theta) ** (-i / s) for s in sections for i in range(s)]
        sec = np.ascontiguousarray(sections, dtype=np.int32)
        freq = np.ascontiguousarray(inv_freq, dtype=np.float32)
        if freq.shape != (int(sec.sum()),):
            raise ValueError(f"inv_freq has shape {freq.shape}, expected ({int(sec.sum())},)")
        check(load().nhip_rotary_create(head_dim, self.axes, _np_ptr(sec), _np_ptr(freq), 1 if neighbours else 0,
                                        ctypes.byref(self.handle)))

    def forward(self, x, positions, inverse=False, out=None, stream=None):
        """x [batch, tokens, heads, head_dim] (any strides of the first
        three), positions int32 [batch or 1, tokens, axes]; out may be x."""
        b, n, h, d = x.shape
        if d != self.head_dim:
            raise ValueError(f"x has {d} channels to a head, expected {self.head_dim}")
        code, dev = _elem(x)
        per = positions.shape[0]
        if per not in (1, b):
            raise ValueError("positions have to have the batch's size or 1")
        pos = _ints(positions, dev, (per, n, self.axes), "positions")
        if out is None:
            out = _output(None, x, x.shape, stream)
        elif out.shape != x.shape:
            raise ValueError(f"out has to have shape {tuple(x.shape)}")
        else:
            _elem(x, out)
        check(load().nhip_rotary_forward(self.handle, x.data_ptr(), code, b, n, h, _strides(x.stride()), pos,
                                         n * self.axes if per > 1 else 0, 1 if inverse else 0, out.data_ptr(),
                                         _strides(out.stride()), _on(stream, dev)))
        return out


@functools.lru_cache(4096)
def _attention(settings, code, b, lq, lk, h, hkv, d, scale, cached=False):
    """(descriptor, workspace bytes)."""
    desc = AttentionDesc(code, b, lq, lk, h, hkv, d, float(d) ** -0.5 if scale is None else float(scale))
    n = ctypes.c_uint64()
    if cached:  # the size goes by the descriptor alone
        check(load().nhip_kv8_attention_workspace_size(ctypes.byref(desc), ctypes.byref(Kv8Desc()), ctypes.byref(n)))
    else:
        check(load().nhip_cross_attention_workspace_size(ctypes.byref(desc), ctypes.byref(n)))
    return desc, n.value


def cross_attention(q, k, v, key_lengths=None, key_mask=None, scale=None, out=None, workspace=None, stream=None):
    """softmax(scale * q k^T) v: q [batch, queries, heads, d], k and v
    [batch, keys, kv_heads, d] (any strides of the first three).  key_lengths:
    int32 [batch]; key_mask: bool [batch, keys] or [keys], True where a key
    counts.  A row that sees no key is 0.  scale: default d ** -0.5."""
    torch = _torch()
    b, lq, h, d = q.shape
    lk, hkv = k.shape[1], k.shape[2]
    code, dev = _elem(q, k, v)
    if k.shape != (b, lk, hkv, d) or v.shape != k.shape:
        raise ValueError(f"k and v have shapes {tuple(k.shape)} and {tuple(v.shape)}: expected [{b}, keys, kv_heads, {d}]")
    desc, need = _attention(_settings, code, b, lq, lk, h, hkv, d, scale)
    lengths = None if key_lengths is None else _ints(key_lengths, dev, (b,), "key_lengths")
    mask, mask_stride = None, 0
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.device != q.device or tuple(key_mask.shape) not in ((b, lk), (lk,)):
            raise ValueError(f"key_mask has to be a bool tensor of shape {(b, lk)} or {(lk,)} on {q.device}")
        if lk > 1 and key_mask.stride(-1) != 1:
            raise ValueError("key_mask's keys have to be contiguous")
        mask, mask_stride = key_mask.data_ptr(), key_mask.stride(0) if key_mask.dim() == 2 else 0
    out = _output(out, q, q.shape, stream)
    ws, ptr, nbytes = _scratch(workspace, need, q, stream)
    check(load().nhip_cross_attention_forward(desc, q.data_ptr(), _strides(q.stride()), k.data_ptr(),
                                              _strides(k.stride()), v.data_ptr(), _strides(v.stride()),
                                              lengths, mask, mask_stride, out.data_ptr(), ptr, nbytes, _on(stream, dev)))
    return out


class KvCache8:
    """Keys and values in 8 bits, in pages of block_tokens tokens with a scale
    for each page and head (include/nhip.h: nhip_kv8_cache).  Which pages a
    sequence has is the caller's: block tables are int32 [batch, pages of a
    sequence]."""

    def __init__(self, pages, kv_heads, head_dim, block_tokens=64, device="cuda"):
        torch = _torch()
        shape = (pages, kv_heads, block_tokens, head_dim)
        self._hold(torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape, dtype=torch.int8, device=device),
                   torch.zeros(shape[:2], dtype=torch.float32, device=device),
                   torch.zeros(shape[:2], dtype=torch.float32, device=device))

    @classmethod
    def of(cls, k, v, k_scale, v_scale):
        """A cache in the caller's tensors: int8 [pages, kv_heads,
        block_tokens, head_dim] and float32 [pages, kv_heads]."""
        self = cls.__new__(cls)
        self._hold(k, v, k_scale, v_scale)
        return self

    def _hold(self, k, v, k_scale, v_scale):
        torch = _torch()
        if not _ELEM:
            _begin()
        for t, dtype, shape in ((k, torch.int8, k.shape), (v, torch.int8, k.shape),
                                (k_scale, torch.float32, k.shape[:2]), (v_scale, torch.float32, k.shape[:2])):
            if not t.is_cuda or t.dtype != dtype or t.shape != shape or t.device != k.device or not t.is_contiguous():
                raise ValueError(f"expected a contiguous {dtype} tensor of shape {tuple(shape)} on {k.device}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self._dev = k.get_device()
        pages, self.kv_heads, self.block_tokens, self.head_dim = k.shape
        self._desc = Kv8Desc(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages,
                             self.kv_heads, self.head_dim, self.block_tokens)

    def append(self, k, v, block_table, starts, counts=None, stream=None):
        """Tokens starts[b] .. of each sequence from k and v [batch, tokens,
        kv_heads, head_dim]: all of them, or the first counts[b]."""
        b, n = k.shape[:2]
        code, dev = _elem(k, v)
        if k.shape != (b, n, self.kv_heads, self.head_dim) or v.shape != k.shape or dev != self._dev:
            raise ValueError(f"k and v have to have shape [batch, tokens, {self.kv_heads}, {self.head_dim}] on {self.k.device}")
        pages = block_table.shape[-1]
        check(load().nhip_kv8_append(self._desc, code, k.data_ptr(), _strides(k.stride()), v.data_ptr(),
                                     _strides(v.stride()), b, n,
                                     _ints(block_table, dev, (b, pages), "block_table"), pages,
                                     _ints(starts, dev, (b,), "starts"),
                                     None if counts is None else _ints(counts, dev, (b,), "counts"),
                                     _on(stream, dev)))

    def read(self, block_table, starts, tokens, dtype, out=None, stream=None):
        """Values of tokens starts[b] .. starts[b] + tokens - 1: (k, v), each
        [batch, tokens, kv_heads, head_dim]."""
        b, pages = block_table.shape
        shape = (b, tokens, self.kv_heads, self.head_dim)
        k, v = out or (None, None)
        k = _output(k, self.k, shape, stream, dtype)
        code, dev = _elem(k)
        v = _output(v, k, shape, stream)
        check(load().nhip_kv8_read(self._desc, code, b, tokens, _ints(block_table, dev, (b, pages), "block_table"), pages,
                                   _ints(starts, dev, (b,), "starts"), k.data_ptr(), v.data_ptr(), _on(stream, dev)))
        return k, v

    def attention(self, q, block_table, lengths, max_length=None, causal=False, scale=None, out=None, workspace=None,
                  stream=None):
        """Attention of q [batch, queries, heads, head_dim] to the first
        lengths[b] cached tokens (at most max_length; default what the block
        table holds).  causal: the queries are the last tokens."""
        b, lq, h, d = q.shape
        code, dev = _elem(q)
        if d != self.head_dim or dev != self._dev:
            raise ValueError(f"q has to have {self.head_dim} channels to a head, on {self.k.device}")
        pages = block_table.shape[-1]
        if max_length is None:
            max_length = pages * self.block_tokens
        desc, need = _attention(_settings, code, b, lq, max_length, h, self.kv_heads, d, scale, True)
        out = _output(out, q, q.shape, stream)
        ws, ptr, nbytes = _scratch(workspace, need, q, stream)
        check(load().nhip_kv8_attention_forward(desc, self._desc, q.data_ptr(), _strides(q.stride()),
                                                _ints(block_table, dev, (b, pages), "block_table"), pages,
                                                _ints(lengths, dev, (b,), "lengths"), 1 if causal else 0,
                                                out.data_ptr(), ptr, nbytes, _on(stream, dev)))
        return out



class Graph:
    """An ncnn model (.param text + .bin payload) lowered onto libnhip
    (include/nhip_graph.h), the device counterpart of the reference's
    compiled model: Graph::load (lib/Graph/graph.cpp:2129-2333) + the
    generated entry (tools/ncnn-compile.cpp:915-932).

    input_shapes: None, or one CHW triple per Input layer (-1 = given at run
    time, the reference's "?" of --input-shape).  describe_only=True parses,
    validates and lowers without any device work (what a compiler on a host
    without a GPU needs); running such a graph is a constraint violation.
    """

    def __init__(self, param_text, bin_bytes=b"", input_shapes=None, describe_only=False):
        L = load()
        param = param_text.encode() if isinstance(param_text, str) else bytes(param_text)
        self._bin = bytes(bin_bytes)
        arr, count = None, 0
        if input_shapes is not None:
            flat = [int(v) for s in input_shapes for v in s]
            arr = (ctypes.c_int64 * max(len(flat), 1))(*flat)
            count = len(input_shapes)
        self.handle = _P()
        fn = L.nhip_graph_describe if describe_only else L.nhip_graph_load
        check(fn(param, len(param), self._bin or None, len(self._bin), arr, count, ctypes.byref(self.handle)))
        ni, no = ctypes.c_int32(), ctypes.c_int32()
        check(L.nhip_graph_num_io(self.handle, ctypes.byref(ni), ctypes.byref(no)))
        self.inputs = [self._io(0, i) for i in range(ni.value)]
        self.outputs = [self._io(1, i) for i in range(no.value)]

    def _io(self, is_output, index):
        rank, dtype, name = ctypes.c_int32(), ctypes.c_int32(), ctypes.c_char_p()
        dims = (ctypes.c_int64 * 4)()
        check(load().nhip_graph_io_info(self.handle, is_output, index, ctypes.byref(rank), dims,
                                        ctypes.byref(dtype), ctypes.byref(name)))
        return dict(name=name.value.decode(), shape=tuple(dims[:rank.value]),
                    dtype=_NP_DTYPE[dtype.value])

    @staticmethod
    def _shape_arg(shapes):
        if shapes is None:
            return None
        flat = [int(v) for s in shapes for v in s]
        return (ctypes.c_int64 * len(flat))(*flat)

    def infer_shapes(self, input_shapes=None):
        """-> list of output shapes for concrete CHW input shapes."""
        n = len(self.outputs)
        out = (ctypes.c_int64 * (4 * n))()
        ranks = (ctypes.c_int32 * n)()
        check(load().nhip_graph_infer_shapes(self.handle, self._shape_arg(input_shapes), out, ranks))
        return [tuple(out[4 * j:4 * j + ranks[j]]) for j in range(n)]

    def run_host(self, *arrays, capacity=None):
        """The reference entry semantics: one image per input (host numpy
        arrays), returns the list of outputs as numpy arrays."""
        xs = [np.ascontiguousarray(a, dtype=io["dtype"]) for a, io in zip(arrays, self.inputs)]
        if len(xs) != len(self.inputs):
            raise ValueError(f"expected {len(self.inputs)} inputs")
        shapes = [a.shape if a.ndim == 3 else (1,) * (3 - a.ndim) + a.shape for a in xs]
        dyn = any(d < 0 for io in self.inputs for d in io["shape"])
        arg = self._shape_arg(shapes) if dyn else None
        oshapes = self.infer_shapes(shapes if dyn else None)
        outs = [np.empty(s, io["dtype"]) for s, io in zip(oshapes, self.outputs)]
        ins = (_P * len(xs))(*[a.ctypes.data for a in xs])
        ops = (_P * len(outs))(*[o.ctypes.data for o in outs])
        cap = None
        if capacity is not None:
            cap = (ctypes.c_uint64 * len(outs))(*capacity)
        check(load().nhip_graph_run_host(self.handle, arg, ins, ops, cap))
        return outs

    def run(self, *tensors, stream=None, out=None):
        """Batch execution: each input a [N, ...] device tensor of N blobs;
        returns device tensors [N, ...] per output (written into `out`, a
        list of preallocated tensors, when given).  On a non-default stream,
        repeated calls with the same inputs and outputs replay a recorded
        hipGraph of the call plan (nhip_graph_run), so steady loops should
        pass `out`."""
        torch = _torch()
        if len(tensors) != len(self.inputs):
            raise ValueError(f"expected {len(self.inputs)} inputs")
        n = int(tensors[0].shape[0])
        xs = [_dev(t, _torch_dtype(io["dtype"]))
              for t, io in zip(tensors, self.inputs)]
        shapes = [tuple(t.shape[1:]) if t.dim() == 4 else (1,) * (4 - t.dim()) + tuple(t.shape[1:])
                  for t in xs]
        dyn = any(d < 0 for io in self.inputs for d in io["shape"])
        oshapes = self.infer_shapes(shapes if dyn else None)
        if out is None:
            outs = [torch.empty((n,) + s, dtype=_torch_dtype(io["dtype"]),
                                device=xs[0].device) for s, io in zip(oshapes, self.outputs)]
        else:
            outs = list(out)
            for o, s, io in zip(outs, oshapes, self.outputs):
                want = _torch_dtype(io["dtype"])
                if tuple(o.shape) != (n,) + tuple(s) or o.dtype != want or not o.is_contiguous() or not o.is_cuda:
                    raise ValueError(f"out tensor must be a contiguous {want} device tensor of shape {(n,) + tuple(s)}")
        ins = (_P * len(xs))(*[t.data_ptr() for t in xs])
        ops = (_P * len(outs))(*[o.data_ptr() for o in outs])
        check(load().nhip_graph_run(self.handle, n, self._shape_arg(shapes) if dyn else None, ins, ops,
                                    _stream(stream)))
        return outs

    def close(self):
        if self.handle:
            load().nhip_graph_destroy(self.handle)
            self.handle = _P()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass
