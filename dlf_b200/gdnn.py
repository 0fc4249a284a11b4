"""Host-side mirror of ``gpgpu::dnn::conv2d`` (gpgpu/include/gdnn.h:201-213) plus the
``Filter2D`` geometry of dlf/include/tensor/dnn.h:9-122 that its callers use.

``conv2d`` keeps the reference's argument order. One argument is added at the end: ``bias``
(``num_kernels`` values), which the reference applies as a separate pass over Y
(``ConvOp::evaluate``, dlf/include/predict.h:1272-1281) and this backend folds into the
convolution's epilogue.
"""
import ctypes
import math
import struct

import torch

from . import lib
from .gblas import (BLASError, StatusCode, _NO_LOCK, _Plans, _caller_scratch, _capturing, _check, _empty, _operator_scratch,
                    _operator_stream, _passing_scratch, _ptr, _stream, _stream_scratch, precision_of)


class Filter2D:
    """Geometry of a 2-D filter: NCHW input, OIHW kernel (dnn.h:9-122)."""

    def __init__(self, input_shape, kernel_shape, group=1, kernel_w=None):
        """Filter2D(input_shape, kernel_shape, group) for convolutions, or
        Filter2D(input_shape, kernel_h, kernel_w) for pooling (dlf/src/tensor/filter.cpp:5-25)."""
        self.batches, self.channels, self.height, self.width = map(int, input_shape)
        if isinstance(kernel_shape, int):
            # pooling form: the second and third arguments are kernel_h, kernel_w
            self.kernel_h = int(kernel_shape)
            self.kernel_w = int(kernel_w if kernel_w is not None else group)
            self.num_kernels, self.group = self.channels, 1
        else:
            self.num_kernels, cpg, self.kernel_h, self.kernel_w = map(int, kernel_shape)
            self.group = int(group)
            if cpg * self.group != self.channels:
                raise ValueError("kernel channels * group != input channels")
        self.pad_top = self.pad_left = self.pad_bottom = self.pad_right = 0
        self.stride_h = self.stride_w = 1
        self.dilation_h = self.dilation_w = 1

    def pads(self, *p):
        if len(p) == 2:
            self.pad_top = self.pad_bottom = int(p[0])
            self.pad_left = self.pad_right = int(p[1])
        else:
            self.pad_top, self.pad_left, self.pad_bottom, self.pad_right = map(int, p)
        return self

    def auto_pad(self, mode):
        """dlf/src/tensor/filter.cpp:51-82."""
        if mode == "VALID":
            self.pad_top = self.pad_left = self.pad_bottom = self.pad_right = 0
        elif mode in ("SAME_UPPER", "SAME_LOWER"):
            def pad(size, kernel, stride, dilation):
                ext = (kernel - 1) * dilation + 1
                total = max(((size - 1) // stride) * stride + ext - size, 0)
                half = total >> 1
                return (half, total - half) if mode == "SAME_UPPER" else (total - half, half)
            self.pad_top, self.pad_bottom = pad(self.height, self.kernel_h, self.stride_h, self.dilation_h)
            self.pad_left, self.pad_right = pad(self.width, self.kernel_w, self.stride_w, self.dilation_w)
        return self

    def strides(self, h, w):
        self.stride_h, self.stride_w = int(h), int(w)
        return self

    def dilations(self, h, w):
        self.dilation_h, self.dilation_w = int(h), int(w)
        return self

    @property
    def output_h(self):  # dnn.h:99-103
        size = self.height + self.pad_top + self.pad_bottom
        ext = self.dilation_h * (self.kernel_h - 1) + 1
        return (size - ext) // self.stride_h + 1 if size >= ext else 1

    @property
    def output_w(self):  # dnn.h:105-109
        size = self.width + self.pad_left + self.pad_right
        ext = self.dilation_w * (self.kernel_w - 1) + 1
        return (size - ext) // self.stride_w + 1 if size >= ext else 1

    def output_shape(self):
        return (self.batches, self.num_kernels, self.output_h, self.output_w)


# Scratch for packed filter banks and channels-last copies, one buffer per (device, stream), grown on demand - the
# role the context's temporary-buffer pool plays in the reference (gpgpu/src/gpgpu.cpp:189-214).
_WORKSPACES = {}


def conv2d(batches, channels, height, width, output_h, output_w, num_kernels, group, kernel_h,
           kernel_w, pad_top, pad_left, pad_bottom, pad_right, stride_h, stride_w, dilation_h,
           dilation_w, im_buffer, kernel_buffer, result_buffer, queue=None, event=None, bias=None,
           residual=None, activation=None):
    """NCHW cross-correlation into result_buffer (gpgpu::dnn::conv2d, gdnn.h:201-213).

    ``bias``, ``residual`` (a tensor shaped like the result, may be the result itself) and
    ``activation`` (None or "relu") fuse what dlf's graph runtime runs as separate passes after
    the convolution: the bias add of ConvOp (dlf/include/predict.h:1272-1281), the Add of a
    residual connection and the Relu that follows it."""
    prec = precision_of(result_buffer)
    if im_buffer.dtype != result_buffer.dtype or kernel_buffer.dtype != result_buffer.dtype:
        raise BLASError(StatusCode.kInvalidValue)
    if bias is not None and bias.dtype != result_buffer.dtype:
        raise BLASError(StatusCode.kInvalidValue)
    if group < 1 or channels % group or num_kernels % group:
        raise BLASError(StatusCode.kInvalidDimension)
    if im_buffer.numel() < batches * channels * height * width:
        raise BLASError(StatusCode.kInsufficientMemoryA)
    if kernel_buffer.numel() < num_kernels * (channels // group) * kernel_h * kernel_w:
        raise BLASError(StatusCode.kInsufficientMemoryB)
    if result_buffer.numel() < batches * num_kernels * output_h * output_w:
        raise BLASError(StatusCode.kInsufficientMemoryC)
    if bias is not None and bias.numel() < num_kernels:
        raise BLASError(StatusCode.kInvalidValue)
    if residual is not None and (residual.dtype != result_buffer.dtype or
                                 residual.numel() < batches * num_kernels * output_h * output_w):
        raise BLASError(StatusCode.kInvalidValue)
    if activation not in (None, "relu"):
        raise BLASError(StatusCode.kInvalidValue)
    s, sp = _stream(queue)
    need = lib().dlf_b200_conv2d_workspace_bytes(
        int(prec), batches, channels, height, width, output_h, output_w, num_kernels, group,
        kernel_h, kernel_w)
    ws, entry = _caller_scratch(result_buffer.device, need), None
    if ws is None and _capturing():
        ws = _passing_scratch(max(need, 256), result_buffer.device, queue)  # (as of a product: never kept scratch in a graph)
    elif ws is None:
        entry = _stream_scratch(_WORKSPACES, result_buffer.device, s.cuda_stream)
    null = ctypes.c_void_p(0)
    with entry.lock if entry is not None else _NO_LOCK:
        if entry is not None:
            ws = entry.at_least(max(need, 256), result_buffer.device, s)
        if event is not None:
            event.start.record(s)
        rc = lib().dlf_b200_conv2d_fused(
            int(prec), batches, channels, height, width, output_h, output_w, num_kernels, group,
            kernel_h, kernel_w, pad_top, pad_left, pad_bottom, pad_right, stride_h, stride_w,
            dilation_h, dilation_w, _ptr(im_buffer), _ptr(kernel_buffer),
            _ptr(bias) if bias is not None else null,
            _ptr(residual) if residual is not None else null, 1 if activation == "relu" else 0,
            _ptr(result_buffer), ctypes.c_void_p(ws.data_ptr()) if ws is not None else null,
            ws.numel() if ws is not None else 0, sp)
        if event is not None:
            event.end.record(s)
    _check(rc)


def conv2d_filter(X, W, Y, filt, bias=None, queue=None, event=None, residual=None, activation=None):
    """dlf::dnn::conv2d(X, W, Y, filter) for device tensors (dlf/include/tensor/dnn_detail.h:154-166)."""
    conv2d(filt.batches, filt.channels, filt.height, filt.width, filt.output_h, filt.output_w,
           filt.num_kernels, filt.group, filt.kernel_h, filt.kernel_w, filt.pad_top,
           filt.pad_left, filt.pad_bottom, filt.pad_right, filt.stride_h, filt.stride_w,
           filt.dilation_h, filt.dilation_w, X, W, Y, queue=queue, event=event, bias=bias,
           residual=residual, activation=activation)


def _pool(fn_name, extra, batches, channels, height, width, output_h, output_w, kernel_h, kernel_w, pad_top,
          pad_left, pad_bottom, pad_right, stride_h, stride_w, dilation_h, dilation_w, x_buffer, y_buffer,
          queue, event):
    prec = precision_of(y_buffer)
    if x_buffer.dtype != y_buffer.dtype:
        raise BLASError(StatusCode.kInvalidValue)
    if x_buffer.numel() < batches * channels * height * width:
        raise BLASError(StatusCode.kInsufficientMemoryA)
    if y_buffer.numel() < batches * channels * output_h * output_w:
        raise BLASError(StatusCode.kInsufficientMemoryC)
    s, sp = _stream(queue)
    if event is not None:
        event.start.record(s)
    rc = getattr(lib(), fn_name)(
        int(prec), batches, channels, height, width, output_h, output_w, kernel_h, kernel_w, pad_top,
        pad_left, pad_bottom, pad_right, stride_h, stride_w, dilation_h, dilation_w, *extra,
        _ptr(x_buffer), _ptr(y_buffer), sp)
    if event is not None:
        event.end.record(s)
    _check(rc)


def maxpool(batches, channels, height, width, output_h, output_w, kernel_h, kernel_w, pad_top, pad_left,
            pad_bottom, pad_right, stride_h, stride_w, dilation_h, dilation_w, x_buffer, y_buffer,
            queue=None, event=None):
    """gpgpu::dnn::maxpool, in the argument order of its definition and of its callers
    (gpgpu/src/gdnn.cpp:1667-1676; dlf/include/tensor/dnn.h:218-229)."""
    _pool("dlf_b200_maxpool", (), batches, channels, height, width, output_h, output_w, kernel_h, kernel_w,
          pad_top, pad_left, pad_bottom, pad_right, stride_h, stride_w, dilation_h, dilation_w, x_buffer,
          y_buffer, queue, event)


def avgpool(batches, channels, height, width, output_h, output_w, kernel_h, kernel_w, pad_top, pad_left,
            pad_bottom, pad_right, stride_h, stride_w, dilation_h, dilation_w, count_include_pad, x_buffer,
            y_buffer, queue=None, event=None):
    """gpgpu::dnn::avgpool (gpgpu/src/gdnn.cpp:1728-1738; dlf/include/tensor/dnn.h:249-261)."""
    _pool("dlf_b200_avgpool", (1 if count_include_pad else 0,), batches, channels, height, width, output_h,
          output_w, kernel_h, kernel_w, pad_top, pad_left, pad_bottom, pad_right, stride_h, stride_w,
          dilation_h, dilation_w, x_buffer, y_buffer, queue, event)


def _filter_args(f):
    return (f.batches, f.channels, f.height, f.width, f.output_h, f.output_w, f.kernel_h, f.kernel_w,
            f.pad_top, f.pad_left, f.pad_bottom, f.pad_right, f.stride_h, f.stride_w, f.dilation_h,
            f.dilation_w)


def max_pooling(X, Y, filt, queue=None, event=None):
    """dlf::dnn::max_pooling(X, Y, filter) for device tensors (dlf/include/tensor/dnn.h:217-229)."""
    maxpool(*_filter_args(filt), X, Y, queue=queue, event=event)


def average_pooling(X, Y, filt, count_include_pad, queue=None, event=None):
    """dlf::dnn::average_pooling(X, Y, filter, count_include_pad) (dnn.h:248-262)."""
    avgpool(*_filter_args(filt), count_include_pad, X, Y, queue=queue, event=event)


def global_max_pooling(X, Y, queue=None, event=None):
    """dlf::dnn::global_max_pooling for device tensors: max_pooling with the whole plane as the
    window (dlf/include/tensor/dnn.h:346-351)."""
    h, w = int(X.shape[2]), int(X.shape[3])
    max_pooling(X, Y, Filter2D(X.shape, h, w).strides(h, w), queue=queue, event=event)


def global_average_pooling(X, Y, queue=None, event=None):
    """dlf::dnn::global_average_pooling for device tensors (dnn.h:361-375)."""
    h, w = int(X.shape[2]), int(X.shape[3])
    average_pooling(X, Y, Filter2D(X.shape, h, w).strides(h, w), False, queue=queue, event=event)


# ---------------------------------------------------------------------------------------------
# Channels-last operators (16-bit, (N, H, W, C) with C a multiple of 8): what an operator-list
# runtime that owns its intermediate tensors uses between its operators. The reference's operators
# are NCHW; these compute the same functions on the permuted tensors.

NHWC, NCHW = 0, 1


def nhwc_supported(filt, dtype, y_layout=NHWC):
    """Whether conv2d_nhwc serves this convolution (the limits of the tensor-map unit's im2col mode;
    the C entry returns kNotImplemented otherwise and launches nothing)."""
    f = filt
    return (dtype in (torch.float16, torch.bfloat16) and f.group == 1 and f.channels % 8 == 0 and
            (y_layout == NCHW or f.num_kernels % 8 == 0) and f.kernel_h <= 16 and f.kernel_w <= 16 and
            f.pad_top < 128 and f.pad_left < 128 and f.stride_h <= 8 and f.stride_w <= 8 and
            f.dilation_h * (f.kernel_h - 1) < 256 and f.dilation_w * (f.kernel_w - 1) < 256 and f.batches < 65536 and
            (f.output_w - 1) * f.stride_w + 1 - f.width - f.pad_left <= 127 and
            (f.output_h - 1) * f.stride_h + 1 - f.height - f.pad_top <= 127)


def pack_filters_nhwc(W, queue=None):
    """OIHW filter bank -> (Cout, KH*KW, Ck), Ck = C rounded up to 64 (zero-filled): the K-major operand
    conv2d_nhwc reads."""
    prec = precision_of(W)
    co, c, kh, kw = (int(d) for d in W.shape)
    n = lib().dlf_b200_nhwc_filter_elems(c, co, kh, kw)
    with torch.cuda.stream(queue) if queue is not None else _NO_LOCK:
        W = W.contiguous()
    out = _empty(n, W.dtype, W.device, queue)
    _, sp = _stream(queue)
    _check(lib().dlf_b200_pack_filters_nhwc(int(prec), c, co, kh, kw, _ptr(W), _ptr(out), sp))
    return out


def nchw_to_nhwc(X, Y=None, queue=None):
    """(N, C, H, W) -> (N, H, W, C') with C' = C rounded up to 8 (the added channels zero)."""
    prec = precision_of(X)
    n, c, h, w = (int(d) for d in X.shape)
    cp = (c + 7) // 8 * 8
    if Y is None:
        Y = _empty((n, h, w, cp), X.dtype, X.device, queue)
    elif Y.numel() < n * h * w * cp or Y.dtype != X.dtype:
        raise BLASError(StatusCode.kInsufficientMemoryC)
    _, sp = _stream(queue)
    _check(lib().dlf_b200_nchw_to_nhwc(int(prec), n, c, h, w, _ptr(X), _ptr(Y), sp))
    return Y


def conv2d_nhwc(X, W_packed, Y, filt, bias=None, residual=None, activation=None, y_layout=NHWC, queue=None):
    """Y = act(conv2d(X, W) + bias + residual) with X (N, H, W, C), the filter bank as
    pack_filters_nhwc writes it, and Y / residual in ``y_layout``. One launch, no scratch."""
    f = filt
    prec = precision_of(Y)
    if X.dtype != Y.dtype or W_packed.dtype != Y.dtype or (bias is not None and bias.dtype != Y.dtype) or \
            (residual is not None and residual.dtype != Y.dtype):
        raise BLASError(StatusCode.kInvalidValue)
    if X.numel() < f.batches * f.channels * f.height * f.width:
        raise BLASError(StatusCode.kInsufficientMemoryA)
    if W_packed.numel() < lib().dlf_b200_nhwc_filter_elems(f.channels, f.num_kernels, f.kernel_h, f.kernel_w):
        raise BLASError(StatusCode.kInsufficientMemoryB)
    n_out = f.batches * f.num_kernels * f.output_h * f.output_w
    if Y.numel() < n_out or (residual is not None and residual.numel() < n_out):
        raise BLASError(StatusCode.kInsufficientMemoryC)
    if activation not in (None, "relu"):
        raise BLASError(StatusCode.kInvalidValue)
    _, sp = _stream(queue)
    null = ctypes.c_void_p(0)
    _check(lib().dlf_b200_conv2d_nhwc(
        int(prec), f.batches, f.channels, f.height, f.width, f.output_h, f.output_w, f.num_kernels, f.kernel_h,
        f.kernel_w, f.pad_top, f.pad_left, f.pad_bottom, f.pad_right, f.stride_h, f.stride_w, f.dilation_h,
        f.dilation_w, _ptr(X), _ptr(W_packed), _ptr(bias) if bias is not None else null,
        _ptr(residual) if residual is not None else null, 1 if activation == "relu" else 0, _ptr(Y), int(y_layout), sp))


def pool_nhwc(X, Y, filt, average=False, count_include_pad=False, queue=None):
    """max / average pooling on (N, H, W, C) tensors; ``filt`` is the pooling Filter2D of the NCHW shape."""
    f = filt
    prec = precision_of(Y)
    if f.dilation_h != 1 or f.dilation_w != 1:
        raise BLASError(StatusCode.kNotImplemented)
    if X.dtype != Y.dtype:
        raise BLASError(StatusCode.kInvalidValue)
    if X.numel() < f.batches * f.channels * f.height * f.width:
        raise BLASError(StatusCode.kInsufficientMemoryA)
    if Y.numel() < f.batches * f.channels * f.output_h * f.output_w:
        raise BLASError(StatusCode.kInsufficientMemoryC)
    _, sp = _stream(queue)
    _check(lib().dlf_b200_pool_nhwc(int(prec), 1 if average else 0, 1 if count_include_pad else 0, f.batches, f.channels,
                                    f.height, f.width, f.output_h, f.output_w, f.kernel_h, f.kernel_w, f.pad_top,
                                    f.pad_left, f.stride_h, f.stride_w, _ptr(X), _ptr(Y), sp))


# ---------------------------------------------------------------------------------------------
# Attention over an encoder's states and over a paged cache (16-bit). The reference leaves its parts to its users: two batched
# products and a softmax between them.

_ATTENTION_WORKSPACES = {}
_MASK_TYPES = (torch.bool, torch.uint8)
# the structures of the C header without their pointers, and the pointers
_ATTENTION_ARGS, _PAGED_ARGS, _APPEND_ARGS = struct.Struct("@if19N"), struct.Struct("@if18N"), struct.Struct("@iN17N")
_SIX_POINTERS, _SEVEN_POINTERS = struct.Struct("@6P"), struct.Struct("@7P")


_ATTENTION_PLANS, _PAGED_PLANS, _APPEND_PLANS = _Plans(), _Plans(), _Plans()


def _head_strides(shape, strides):
    """Strides of a tensor of heads for the library, without the last dimension's; where there is only one, 8 elements stand for
    whatever is written."""
    if strides[-1] != 1 and shape[-1] != 1:
        raise BLASError(StatusCode.kNotImplemented)
    return [s if n > 1 else 8 for n, s in zip(shape[:-1], strides)]


def _typed(tensors, dtype, dims):
    for t in tensors:
        if t.dtype != dtype:
            raise BLASError(StatusCode.kInvalidValue)
        if t.dim() != dims or 0 in t.shape:
            raise BLASError(StatusCode.kInvalidDimension)


def _placed(tensors, device):
    for t in tensors:
        if t.device != device or device.type != "cuda":
            raise BLASError(StatusCode.kInvalidMatrixA)


def _device_ints(t, count, device):
    if t.dtype != torch.int32 or not t.is_contiguous():
        raise BLASError(StatusCode.kInvalidValue)
    if t.numel() != count:
        raise BLASError(StatusCode.kInvalidDimension)
    if t.device != device:
        raise BLASError(StatusCode.kInvalidMatrixA)
    return t.data_ptr()


def _default_scale(scale, size):
    scale = 1.0 / math.sqrt(size) if scale is None else float(scale)
    if not 0.0 < scale * 1.4426950408889634 <= 3.4028234e38:  # (the factor of exp2, in single precision)
        raise BLASError(StatusCode.kInvalidValue)
    return scale


def _attention_call(fn, args, need, device, queue, event):
    """fn(args, [workspace, bytes,] stream) with scratch of `need` bytes (None: fn takes none)."""
    handle = _operator_stream(queue, device)
    ws, entry = _operator_scratch(_ATTENTION_WORKSPACES, need, device, queue, handle) if need else (None, None)
    with entry.lock if entry is not None else _NO_LOCK:
        if entry is not None:
            ws = entry.at_least(need, device, queue)
        if event is not None:
            s = queue if queue is not None else torch.cuda.current_stream()
            event.start.record(s)
        if need is None:
            rc = fn(args, handle)
        else:
            rc = fn(args, ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, handle)
        if event is not None:
            event.end.record(s)
    _check(rc)


def _attention_plan(Q, K, V, Y, scale, key_mask):
    _typed((Q, K, V, Y), Y.dtype, 4)
    b, lq, h, d = Q.shape
    lk, hk = K.shape[1:3]
    if K.shape[0] != b or K.shape[3] != d or V.shape != K.shape or Y.shape != Q.shape or h % hk:
        raise BLASError(StatusCode.kInvalidDimension)
    mask_ld = 0
    if key_mask is not None:
        if key_mask.dtype not in _MASK_TYPES or tuple(key_mask.shape) != (b, lk) or (lk > 1 and key_mask.stride(1) != 1):
            raise BLASError(StatusCode.kInvalidValue)
        mask_ld = key_mask.stride(0) if b > 1 else lk
    strides = [s for t in (Q, K, V, Y) for s in _head_strides(t.shape, t.stride())]
    args = _ATTENTION_ARGS.pack(int(precision_of(Y)), _default_scale(scale, d), b, lq, lk, h, hk, d, *strides, mask_ld)
    _placed((Q, K, V, Y) + (() if key_mask is None else (key_mask,)), Y.device)
    return args, lib().dlf_b200_attention_workspace_bytes(b, lq, lk, h, hk, d), b, Y.device


def attention(Q, K, V, Y, scale=None, key_lengths=None, key_mask=None, queue=None, event=None):
    """Y = softmax(scale * Q K^T) V for each head: the queries Q (batch, queries, heads, size) over the keys K and values V (batch,
    keys, kv_heads, size) of another length, for instance an encoder's states. float16 or bfloat16, size a multiple of 8 up to
    128, heads a multiple of kv_heads (head h reads kv head h // (heads // kv_heads)); ``scale`` is 1 / sqrt(size) if not given.

    ``key_lengths`` (batch, int32) and ``key_mask`` (batch, keys; bool or uint8, 0 = left out) say which keys count; those that do not
    may hold anything. A query with no key gets zeros. Scores, their statistics and all sums have 32 bits; a key's weight is rounded to the
    values' type once where there are many queries, and kept in two parts where there are few (up to 32 with heads of up to 64 values, else 16;
    over up to 128 keys 8). Any strides that are multiples of 8 elements, over 16-byte aligned
    addresses, with a head's values contiguous; Q, K, V and the mask may be shared by the batch (expanded). Y must not overlap the
    inputs."""
    if scale is not None:
        scale = float(scale)  # (its value belongs to the key below, not the object)
    key = (Q.dtype, K.dtype, V.dtype, Y.dtype, Q.device, K.device, V.device, Y.device, Q.shape, K.shape, V.shape, Y.shape, Q.stride(), K.stride(),
           V.stride(), Y.stride(), scale,
           None if key_mask is None else (key_mask.dtype, key_mask.device, key_mask.shape, key_mask.stride()))
    plan = _ATTENTION_PLANS.get(key)
    if plan is None:
        plan = _ATTENTION_PLANS.keep(key, _attention_plan(Q, K, V, Y, scale, key_mask))
    args, need, batch, device = plan
    pointers = _SIX_POINTERS.pack(Q.data_ptr(), K.data_ptr(), V.data_ptr(), Y.data_ptr(),
                                  0 if key_lengths is None else _device_ints(key_lengths, batch, device),
                                  0 if key_mask is None else key_mask.data_ptr())
    _attention_call(lib().dlf_b200_attention, args + pointers, need, device, queue, event)


def _table_plan(K_pages, V_pages, page_table):
    """(strides of the cache's tensors, width and leading dimension of the page table)"""
    if V_pages.shape != K_pages.shape or page_table.dim() != 2 or 0 in page_table.shape:
        raise BLASError(StatusCode.kInvalidDimension)
    n, width = page_table.shape
    if page_table.dtype != torch.int32 or (width > 1 and page_table.stride(1) != 1):
        raise BLASError(StatusCode.kInvalidValue)
    strides = [_head_strides(t.shape, t.stride()) for t in (K_pages, V_pages)]
    return strides, width, page_table.stride(0) if n > 1 else width


def _paged_plan(Q, K_pages, V_pages, page_table, Y, scale):
    _typed((Q, Y), Y.dtype, 3)
    _typed((K_pages, V_pages), Y.dtype, 4)
    b, h, d = Q.shape
    pages, page_size, hk, dk = K_pages.shape
    (ks, vs), width, ld = _table_plan(K_pages, V_pages, page_table)
    if dk != d or Y.shape != Q.shape or page_table.shape[0] != b or h % hk:
        raise BLASError(StatusCode.kInvalidDimension)
    args = _PAGED_ARGS.pack(int(precision_of(Y)), _default_scale(scale, d), b, h, hk, d, pages, page_size, width, ld,
                            *_head_strides(Q.shape, Q.stride()), *ks, *vs, *_head_strides(Y.shape, Y.stride()))
    _placed((Q, K_pages, V_pages, page_table, Y), Y.device)
    return args, lib().dlf_b200_paged_attention_workspace_bytes(b, h, hk, d), b, Y.device


def paged_attention(Q, K_pages, V_pages, page_table, lengths, Y, scale=None, queue=None, event=None):
    """Attention of one new token of every sequence over its paged cache: Q and Y (batch, heads, size), the cache K_pages and
    V_pages (pages, page_size, kv_heads, size; any strides as in ``attention``). Position i of sequence b lies in page
    page_table[b][i // page_size] (int32) at i % page_size; lengths[b] (int32) positions count, the new token's among them if
    ``paged_append`` has put it there. Table entries beyond a sequence's length may be anything."""
    if scale is not None:
        scale = float(scale)  # (its value belongs to the key below, not the object)
    key = (Q.dtype, K_pages.dtype, V_pages.dtype, Y.dtype, page_table.dtype, Q.device, K_pages.device, V_pages.device, Y.device,
           page_table.device, Q.shape, K_pages.shape, V_pages.shape, Y.shape, page_table.shape, Q.stride(), K_pages.stride(), V_pages.stride(),
           Y.stride(), page_table.stride(), scale)
    plan = _PAGED_PLANS.get(key)
    if plan is None:
        plan = _PAGED_PLANS.keep(key, _paged_plan(Q, K_pages, V_pages, page_table, Y, scale))
    args, need, batch, device = plan
    pointers = _SIX_POINTERS.pack(Q.data_ptr(), K_pages.data_ptr(), V_pages.data_ptr(), Y.data_ptr(), page_table.data_ptr(),
                                  _device_ints(lengths, batch, device))
    _attention_call(lib().dlf_b200_paged_attention, args + pointers, need, device, queue, event)


def _append_plan(K, V, K_pages, V_pages, page_table):
    _typed((K, V), K_pages.dtype, 3)
    _typed((K_pages, V_pages), K_pages.dtype, 4)
    pages, page_size, hk, d = K_pages.shape
    (ks, vs), width, ld = _table_plan(K_pages, V_pages, page_table)
    if K.shape != V.shape or tuple(K.shape[1:]) != (hk, d):
        raise BLASError(StatusCode.kInvalidDimension)
    args = _APPEND_ARGS.pack(int(precision_of(K_pages)), K.shape[0], hk, d, page_table.shape[0], pages, page_size, width, ld,
                             *_head_strides(K.shape, K.stride()), *_head_strides(V.shape, V.stride()), *ks, *vs)
    _placed((K, V, K_pages, V_pages, page_table), K_pages.device)
    return args, K.shape[0], K_pages.device


def paged_append(K, V, K_pages, V_pages, page_table, positions, sequences=None, queue=None, event=None):
    """New keys and values K and V (tokens, kv_heads, size) into a paged cache (see ``paged_attention``): token i to position
    positions[i] of sequence sequences[i] (both int32; without ``sequences``, of sequence i). A position below 0 marks a token that is padding and goes
    nowhere. The rest of the cache stays as it is."""
    key = (K.dtype, V.dtype, K_pages.dtype, V_pages.dtype, page_table.dtype, K.device, V.device, K_pages.device, V_pages.device,
           page_table.device, K.shape, V.shape, K_pages.shape, V_pages.shape, page_table.shape, K.stride(), V.stride(), K_pages.stride(),
           V_pages.stride(), page_table.stride())
    plan = _APPEND_PLANS.get(key)
    if plan is None:
        plan = _APPEND_PLANS.keep(key, _append_plan(K, V, K_pages, V_pages, page_table))
    args, tokens, device = plan
    pointers = _SEVEN_POINTERS.pack(K.data_ptr(), V.data_ptr(), K_pages.data_ptr(), V_pages.data_ptr(), page_table.data_ptr(),
                                    _device_ints(positions, tokens, device),
                                    0 if sequences is None else _device_ints(sequences, tokens, device))
    _attention_call(lib().dlf_b200_paged_append, args + pointers, None, device, queue, event)
