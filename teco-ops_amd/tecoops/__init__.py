"""tecoops — PyTorch-ROCm front end of the MI355X operator library.

Mirrors the reference package api/tecoops/__init__.py:3-5 and the wrappers of
api/tecoops/../torch_ext.cpp:61-206: the same function names, positional
arguments and in-place semantics (outputs are caller-allocated tensors; the
functions return None), with device='cuda' in place of 'sdaa'.  Every call
goes through the C ABI of libtecoops.so on the current torch stream; there is
no CPU fallback.

Differences from the reference wrappers, all toward its documented intent:
  * each call binds torch.cuda.current_stream() (the reference never calls
    tecoopsSetStream and runs on the null stream, torch_ext.cpp:35-42);
  * flash_attn_varlen_func passes cu_seqlens_q to the device instead of copying
    it to the host (torch_ext.cpp:119-126), honours softmax_scale and causal,
    and takes the element type (fp16 or bf16) from q;
  * causal_conv1d_fn_torch reads the [dim, tokens] layout in place instead of
    transposing x and out (torch_ext.cpp:186-205).
"""
import ctypes
import math
import os
import sys
import threading

import torch

from . import _lib
from ._lib import TecoopsError  # noqa: F401

# TORCH_LIBRARY(tecoops) registrations (libtecoops_torch.so): the same ops as
# torch.ops.tecoops.*, with torch schemas and the current-stream binding done
# in C++.  Loaded when built; the Python functions below call the C ABI
# directly and do not depend on it.
_TORCH_LIB = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libtecoops_torch.so")
ops = None
if os.path.exists(_TORCH_LIB):
    torch.ops.load_library(_TORCH_LIB)
    ops = torch.ops.tecoops

__all__ = [
    "flatten_rays", "morton3D_invert", "reshape_and_cache", "rms_norm",
    "flash_attn_varlen_func", "causal_conv1d_fn_torch",
    # extensions
    "rotary_embedding", "rotary_reshape_and_cache", "gemv", "gemv_int8", "causal_conv1d",
    "memset", "linear", "moe_layer", "rotary_embedding_axes", "rotary_axes_reshape_and_cache",
    "qk_norm_rotary", "qk_norm_rotary_reshape_and_cache", "reshape_and_cache_int4",
    "flash_attn_varlen_int4", "gemv_int4", "ops",
]

_tls = threading.local()   # per thread: {device index: _Handle}
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


class _Handle:
    """One tecoops handle of one (thread, device), bound to that thread's
    current torch stream of the device.  Threads never share a handle, so a
    thread cannot enqueue on another thread's stream, and the handle orders
    its split-KV scratch across the streams it is used on."""

    def __init__(self):
        self.h = ctypes.c_void_p()
        _lib.call("tecoopsCreate", ctypes.byref(self.h))
        self.stream = None

    def __del__(self):
        # the thread ended: its handle (and scratch) go with it
        try:
            if self.h and not sys.is_finalizing():
                _lib.lib().tecoopsDestroy(self.h)
        except Exception:
            pass


def _handle(device):
    """The calling thread's handle for `device`, bound to the thread's current
    torch stream there (rebound only when that stream changes)."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    handles = getattr(_tls, "handles", None)
    if handles is None:
        handles = _tls.handles = {}
    entry = handles.get(idx)
    if entry is None:
        entry = handles[idx] = _Handle()
    stream = _raw_stream(idx) if _raw_stream else torch.cuda.current_stream(idx).cuda_stream
    if stream != entry.stream:
        _lib.call("tecoopsSetStream", entry.h, ctypes.c_void_p(stream))
        entry.stream = stream
    return entry.h


def _dtype_code(t):
    if t.dtype == torch.float16:
        return _lib.DATA_HALF
    if t.dtype == torch.bfloat16:
        return _lib.DATA_BFLOAT16
    raise TypeError(f"tecoops: unsupported dtype {t.dtype} (float16 or bfloat16)")


def _ptr(t):
    return None if t is None else t.data_ptr()   # an int: the argtypes make it a pointer


def _check_cuda(*ts):
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("tecoops: tensors must live on a cuda (ROCm) device")


def _check_contiguous(**ts):
    """The C ABI takes plain pointers with packed row-major extents."""
    for name, t in ts.items():
        if t is not None and not t.is_contiguous():
            raise ValueError(f"tecoops: {name} must be contiguous")


def _check_dtype(t, name, *dtypes):
    if t is not None and t.dtype not in dtypes:
        raise TypeError(f"tecoops: {name} must be {' or '.join(str(d) for d in dtypes)}, "
                        f"got {t.dtype}")


def _check_device(device, **ts):
    for name, t in ts.items():
        if t is not None and t.device != device:
            raise ValueError(f"tecoops: {name} must be on {device}, got {t.device}")


def _check_rows(t, name, width):
    """A [rows, width] tensor whose rows are packed (rows may be any distance
    apart): the distance in elements."""
    if t.dim() != 2 or t.shape[1] != width or (width > 1 and t.stride(1) != 1):
        raise ValueError(f"tecoops: {name} must be [rows, {width}] with packed rows")
    if t.shape[0] > 1 and t.stride(0) < width:
        raise ValueError(f"tecoops: rows of {name} must not overlap")
    return t.stride(0) if t.shape[0] > 1 else width


def _choice(table, value, what):
    try:
        return table[value]
    except (KeyError, TypeError):
        raise ValueError(f"tecoops: {what} must be one of "
                         f"{', '.join(str(k) for k in table)}, got {value!r}") from None


def _call_on(device, name, *args):
    """_lib.call with `device` current: a launch goes to the current device."""
    if device.index is None or device.index == torch.cuda.current_device():
        _lib.call(name, *args)
    else:
        with torch.cuda.device(device):
            _lib.call(name, *args)


class _Desc:
    """tecoopsTensorDescriptor_t for a row-major tensor, freed on exit."""

    def __init__(self, t, dtype_code):
        self.d = ctypes.c_void_p()
        _lib.call("tecoopsCreateTensorDescriptor", ctypes.byref(self.d))
        dims = (ctypes.c_int * t.dim())(*t.shape)
        strides = (ctypes.c_int * t.dim())(*t.stride())
        _lib.call("tecoopsSetTensorNdDescriptor", self.d, dtype_code, t.dim(), dims, strides)

    def __enter__(self):
        return self.d

    def __exit__(self, *exc):
        _lib.lib().tecoopsDestroyTensorDescriptor(self.d)


class _DescSlots:
    """The descriptors of one thread's flash-attention calls, one slot per
    argument, filled anew when the tensor's type, shape or strides differ from
    what the slot holds.  Creating, filling and freeing five of them took about
    half of a call's host time: a decode of 4 sequences of 255..4095 keys, whose
    kernels take 16 us, had a host time of 16.6 us per call, now 7.0."""

    def __init__(self, slots):
        self.d = [ctypes.c_void_p() for _ in range(slots)]
        self.held = [None] * slots
        for d in self.d:
            _lib.call("tecoopsCreateTensorDescriptor", ctypes.byref(d))

    def fill(self, slot, t, code):
        d, shape, strides = self.d[slot], t.shape, t.stride()
        want = (code, shape, strides)
        if self.held[slot] != want:
            self.held[slot] = None
            n = len(shape)
            _lib.call("tecoopsSetTensorNdDescriptor", d, code, n, (ctypes.c_int * n)(*shape),
                      (ctypes.c_int * n)(*strides))
            self.held[slot] = want
        return d

    def __del__(self):
        # the thread ended
        try:
            if not sys.is_finalizing():
                for d in self.d:
                    _lib.lib().tecoopsDestroyTensorDescriptor(d)
        except Exception:
            pass


def _desc_slots():
    slots = getattr(_tls, "descs", None)
    if slots is None:
        slots = _tls.descs = _DescSlots(5)
    return slots


# ------------------------------------------------------------------ reference API

def flatten_rays(rays, N, M, res):
    """Reference NeRF op (outside the LLM path): not supported."""
    _lib.call("tecoopsFlattenRays", _handle(rays.device), _ptr(rays), N, M, _ptr(res), 0)


def morton3D_invert(indices, N, coords):
    """Reference NeRF op (outside the LLM path): not supported."""
    _lib.call("tecoopsMorton3DInvert", _handle(indices.device), _ptr(indices), N, _ptr(coords))


def reshape_and_cache(key, value, slot_mapping, key_cache, value_cache):
    """key/value [T, Hkv, D]; caches [num_blocks, Hkv, block_size, D];
    slot_mapping int64 [T] (reference torch_ext.cpp:61-79)."""
    _check_cuda(key, value, slot_mapping, key_cache, value_cache)
    _check_contiguous(key=key, value=value, slot_mapping=slot_mapping, key_cache=key_cache,
                      value_cache=value_cache)
    if slot_mapping.dtype != torch.int64:
        raise TypeError("slot_mapping must be int64")
    T, H, D = key.shape
    _lib.call("tecoopsReshapeAndCacheEx", _handle(key.device), _ptr(key), _ptr(value),
              _ptr(slot_mapping), _ptr(key_cache), _ptr(value_cache), T, H, D,
              key_cache.shape[0], key_cache.shape[2], _dtype_code(key))


def rms_norm(input, weight, residual, output, residual_out, eps):
    """(reference torch_ext.cpp:81-97)."""
    _check_cuda(input, weight, residual, output, residual_out)
    _check_contiguous(input=input, weight=weight, residual=residual, output=output,
                      residual_out=residual_out)
    D = input.shape[-1]
    N = input.numel() // D if D else 0      # leading dims are rows, as in the plugin
    for name, t in (("weight", weight), ("residual", residual), ("output", output),
                    ("residual_out", residual_out)):
        _check_dtype(t, name, input.dtype)
    if weight.numel() != D or output.numel() != input.numel():
        raise ValueError("tecoops.rms_norm: weight must hold hidden_size elements and output "
                         "match input")
    for name, t in (("residual", residual), ("residual_out", residual_out)):
        if t is not None and t.numel() != input.numel():
            raise ValueError(f"tecoops.rms_norm: {name} must match input")
    _lib.call("tecoopsRmsNormEx", _handle(input.device), _ptr(input), _ptr(weight),
              _ptr(residual), _ptr(output), _ptr(residual_out), N, D, float(eps),
              _dtype_code(input))


def flash_attn_varlen_func(q, k, v, max_seqlen_q, cu_seqlens_q, max_seqlen_k, cu_seqlens_k,
                           seqused_k, softmax_scale, causal, window_size, block_table,
                           return_softmax_lse, out):
    """Paged varlen attention (reference torch_ext.cpp:99-165).

    q [sum(L), H, D]; k/v caches [num_blocks, Hkv, block_size, D];
    cu_seqlens_q int32 [B+1]; seqused_k int32 [B]; block_table int32 [B, nb].
    cu_seqlens_k, window_size and return_softmax_lse are accepted and ignored,
    as in the reference."""
    _check_cuda(q, k, v, cu_seqlens_q, seqused_k, block_table, out)
    code = _dtype_code(q)
    scale = float(softmax_scale) if softmax_scale is not None and softmax_scale > 0 else -1.0
    fill = _desc_slots().fill
    _lib.call("tecoopsFlashAttentionEx", _handle(q.device), int(max_seqlen_q), int(max_seqlen_k),
              None, _ptr(cu_seqlens_q), _ptr(seqused_k),
              fill(0, block_table, _lib.DATA_INT32), _ptr(block_table), fill(1, q, code), _ptr(q),
              fill(2, k, code), _ptr(k), fill(3, v, code), _ptr(v), fill(4, out, code), _ptr(out),
              scale, int(bool(causal)), None)


def causal_conv1d_fn_torch(out, conv_states, x, weight, query_start_loc, cache_indices,
                           has_initial_state, pad_slot_id):
    """x, out [dim, total_tokens]; weight [width, dim]; conv_states
    [entries, width-1, dim]; query_start_loc int32 [B+1] (reference
    torch_ext.cpp:167-206).  SiLU is applied, as in the reference."""
    _check_cuda(out, conv_states, x, weight, query_start_loc, cache_indices, has_initial_state)
    dim, total = x.shape
    width = weight.shape[0]
    batch = query_start_loc.shape[0] - 1
    _lib.call("tecoopsCausalConv1dEx", _handle(x.device), batch, total, dim, width,
              _ptr(x), 0, x.stride(1), x.stride(0), _ptr(out), 0, out.stride(1), out.stride(0),
              _ptr(weight), weight.stride(1), weight.stride(0), None, _ptr(conv_states),
              conv_states.stride(0) if conv_states is not None else 0, _ptr(query_start_loc),
              _ptr(cache_indices), _ptr(has_initial_state), int(pad_slot_id), 0, 1)


# ---------------------------------------------------------------------- extensions

def causal_conv1d(x, weight, bias, out, conv_states=None, cache_indices=None,
                  has_initial_state=None, pad_slot_id=-1, activation="silu"):
    """Batched causal conv on x [B, dim, L] with weight [dim, width] and optional
    bias [dim]; writes out [B, dim, L]."""
    _check_cuda(x, weight, bias, out, conv_states, cache_indices, has_initial_state)
    B, dim, L = x.shape
    width = weight.shape[1]
    _lib.call("tecoopsCausalConv1dEx", _handle(x.device), B, L, dim, width,
              _ptr(x), x.stride(0), x.stride(2), x.stride(1),
              _ptr(out), out.stride(0), out.stride(2), out.stride(1),
              _ptr(weight), weight.stride(0), weight.stride(1), _ptr(bias), _ptr(conv_states),
              conv_states.stride(0) if conv_states is not None else 0, None,
              _ptr(cache_indices), _ptr(has_initial_state), int(pad_slot_id), 0,
              int(activation in ("silu", "swish", True)))


def rotary_embedding(positions, query, key, head_size, cos_sin_cache=None, is_neox=True,
                     base=10000.0, rot_dim=None):
    """In place on query [T, H*D or H, D] and key [T, Hkv*D or Hkv, D]."""
    _check_cuda(positions, query, key, cos_sin_cache)
    T = positions.numel()
    H = query.numel() // (T * head_size)
    Hkv = key.numel() // (T * head_size) if key is not None else 0
    rd = rot_dim if rot_dim is not None else (
        cos_sin_cache.shape[1] if cos_sin_cache is not None else head_size)
    if cos_sin_cache is not None and cos_sin_cache.dtype != torch.float32:
        raise TypeError("cos_sin_cache must be float32")
    _lib.call("tecoopsRotaryEmbedding", _handle(query.device), _ptr(positions), _ptr(query),
              _ptr(key), T, H, Hkv, head_size, rd, query.stride(0),
              key.stride(0) if key is not None else 0, _ptr(cos_sin_cache),
              cos_sin_cache.shape[0] if cos_sin_cache is not None else 0, float(base),
              int(bool(is_neox)), _dtype_code(query))


def rotary_reshape_and_cache(positions, query, key, value, slot_mapping, key_cache, value_cache,
                             head_size, cos_sin_cache=None, is_neox=True, base=10000.0,
                             rot_dim=None, write_key=False):
    """Decode step: rotary on query (in place) and key, then the rotated key and
    value stored into the paged caches [num_blocks, Hkv, block_size, head_size]
    at slot_mapping (int64); key is updated in place only when write_key."""
    _check_cuda(positions, query, key, value, slot_mapping, key_cache, value_cache, cos_sin_cache)
    if slot_mapping.dtype != torch.int64 or positions.dtype != torch.int64:
        raise TypeError("positions and slot_mapping must be int64")
    if cos_sin_cache is not None and cos_sin_cache.dtype != torch.float32:
        raise TypeError("cos_sin_cache must be float32")
    T = positions.numel()
    H = query.numel() // (T * head_size)
    Hkv = key.numel() // (T * head_size)
    rd = rot_dim if rot_dim is not None else (
        cos_sin_cache.shape[1] if cos_sin_cache is not None else head_size)
    _lib.call("tecoopsRotaryReshapeAndCache", _handle(query.device), _ptr(positions), _ptr(query),
              _ptr(key), _ptr(value), _ptr(slot_mapping), _ptr(key_cache), _ptr(value_cache),
              T, H, Hkv, head_size, rd, query.stride(0), key.stride(0), value.stride(0),
              _ptr(cos_sin_cache), cos_sin_cache.shape[0] if cos_sin_cache is not None else 0,
              float(base), int(bool(is_neox)), key_cache.shape[0], key_cache.shape[2],
              int(bool(write_key)), _dtype_code(query))


def gemv(weight, x, out):
    """out[b, n] = sum_k weight[n, k] x[b, k]; weight [N, K], x [B, K], out [B, N]."""
    _check_cuda(weight, x, out)
    _check_contiguous(weight=weight, x=x, out=out)
    _check_dtype(weight, "weight", x.dtype)
    _check_dtype(out, "out", x.dtype)
    N, K = weight.shape
    B = x.shape[0] if x.dim() == 2 else 1
    if x.shape[-1] != K or out.numel() != B * N:
        raise ValueError(f"tecoops.gemv: x must be [B, {K}] and out [B, {N}]")
    _lib.call("tecoopsGemv", _handle(x.device), _ptr(weight), _ptr(x), _ptr(out), B, N, K,
              _dtype_code(x))


def gemv_int8(weight, scales, x, out):
    """out[b, n] = scales[n] * sum_k weight[n, k] x[b, k]; weight int8 [N, K]."""
    _check_cuda(weight, scales, x, out)
    _check_contiguous(weight=weight, scales=scales, x=x, out=out)
    _check_dtype(weight, "weight", torch.int8)
    _check_dtype(scales, "scales", torch.float16)
    _check_dtype(x, "x", torch.float16)
    _check_dtype(out, "out", torch.float16)
    N, K = weight.shape
    B = x.shape[0] if x.dim() == 2 else 1
    if x.shape[-1] != K or out.numel() != B * N or scales.numel() != N:
        raise ValueError(f"tecoops.gemv_int8: x must be [B, {K}], out [B, {N}], scales [{N}]")
    _lib.call("tecoopsGemvInt8", _handle(x.device), _ptr(weight), _ptr(scales), _ptr(x),
              _ptr(out), B, N, K)


def _fast(name):
    """The torch op `name` of libtecoops_torch.so, or None when it is not built.
    Its C++ checks and launch take about a third of the host time of a ctypes call
    behind Python ones (12.7 us for the latter, which a product of one row with a
    [4096, 4096] weight does not hide).  When it raises, the Python checks say what
    was wrong with the arguments; what they let pass is raised by _raise.  It is not
    called again: it may have launched, and some of the outputs are inputs too."""
    return None if ops is None else getattr(ops, name).default


def _raise(refused, name):
    """The error that the torch op raised for arguments which the Python checks accept
    (the one in the list `refused`): the TecoopsError of the C function's status when it
    ended in one, else itself.  No frame keeps it, so that the tensors of a failed call
    live no longer than the caller's."""
    error = refused.pop()
    try:
        status = _lib.status_of(str(error))
        if status is None:
            raise error
        raise TecoopsError(status, name) from error
    finally:
        del error


_linear, _moe_layer = _fast("linear"), _fast("moe_layer")
_rotary_axes, _rotary_axes_cache = (_fast("rotary_embedding_axes"),
                                    _fast("rotary_axes_reshape_and_cache"))


def linear(x, weight, out, bias=None, residual=None, activation=None, gated=False):
    """out[m, n] = act(sum_k x[m, k] weight[n, k] + bias[n]) + residual[m, n].

    x [M, K], residual and out [M, N] (rows packed, any distance apart); weight
    [N, K] and bias [N] contiguous.  activation: None, "relu", "silu", "gelu" or
    "gelu_tanh".  gated: weight [2N, K] and bias [2N] hold the gate rows, then
    the up rows, and out = act(gate) * up + residual.  residual may be out
    itself; out must not overlap another input.  float16 or bfloat16; sums and
    epilogue in float32."""
    refused = []
    if _linear is not None:
        try:
            return _linear(x, weight, out, bias, residual, "none" if activation is None else activation,
                           bool(gated))
        except (RuntimeError, TypeError, ValueError) as e:
            refused.append(e.with_traceback(None))
    _check_cuda(x, weight, out, bias, residual)
    code, device = _dtype_code(x), x.device
    if weight.dim() != 2 or x.dim() != 2 or out.dim() != 2:
        raise ValueError("tecoops.linear: x [M, K], weight [N, K], out [M, N]")
    rows, K = weight.shape
    M, N = out.shape
    if x.shape[0] != M or rows != (2 * N if gated else N):
        raise ValueError(f"tecoops.linear: weight must be [{2 * N if gated else N}, {x.shape[1]}] "
                         f"and x [{M}, K] for out [{M}, {N}]")
    _check_contiguous(weight=weight, bias=bias)
    _check_device(device, weight=weight, out=out, bias=bias, residual=residual)
    for name, t in (("weight", weight), ("out", out), ("bias", bias), ("residual", residual)):
        _check_dtype(t, name, x.dtype)
    if bias is not None and bias.numel() != rows:
        raise ValueError(f"tecoops.linear: bias must hold {rows} elements")
    xs, os_ = _check_rows(x, "x", K), _check_rows(out, "out", N)
    rs = 0
    if residual is not None:
        rs = _check_rows(residual, "residual", N)
        if residual.shape[0] != M:
            raise ValueError(f"tecoops.linear: residual must be [{M}, {N}]")
    act = _choice(_lib.ACTIVATIONS, activation, "activation")
    if refused:
        _raise(refused, "tecoopsLinear")
    if M == 0:
        return
    space = _workspace(device, "tecoopsGetLinearWorkspaceSize", M, N, K, int(bool(gated)))
    _call_on(device, "tecoopsLinear", _handle(device), _ptr(x), xs, _ptr(weight), _ptr(bias),
             _ptr(residual), rs, _ptr(out), os_, M, N, K, act, int(bool(gated)), _ptr(space),
             0 if space is None else space.numel(), code)


def moe_layer(x, w_in, w_out, router_logits, top_k, out, renormalize=True, activation="silu",
              topk_ids=None, topk_weights=None):
    """Mixture-of-experts layer for a decode batch: softmax over router_logits
    [T, E] (float32 or x's type), each token's top_k experts (ties to the lowest
    index; -inf and NaN never chosen), and the sum of their outputs
    (act(x Wg^T) * (x Wu^T)) W_out^T with the routing weights, renormalised over
    the chosen or not.  Right for any T, but made for few: every 512 tokens read
    the experts' weights again.

    x [T, H] (rows packed, any distance apart); w_in [E, 2I, H], an expert's gate
    rows before its up rows; w_out [E, H, I]; out [T, H], zero for a token all of
    whose logits are -inf; out must not overlap an input.  topk_ids int32 and
    topk_weights float32 [T, top_k] are written when given, best first, -1 and 0
    where there is none."""
    refused = []
    if _moe_layer is not None:
        try:
            return _moe_layer(x, w_in, w_out, router_logits, int(top_k), out, bool(renormalize),
                              "none" if activation is None else activation, topk_ids,
                              topk_weights)
        except (RuntimeError, TypeError, ValueError) as e:
            refused.append(e.with_traceback(None))
    _check_cuda(x, w_in, w_out, router_logits, out, topk_ids, topk_weights)
    code, device = _dtype_code(x), x.device
    if w_in.dim() != 3 or w_out.dim() != 3 or x.dim() != 2 or router_logits.dim() != 2:
        raise ValueError("tecoops.moe_layer: x [T, H], w_in [E, 2I, H], w_out [E, H, I], "
                         "router_logits [T, E]")
    (E, H, I), T = w_out.shape, x.shape[0]
    if w_in.shape != (E, 2 * I, H) or router_logits.shape != (T, E) or out.shape != (T, H):
        raise ValueError(f"tecoops.moe_layer: w_in must be [{E}, {2 * I}, {H}], router_logits "
                         f"[{T}, {E}] and out [{T}, {H}]")
    _check_contiguous(w_in=w_in, w_out=w_out, router_logits=router_logits, out=out,
                      topk_ids=topk_ids, topk_weights=topk_weights)
    _check_device(device, w_in=w_in, w_out=w_out, router_logits=router_logits, out=out,
                  topk_ids=topk_ids, topk_weights=topk_weights)
    for name, t in (("w_in", w_in), ("w_out", w_out), ("out", out)):
        _check_dtype(t, name, x.dtype)
    _check_dtype(router_logits, "router_logits", torch.float32, x.dtype)
    _check_dtype(topk_ids, "topk_ids", torch.int32)
    _check_dtype(topk_weights, "topk_weights", torch.float32)
    top_k = int(top_k)
    for name, t in (("topk_ids", topk_ids), ("topk_weights", topk_weights)):
        if t is not None and t.shape != (T, top_k):
            raise ValueError(f"tecoops.moe_layer: {name} must be [{T}, {top_k}]")
    xs = _check_rows(x, "x", H)
    act = _choice(_lib.ACTIVATIONS, activation, "activation")
    if refused:
        _raise(refused, "tecoopsMoeLayer")
    if T == 0:
        return
    space = _workspace(device, "tecoopsGetMoeLayerWorkspaceSize", T, H, I, E, top_k)
    _call_on(device, "tecoopsMoeLayer", _handle(device), _ptr(x), xs, _ptr(w_in), _ptr(w_out),
             _ptr(router_logits), _lib.DATA_FLOAT if router_logits.dtype == torch.float32 else code,
             _ptr(out), _ptr(topk_ids), _ptr(topk_weights), T, H, I, E, top_k,
             int(bool(renormalize)), act, _ptr(space), space.numel(), code)


def _workspace(device, size, *args):
    """A workspace of the bytes that the C function `size` asks for, from
    torch's allocator (stream-ordered, and of a graph's own pool under capture),
    or None."""
    n = ctypes.c_size_t()
    _call_on(device, size, *args, ctypes.byref(n))
    return torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None


def _axes_args(name, positions, query, key, head_size, sections, cos_sin_cache, base, rot_dim,
               layout):
    """Checks shared by the rotary functions of several axes; the C arguments
    before and after the pointers.  None: no tokens."""
    _check_cuda(positions, query, key, cos_sin_cache)
    device = query.device
    _check_device(device, positions=positions, key=key, cos_sin_cache=cos_sin_cache)
    sections, head_size = [int(n) for n in sections], int(head_size)
    if head_size <= 0:
        raise ValueError(f"tecoops.{name}: head_size must be positive")
    if positions.dtype != torch.int64:
        raise TypeError(f"tecoops.{name}: positions must be int64")
    if positions.dim() != 2 or positions.shape[0] != len(sections):
        raise ValueError(f"tecoops.{name}: positions must be [axes, tokens], one axis per section")
    T = positions.shape[1]
    if T > 1 and positions.stride(1) != 1:
        raise ValueError(f"tecoops.{name}: the tokens of an axis of positions must be adjacent")
    heads, strides = [], []
    for what, t in (("query", query), ("key", key)):
        if t is None:
            heads.append(0)
            strides.append(0)
            continue
        _check_dtype(t, what, query.dtype)
        row = math.prod(t.shape[1:])
        if t.dim() not in (2, 3) or t.shape[0] != T or row == 0 or row % head_size:
            raise ValueError(f"tecoops.{name}: {what} must be [tokens, heads * head_size] or "
                             "[tokens, heads, head_size]")
        if t.dim() == 3 and t.shape[1] > 1 and t.stride(1) != t.shape[2] or \
                t.shape[-1] > 1 and t.stride(-1) != 1:
            raise ValueError(f"tecoops.{name}: the heads of a token of {what} must be adjacent")
        heads.append(row // head_size)
        strides.append(t.stride(0) if T > 1 else row)
    if cos_sin_cache is not None:
        _check_dtype(cos_sin_cache, "cos_sin_cache", torch.float32)
        _check_contiguous(cos_sin_cache=cos_sin_cache)
        if cos_sin_cache.dim() != 2 or rot_dim not in (None, cos_sin_cache.shape[1]):
            raise ValueError(f"tecoops.{name}: cos_sin_cache must be [positions, rot_dim]")
        rot_dim = cos_sin_cache.shape[1]
    elif rot_dim is None:
        rot_dim = head_size
    lay = _choice(_lib.ROTARY_LAYOUTS, layout, "layout")
    before = (_ptr(positions), positions.stride(0) if len(sections) > 1 else T, len(sections),
              (ctypes.c_int * len(sections))(*sections), lay)
    sizes = (T, heads[0], heads[1], int(head_size), int(rot_dim), strides[0], strides[1])
    table = (_ptr(cos_sin_cache), cos_sin_cache.shape[0] if cos_sin_cache is not None else 0,
             float(base))
    return device, before, sizes, table, _dtype_code(query)


def rotary_embedding_axes(positions, query, key, head_size, sections, cos_sin_cache=None,
                          is_neox=True, base=10000.0, rot_dim=None, layout="contiguous"):
    """Rotary positions of several axes (time, height, width of images and
    video), in place on query [T, H*D or H, D] and key likewise (or None; the
    rows may be slices of a wider product's).

    positions int64 [axes, T] (for plain text, [1, T] expanded); sections: the
    number of frequencies of each axis, rot_dim / 2 together.  layout:
    "contiguous" gives each axis a range of the frequencies, "interleaved"
    frequency i to axis i % axes while that axis has any left (else to the
    first), "per_axis" ranges with frequencies of their own, base^(-j / n) for
    the j-th of an axis' n.  With a cos_sin_cache (float32 [positions, rot_dim]) a
    token with a position outside it is left as it is; without, angles are
    computed in 64 bits (base is taken in float32)."""
    refused = []
    if _rotary_axes is not None and (rot_dim is None or rot_dim > 0):
        try:
            return _rotary_axes(positions, query, key, int(head_size), [int(n) for n in sections],
                                cos_sin_cache, bool(is_neox), float(base), int(rot_dim or 0), layout)
        except (RuntimeError, TypeError, ValueError) as e:
            refused.append(e.with_traceback(None))
    device, before, sizes, table, code = _axes_args("rotary_embedding_axes", positions, query, key,
                                                    head_size, sections, cos_sin_cache, base,
                                                    rot_dim, layout)
    if refused:
        _raise(refused, "tecoopsRotaryEmbeddingAxes")
    if sizes[0] == 0:
        return
    _call_on(device, "tecoopsRotaryEmbeddingAxes", _handle(device), *before, _ptr(query), _ptr(key),
             *sizes, *table, int(bool(is_neox)), code)


def rotary_axes_reshape_and_cache(positions, query, key, value, slot_mapping, key_cache,
                                  value_cache, head_size, sections, cos_sin_cache=None,
                                  is_neox=True, base=10000.0, rot_dim=None, layout="contiguous",
                                  write_key=False):
    """rotary_embedding_axes on query (in place) and key, and the rotated key and
    value stored into the paged caches [num_blocks, Hkv, block_size, head_size]
    at slot_mapping (int64; slots outside the cache are not stored); key is
    updated in place only when write_key."""
    refused = []
    if _rotary_axes_cache is not None and (rot_dim is None or rot_dim > 0):
        try:
            return _rotary_axes_cache(positions, query, key, value, slot_mapping, key_cache,
                                      value_cache, int(head_size), [int(n) for n in sections],
                                      cos_sin_cache, bool(is_neox), float(base), int(rot_dim or 0),
                                      layout, bool(write_key))
        except (RuntimeError, TypeError, ValueError) as e:
            refused.append(e.with_traceback(None))
    name = "rotary_axes_reshape_and_cache"
    if key is None:
        raise ValueError(f"tecoops.{name}: key must be given")
    _check_cuda(value, slot_mapping, key_cache, value_cache)
    device, before, sizes, table, code = _axes_args(name, positions, query, key, head_size,
                                                    sections, cos_sin_cache, base, rot_dim, layout)
    T, _, Hkv, D = sizes[:4]
    _check_device(device, value=value, slot_mapping=slot_mapping, key_cache=key_cache,
                  value_cache=value_cache)
    _check_dtype(slot_mapping, "slot_mapping", torch.int64)
    for what, t in (("value", value), ("key_cache", key_cache), ("value_cache", value_cache)):
        _check_dtype(t, what, query.dtype)
    _check_contiguous(slot_mapping=slot_mapping, key_cache=key_cache, value_cache=value_cache)
    if slot_mapping.numel() != T:
        raise ValueError(f"tecoops.{name}: slot_mapping must hold {T} slots")
    if key_cache.dim() != 4 or key_cache.shape[1] != Hkv or key_cache.shape[3] != D or \
            value_cache.shape != key_cache.shape:
        raise ValueError(f"tecoops.{name}: caches must be [num_blocks, {Hkv}, block_size, {D}]")
    if value.dim() not in (2, 3) or value.shape[0] != T or math.prod(value.shape[1:]) != Hkv * D:
        raise ValueError(f"tecoops.{name}: value must match key")
    if value.dim() == 3 and value.shape[1] > 1 and value.stride(1) != value.shape[2] or \
            value.shape[-1] > 1 and value.stride(-1) != 1:
        raise ValueError(f"tecoops.{name}: the heads of a token of value must be adjacent")
    if refused:
        _raise(refused, "tecoopsRotaryAxesReshapeAndCache")
    if T == 0:
        return
    _call_on(device, "tecoopsRotaryAxesReshapeAndCache", _handle(device), *before, _ptr(query),
             _ptr(key), _ptr(value), _ptr(slot_mapping), _ptr(key_cache), _ptr(value_cache), *sizes,
             value.stride(0) if T > 1 else Hkv * D, *table, int(bool(is_neox)), key_cache.shape[0],
             key_cache.shape[2], int(bool(write_key)), code)


_qk_norm, _qk_norm_cache = _fast("qk_norm_rotary"), _fast("qk_norm_rotary_reshape_and_cache")
_cache_int4, _attn_int4, _gemv_int4 = (_fast("reshape_and_cache_int4"),
                                       _fast("flash_attn_varlen_int4"), _fast("gemv_int4"))


def _one_or_more_axes(positions, sections, cos_sin_cache, head_size, rot_dim):
    """positions as [axes, T] and the sections: [T] and None are one axis."""
    if positions.dim() == 1:
        positions = positions.unsqueeze(0)
    if sections is None:
        if cos_sin_cache is not None and cos_sin_cache.dim() == 2:
            rot_dim = cos_sin_cache.shape[1]
        sections = [(head_size if rot_dim is None else rot_dim) // 2]
    return positions, sections


def _check_weight(t, name, query, head_size):
    if t is None or t.dim() != 1 or t.shape[0] != head_size:
        raise ValueError(f"tecoops: {name} must be [{head_size}]")
    _check_dtype(t, name, query.dtype)
    _check_contiguous(**{name: t})
    _check_device(query.device, **{name: t})


def _check_caches(name, T, Hkv, D, dtype, device, value, slot_mapping, key_cache, value_cache):
    _check_cuda(value, slot_mapping, key_cache, value_cache)
    _check_device(device, value=value, slot_mapping=slot_mapping, key_cache=key_cache,
                  value_cache=value_cache)
    _check_dtype(slot_mapping, "slot_mapping", torch.int64)
    for what, t in (("value", value), ("key_cache", key_cache), ("value_cache", value_cache)):
        _check_dtype(t, what, dtype)
    _check_contiguous(slot_mapping=slot_mapping, key_cache=key_cache, value_cache=value_cache)
    if slot_mapping.numel() != T:
        raise ValueError(f"tecoops.{name}: slot_mapping must hold {T} slots")
    if key_cache.dim() != 4 or key_cache.shape[1] != Hkv or key_cache.shape[3] != D or \
            value_cache.shape != key_cache.shape:
        raise ValueError(f"tecoops.{name}: caches must be [num_blocks, {Hkv}, block_size, {D}]")
    if value.dim() not in (2, 3) or value.shape[0] != T or math.prod(value.shape[1:]) != Hkv * D:
        raise ValueError(f"tecoops.{name}: value must match key")
    if value.dim() == 3 and value.shape[1] > 1 and value.stride(1) != value.shape[2] or \
            value.shape[-1] > 1 and value.stride(-1) != 1:
        raise ValueError(f"tecoops.{name}: the heads of a token of value must be adjacent")


def qk_norm_rotary(positions, query, key, query_weight, key_weight, head_size, eps=1e-6,
                   cos_sin_cache=None, is_neox=True, base=10000.0, rot_dim=None, sections=None,
                   layout="contiguous"):
    """The norm of each head of query and key, then the rotation, in one pass, in
    place on query [T, H*D or H, D] and key likewise (or None, with its weight):
    x / sqrt(mean(x^2) + eps) * weight over the D = head_size elements of a head,
    turned by the token's position; float32 throughout, one rounding.

    positions int64 [T], or [axes, T] with sections and layout as in
    rotary_embedding_axes.  query_weight and key_weight [D] of query's type.  The
    rows may be slices of a wider product's.  A token with a position outside the
    cos_sin_cache is left as it is, not normalised either."""
    refused = []
    if _qk_norm is not None and (rot_dim is None or rot_dim > 0) and sections != []:
        try:
            return _qk_norm(positions, query, key, query_weight, key_weight, int(head_size), float(eps),
                            [] if sections is None else [int(n) for n in sections], cos_sin_cache,
                            bool(is_neox), float(base), int(rot_dim or 0), layout)
        except (RuntimeError, TypeError, ValueError) as e:
            refused.append(e.with_traceback(None))
    name = "qk_norm_rotary"
    positions, sections = _one_or_more_axes(positions, sections, cos_sin_cache, head_size, rot_dim)
    device, before, sizes, table, code = _axes_args(name, positions, query, key, head_size, sections,
                                                    cos_sin_cache, base, rot_dim, layout)
    _check_weight(query_weight, "query_weight", query, head_size)
    if key is not None:
        _check_weight(key_weight, "key_weight", query, head_size)
    if refused:
        _raise(refused, "tecoopsQkNormRotary")
    if sizes[0] == 0:
        return
    _call_on(device, "tecoopsQkNormRotary", _handle(device), *before, _ptr(query), _ptr(key),
             _ptr(query_weight), _ptr(key_weight), float(eps), *sizes, *table, int(bool(is_neox)), code)


def qk_norm_rotary_reshape_and_cache(positions, query, key, value, query_weight, key_weight,
                                     slot_mapping, key_cache, value_cache, head_size, eps=1e-6,
                                     cos_sin_cache=None, is_neox=True, base=10000.0, rot_dim=None,
                                     sections=None, layout="contiguous", write_key=False):
    """qk_norm_rotary on query (in place) and key, and the key that comes of it and
    value stored into the paged caches [num_blocks, Hkv, block_size, head_size] at
    slot_mapping (int64; slots outside the cache are not stored); key is updated in
    place only when write_key."""
    refused = []
    if _qk_norm_cache is not None and (rot_dim is None or rot_dim > 0) and sections != []:
        try:
            return _qk_norm_cache(positions, query, key, value, query_weight, key_weight, slot_mapping,
                                  key_cache, value_cache, int(head_size), float(eps),
                                  [] if sections is None else [int(n) for n in sections],
                                  cos_sin_cache, bool(is_neox), float(base), int(rot_dim or 0), layout,
                                  bool(write_key))
        except (RuntimeError, TypeError, ValueError) as e:
            refused.append(e.with_traceback(None))
    name = "qk_norm_rotary_reshape_and_cache"
    if key is None:
        raise ValueError(f"tecoops.{name}: key must be given")
    positions, sections = _one_or_more_axes(positions, sections, cos_sin_cache, head_size, rot_dim)
    device, before, sizes, table, code = _axes_args(name, positions, query, key, head_size, sections,
                                                    cos_sin_cache, base, rot_dim, layout)
    _check_weight(query_weight, "query_weight", query, head_size)
    _check_weight(key_weight, "key_weight", query, head_size)
    T, _, Hkv, D = sizes[:4]
    _check_caches(name, T, Hkv, D, query.dtype, device, value, slot_mapping, key_cache, value_cache)
    if refused:
        _raise(refused, "tecoopsQkNormRotaryReshapeAndCache")
    if T == 0:
        return
    _call_on(device, "tecoopsQkNormRotaryReshapeAndCache", _handle(device), *before, _ptr(query),
             _ptr(key), _ptr(value), _ptr(query_weight), _ptr(key_weight), float(eps),
             _ptr(slot_mapping), _ptr(key_cache), _ptr(value_cache), *sizes,
             value.stride(0) if T > 1 else Hkv * D, *table, int(bool(is_neox)), key_cache.shape[0],
             key_cache.shape[2], int(bool(write_key)), code)


def _check_cache_int4(name, device, dtype, D, key_cache, value_cache, key_scales, value_scales):
    _check_cuda(key_cache, value_cache, key_scales, value_scales)
    held = dict(key_cache=key_cache, value_cache=value_cache, key_scales=key_scales,
                value_scales=value_scales)
    _check_device(device, **held)
    _check_contiguous(**held)
    for what, t in held.items():
        _check_dtype(t, what, torch.uint8 if what.endswith("cache") else dtype)
    if key_cache.dim() != 4 or 2 * key_cache.shape[3] != D or value_cache.shape != key_cache.shape:
        raise ValueError(f"tecoops.{name}: caches must be uint8 [num_blocks, kv heads, block_size, "
                         f"{D} / 2]")
    if key_scales.shape != (*key_cache.shape[:3], 2) or value_scales.shape != key_scales.shape:
        raise ValueError(f"tecoops.{name}: scales must be [num_blocks, kv heads, block_size, 2]")


def reshape_and_cache_int4(key, value, slot_mapping, key_cache, value_cache, key_scales,
                           value_scales):
    """key/value [T, Hkv, D] (heads of a token adjacent, tokens any distance apart)
    stored in 4 bits at slot_mapping (int64 [T]; slots outside the cache are not
    stored, a slot is at most once in a call): a row x of a head as codes n of 0..15
    and a pair (scale, low) that stands for scale * n + low, low = min x, scale =
    (max x - min x) / 15 in key's type, n = (x - low) / scale to the nearest.  A row
    with a NaN or an infinity reads as NaN.

    key_cache / value_cache uint8 [num_blocks, Hkv, block_size, D / 2], element 2j
    in the low half of byte j; key_scales / value_scales of key's type [num_blocks,
    Hkv, block_size, 2].  D a multiple of 8 up to 512."""
    refused = []
    if _cache_int4 is not None:
        try:
            return _cache_int4(key, value, slot_mapping, key_cache, value_cache, key_scales,
                               value_scales)
        except (RuntimeError, TypeError, ValueError) as e:
            refused.append(e.with_traceback(None))
    name = "reshape_and_cache_int4"
    _check_cuda(key, value, slot_mapping)
    code, device = _dtype_code(key), key.device
    _check_device(device, value=value, slot_mapping=slot_mapping)
    _check_dtype(value, "value", key.dtype)
    _check_dtype(slot_mapping, "slot_mapping", torch.int64)
    _check_contiguous(slot_mapping=slot_mapping)
    if key.dim() != 3 or value.shape != key.shape or slot_mapping.numel() != key.shape[0]:
        raise ValueError(f"tecoops.{name}: key / value [tokens, kv heads, head_size], slot_mapping "
                         "[tokens]")
    T, H, D = key.shape
    _check_cache_int4(name, device, key.dtype, D, key_cache, value_cache, key_scales, value_scales)
    if key_cache.shape[1] != H:
        raise ValueError(f"tecoops.{name}: the caches must hold {H} kv heads")
    for what, t in (("key", key), ("value", value)):
        if D > 1 and t.stride(2) != 1 or H > 1 and t.stride(1) != D or T > 1 and t.stride(0) < H * D:
            raise ValueError(f"tecoops.{name}: the heads of a token of {what} must be adjacent")
    if refused:
        _raise(refused, "tecoopsReshapeAndCacheInt4")
    if T == 0:
        return
    _call_on(device, "tecoopsReshapeAndCacheInt4", _handle(device), _ptr(key), _ptr(value),
             _ptr(slot_mapping), _ptr(key_cache), _ptr(value_cache), _ptr(key_scales),
             _ptr(value_scales), T, H, D, key.stride(0) if T > 1 else H * D,
             value.stride(0) if T > 1 else H * D, key_cache.shape[0], key_cache.shape[2], code)


def flash_attn_varlen_int4(q, key_cache, value_cache, key_scales, value_scales, max_seqlen_q,
                           cu_seqlens_q, max_seqlen_k, seqused_k, softmax_scale, causal, block_table,
                           out):
    """flash_attn_varlen_func over a cache held in 4 bits (reshape_and_cache_int4).

    q, out [sum(L), H, D] contiguous; cu_seqlens_q int32 [B+1]; seqused_k int32 [B];
    block_table int32 [B, blocks] (rows any distance apart).  softmax_scale None: 1 /
    sqrt(D).  max_seqlen_q and max_seqlen_k shape the launch only.  Rows of no
    sequence and rows without a visible key are 0; what the cache holds behind a
    sequence's last key is not used."""
    refused = []
    scale = float(softmax_scale) if softmax_scale is not None and softmax_scale > 0 else -1.0
    if _attn_int4 is not None:
        try:
            return _attn_int4(q, key_cache, value_cache, key_scales, value_scales, int(max_seqlen_q),
                              cu_seqlens_q, int(max_seqlen_k), seqused_k, scale, bool(causal),
                              block_table, out)
        except (RuntimeError, TypeError, ValueError) as e:
            refused.append(e.with_traceback(None))
    name = "flash_attn_varlen_int4"
    _check_cuda(q, cu_seqlens_q, seqused_k, block_table, out)
    code, device = _dtype_code(q), q.device
    _check_device(device, cu_seqlens_q=cu_seqlens_q, seqused_k=seqused_k, block_table=block_table,
                  out=out)
    if q.dim() != 3 or out.shape != q.shape:
        raise ValueError(f"tecoops.{name}: q and out must be [rows, heads, head_size]")
    _check_dtype(out, "out", q.dtype)
    _check_contiguous(q=q, out=out, cu_seqlens_q=cu_seqlens_q, seqused_k=seqused_k)
    T, H, D = q.shape
    _check_cache_int4(name, device, q.dtype, D, key_cache, value_cache, key_scales, value_scales)
    for what, t in (("cu_seqlens_q", cu_seqlens_q), ("seqused_k", seqused_k),
                    ("block_table", block_table)):
        _check_dtype(t, what, torch.int32)
    B = seqused_k.numel()
    if B == 0 or cu_seqlens_q.numel() != B + 1 or block_table.dim() != 2 or \
            block_table.shape[0] != B or block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError(f"tecoops.{name}: cu_seqlens_q must be [batch + 1], seqused_k [batch] and "
                         "block_table [batch, blocks] with adjacent entries in a row")
    if refused:
        _raise(refused, "tecoopsFlashAttentionInt4")
    if T == 0:
        return
    NB, Hkv, BS = key_cache.shape[:3]
    most_q = min(max(int(max_seqlen_q), 0), 0x7fffffff)
    cap = max(1, min(block_table.shape[1] * BS, 0x7fffffff))
    most_k = min(int(max_seqlen_k), cap) if max_seqlen_k > 0 else cap
    space = _workspace(device, "tecoopsGetFlashAttentionInt4WorkspaceSize", B, T, H, Hkv, D, most_q,
                       most_k)
    _call_on(device, "tecoopsFlashAttentionInt4", _handle(device), most_q, most_k, _ptr(cu_seqlens_q),
             _ptr(seqused_k), _ptr(block_table), block_table.stride(0) if B > 1 else block_table.shape[1],
             B, block_table.shape[1], _ptr(q), _ptr(key_cache), _ptr(value_cache), _ptr(key_scales),
             _ptr(value_scales), _ptr(out), T, H, Hkv, D, NB, BS, scale, int(bool(causal)), _ptr(space),
             0 if space is None else space.numel(), code)


def gemv_int4(weight, scales, x, out, zeros=None):
    """out[b, n] = sum_k W[n, k] x[b, k] with 4-bit weights, W[n, k] = (code - zero) *
    scale of the group that k is in; float32 sums, one rounding.

    weight uint8 [N, K / 2], code 2j of a row in the low half of byte j; scales and
    zeros (None: 8) of x's type [N, K / group], group a multiple of 32; x [B, K] or
    [K], out [B, N].  For decode batches."""
    refused = []
    if _gemv_int4 is not None:
        try:
            return _gemv_int4(weight, scales, x, out, zeros)
        except (RuntimeError, TypeError, ValueError) as e:
            refused.append(e.with_traceback(None))
    _check_cuda(weight, scales, x, out, zeros)
    code, device = _dtype_code(x), x.device
    _check_device(device, weight=weight, scales=scales, out=out, zeros=zeros)
    _check_contiguous(weight=weight, scales=scales, x=x, out=out, zeros=zeros)
    _check_dtype(weight, "weight", torch.uint8)
    for name, t in (("scales", scales), ("out", out), ("zeros", zeros)):
        _check_dtype(t, name, x.dtype)
    if x.dim() not in (1, 2) or weight.dim() != 2 or scales.dim() != 2:
        raise ValueError("tecoops.gemv_int4: weight [N, K / 2], scales [N, K / group], x [B, K] or [K]")
    N, K = weight.shape[0], 2 * weight.shape[1]
    B = x.shape[0] if x.dim() == 2 else 1
    if x.shape[-1] != K or out.numel() != B * N or scales.shape[0] != N or scales.shape[1] == 0 or \
            K == 0 or K % scales.shape[1]:
        raise ValueError(f"tecoops.gemv_int4: scales must be [{N}, K / group], x [B, {K}] and out "
                         f"[B, {N}]")
    if zeros is not None and zeros.shape != scales.shape:
        raise ValueError("tecoops.gemv_int4: zeros must match scales")
    if refused:
        _raise(refused, "tecoopsGemvInt4")
    if B == 0:
        return
    space = _workspace(device, "tecoopsGetGemvInt4WorkspaceSize", B, N, K)
    _call_on(device, "tecoopsGemvInt4", _handle(device), _ptr(weight), _ptr(scales), _ptr(zeros),
             _ptr(x), _ptr(out), B, N, K, K // scales.shape[1], _ptr(space),
             0 if space is None else space.numel(), code)


def memset(t, value):
    """Byte fill of a tensor's storage (value truncated to uint8)."""
    _check_cuda(t)
    _lib.call("tecoopsMemset", _handle(t.device), _ptr(t), int(value),
              t.numel() * t.element_size())
