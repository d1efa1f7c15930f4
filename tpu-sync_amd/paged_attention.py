"""Operators that fill and read the paged KV pool (libkvx's attention kernels).

``norm_rope`` is the RMS norm of query and key heads and the position rotation
in one pass. ``append_kv`` and ``attend`` are methods of ``KVCacheManager``;
their argument handling is here. The three are a step's work around the cache:

    q, _ = norm_rope(q, None, positions, inv_freq, q_weight=wq)
    mgr.append_kv(2 * i, 2 * i + 1, k, v, tables, lengths, inv_freq=inv_freq, k_weight=wk)
    out = mgr.attend(2 * i, 2 * i + 1, q, tables, lengths)

They are serving operators with no backward pass: tensors that require
gradients are refused while gradients are recorded. Calls are enqueued on
``stream`` (default: torch's current stream), allocate their outputs and
workspace from torch's allocator on that stream, and can be captured into a
graph. This module only passes pointers; the checks behind it are libkvx's.
"""
import contextlib
import ctypes
from typing import Optional, Tuple

from . import _capi
from .kv_cache_manager import _stream_ptr

_TYPES = {}


def _types():
    if not _TYPES:
        import torch
        _TYPES.update({torch.bfloat16: _capi.BF16, torch.float16: _capi.F16,
                       torch.float32: _capi.F32, torch.float8_e4m3fn: _capi.E4M3})
    return _TYPES


def _device_tensor(t, what, device):
    if not getattr(t, "is_cuda", False):
        raise ValueError(f"{what} must be a tensor on a HIP device, got {getattr(t, 'device', t)}")
    index = t.device.index or 0
    if device is not None and index != device:
        raise ValueError(f"{what} is on device {index}, expected device {device}")
    return index


def _rows(t, what, device, dtype=None, shape=None):
    """Checks a [tokens, heads, head_dim] tensor whose last dimension is
    contiguous; returns its (token, head) strides."""
    _device_tensor(t, what, device)
    if t.dim() != 3:
        raise ValueError(f"{what} must be [tokens, heads, head_dim], got {tuple(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be {tuple(shape)}, got {tuple(t.shape)}")
    if t.requires_grad:
        import torch
        if torch.is_grad_enabled():
            raise ValueError(f"{what} requires gradients: there is no backward pass")
    token, head, last = t.stride()
    if last != 1 and t.shape[2] != 1:
        raise ValueError(f"{what} must be contiguous in its last dimension")
    return token, head


def _vector(t, what, device, dtypes, n):
    _device_tensor(t, what, device)
    if t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{what} must be a contiguous tensor of {n} elements, "
                         f"got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} must be one of {', '.join(str(d) for d in dtypes)}, "
                         f"got {t.dtype}")
    return t.data_ptr()


def _weight(args, t, what, device, dtype, n):
    import torch
    if t is None:
        return 0
    ptr = _vector(t, what, device, (dtype, torch.float32), n)
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{what} requires gradients: there is no backward pass")
    args.weight_dtype = _types()[t.dtype]
    return ptr


def _rotation(args, device, inv_freq, positions, tokens, head_dim):
    import torch
    if inv_freq is None:
        return
    _device_tensor(inv_freq, "inv_freq", device)
    n = inv_freq.shape[0] if inv_freq.dim() == 1 else -1
    if not 1 <= 2 * n <= head_dim:
        raise ValueError(f"inv_freq must have 1 to {head_dim // 2} elements, "
                         f"got {tuple(inv_freq.shape)}")
    args.inv_freq = _vector(inv_freq, "inv_freq", device, (torch.float32,), n)
    args.rotary_dim = 2 * n
    if positions is not None:
        args.positions = _vector(positions, "positions", device, (torch.int32, torch.int64),
                                 tokens)
        args.positions_64 = int(positions.dtype == torch.int64)


@contextlib.contextmanager
def _torch_stream(stream, device):
    import torch
    if isinstance(stream, torch.cuda.Stream):
        use = stream
    else:
        ptr = _stream_ptr(stream)
        use = (torch.cuda.ExternalStream(ptr, device=device) if ptr
               else torch.cuda.default_stream(device))
    with torch.cuda.stream(use):
        yield


def _on_stream(stream, device):
    """(stream handle, context in which torch allocates for that stream)."""
    if stream is None:
        import torch
        return torch.cuda.current_stream(device).cuda_stream, contextlib.nullcontext()
    return _stream_ptr(stream), _torch_stream(stream, device)


def norm_rope(q, k, positions, inv_freq, *, q_weight=None, k_weight=None, eps: float = 1e-6,
              interleaved: bool = False, out_q=None, out_k=None, stream=None) -> Tuple:
    """RMS norm and position rotation of every head of ``q`` and ``k``.

    Args:
      q, k: [tokens, heads, head_dim] of bf16, fp16 or fp32, head_dim up to
        256; any strides but a contiguous last dimension (parts of a fused
        projection). ``k`` may be None.
      positions: int32 or int64 [tokens].
      inv_freq: fp32 [rotary_dim / 2] with rotary_dim <= head_dim; the angle of
        pair i is position * inv_freq[i], good to 2^-25 turns for positions up to
        2^53. Dimensions from rotary_dim on are not rotated. None: norm only.
      q_weight, k_weight: [head_dim], of the rows' type or fp32; None: no norm.
      interleaved: pairs are (2i, 2i + 1) instead of (i, i + rotary_dim / 2).
      out_q, out_k: results; the input itself, or apart from the inputs.
        Default: new contiguous tensors.
    Returns (q, k) results, k's None without ``k``.
    """
    import torch
    args = _capi.NormRopeArgs()
    device = _device_tensor(q, "q", None)
    args.q_token_stride, args.q_head_stride = _rows(q, "q", device)
    tokens, args.q_heads, dim = q.shape
    dtype = q.dtype
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"q must be bfloat16, float16 or float32, got {dtype}")
    if inv_freq is not None and positions is None:
        raise ValueError("positions are needed with inv_freq")
    args.device, args.dtype, args.tokens, args.head_dim = device, _types()[dtype], tokens, dim
    args.q = q.data_ptr()
    if k is not None:
        args.k_token_stride, args.k_head_stride = _rows(k, "k", device, dtype,
                                                        (tokens, k.shape[1], dim)
                                                        if k.dim() == 3 else None)
        args.k_heads, args.k = k.shape[1], k.data_ptr()
    elif out_k is not None:
        raise ValueError("out_k without k")
    args.eps, args.interleaved = eps, int(interleaved)
    args.q_weight = _weight(args, q_weight, "q_weight", device, dtype, dim)
    args.k_weight = _weight(args, k_weight, "k_weight", device, dtype, dim)
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("q_weight and k_weight must have the same dtype")
    _rotation(args, device, inv_freq, positions, tokens, dim)
    handle, context = _on_stream(stream, device)
    with context:
        if out_q is None:
            out_q = torch.empty(q.shape, dtype=dtype, device=q.device)
        if out_k is None and k is not None:
            out_k = torch.empty(k.shape, dtype=dtype, device=q.device)
    args.q_out_token_stride, args.q_out_head_stride = _rows(out_q, "out_q", device, dtype, q.shape)
    args.q_out = out_q.data_ptr()
    if k is not None:
        args.k_out_token_stride, args.k_out_head_stride = _rows(out_k, "out_k", device, dtype,
                                                                k.shape)
        args.k_out = out_k.data_ptr()
    _capi.check(_capi.load().kvx_norm_rope(ctypes.byref(args), handle), "norm_rope")
    return out_q, out_k


def _cache(args, mgr, k_layer, v_layer, shard_idx, dtype):
    """Describes two of the manager's storages; returns their (heads, head_dim)."""
    import torch
    if mgr._device is None:
        raise _capi.KvxError(9, "needs a device-backed KVCacheManagerBase", "KVCacheManager")
    layers = mgr._tensors
    shapes = []
    for layer in (k_layer, v_layer):
        if not 0 <= layer < mgr.num_kv_layers or not 0 <= shard_idx < len(layers[layer]):
            raise _capi.KvxError(11, "layer or shard index out of range", "KVCacheManager")
        t = layers[layer][shard_idx]
        if t.dim() != 4:
            raise ValueError("the cache's storages must be [blocks, tokens, heads, head_dim] "
                             f"tensors, got {tuple(t.shape)}")
        if t.dtype not in (dtype, torch.float8_e4m3fn):
            raise ValueError(f"the cache must be {dtype} or float8_e4m3fn, got {t.dtype}")
        shapes.append((t.dtype,) + tuple(t.shape[1:]))
    if shapes[0] != shapes[1]:
        raise ValueError("the key and value storages must have the same type and block shape")
    cache = args.cache
    cache.k_layer, cache.v_layer, cache.shard = k_layer, v_layer, shard_idx
    kind, cache.block_tokens, cache.heads, cache.head_dim = shapes[0]
    cache.dtype = _types()[kind]
    if cache.dtype == _capi.E4M3:
        # Scale tables follow the KV storages, one a storage.
        n = mgr.num_kv_layers
        if len(layers) != 2 * n:
            raise ValueError("a float8 cache needs one scale table a KV storage "
                             f"({n}), got {len(layers) - n}")
        for layer in (n + k_layer, n + v_layer):
            if layers[layer][shard_idx].dtype != torch.float32:
                raise ValueError("scale tables must be float32")
        cache.k_scale_layer, cache.v_scale_layer = n + k_layer, n + v_layer
    return cache.heads, cache.head_dim


def _batch(args, device, tables, lengths, starts, tokens):
    import torch
    batch = args.batch
    _device_tensor(tables, "tables", device)
    if tables.dim() != 2 or tables.dtype != torch.int32:
        raise ValueError(f"tables must be an int32 [sequences, blocks] tensor, got "
                         f"{tables.dtype} {tuple(tables.shape)}")
    n, batch.table_width = tables.shape
    if batch.table_width > 1 and tables.stride(1) != 1:
        raise ValueError("tables must be contiguous in their last dimension")
    batch.tables, batch.table_stride = tables.data_ptr(), tables.stride(0)
    batch.lengths = _vector(lengths, "lengths", device, (torch.int32,), n)
    batch.sequences = n
    if starts is not None:
        batch.starts = _vector(starts, "starts", device, (torch.int32,), n + 1)
    elif tokens != n:
        raise ValueError(f"without starts there is one token a sequence: {tokens} tokens, "
                         f"{n} sequences")


def append_kv(mgr, k_layer, v_layer, k, v, tables, lengths, *, starts, inv_freq, positions,
              k_weight, eps, interleaved, shard_idx, stream) -> None:
    args = _capi.AppendKvArgs()
    device = mgr._device
    args.k_token_stride, args.k_head_stride = _rows(k, "k", device)
    dtype = k.dtype
    heads, dim = _cache(args, mgr, k_layer, v_layer, shard_idx, dtype)
    tokens = k.shape[0]
    shape = (tokens, heads, dim)
    if tuple(k.shape) != shape:
        raise ValueError(f"k must be {shape}, got {tuple(k.shape)}")
    args.v_token_stride, args.v_head_stride = _rows(v, "v", device, dtype, shape)
    args.k, args.v, args.tokens, args.dtype = k.data_ptr(), v.data_ptr(), tokens, _types()[dtype]
    _batch(args, device, tables, lengths, starts, tokens)
    if positions is not None and inv_freq is None:
        raise ValueError("positions without inv_freq")
    _rotation(args, device, inv_freq, positions, tokens, dim)
    args.k_weight = _weight(args, k_weight, "k_weight", device, dtype, dim)
    args.eps, args.interleaved = eps, int(interleaved)
    handle, _ = _on_stream(stream, device)
    _capi.check(_capi.load().kvx_manager_append_kv(mgr._h, ctypes.byref(args), handle),
                "KVCacheManager append_kv")


def attend(mgr, k_layer, v_layer, q, tables, lengths, *, starts, group_starts, prefix_lengths,
           scale, causal, out, return_lse, shard_idx, stream):
    import torch
    args = _capi.AttendArgs()
    device = mgr._device
    args.q_token_stride, args.q_head_stride = _rows(q, "q", device)
    dtype = q.dtype
    _, dim = _cache(args, mgr, k_layer, v_layer, shard_idx, dtype)
    tokens, args.q_heads, q_dim = q.shape
    if q_dim != dim:
        raise ValueError(f"q must have head_dim {dim}, got {q_dim}")
    args.q, args.tokens, args.dtype = q.data_ptr(), tokens, _types()[dtype]
    _batch(args, device, tables, lengths, starts, tokens)
    if (group_starts is None) != (prefix_lengths is None):
        raise ValueError("group_starts and prefix_lengths go together")
    if group_starts is not None:
        groups = prefix_lengths.shape[0] if prefix_lengths.dim() == 1 else -1
        args.prefix_lengths = _vector(prefix_lengths, "prefix_lengths", device, (torch.int32,),
                                      groups)
        args.group_starts = _vector(group_starts, "group_starts", device, (torch.int32,),
                                    groups + 1)
        args.groups = groups
    args.scale = dim ** -0.5 if scale is None else scale
    args.non_causal = int(not causal)
    lib = _capi.load()
    where = "KVCacheManager attend"
    need = ctypes.c_int64()
    _capi.check(lib.kvx_manager_attend_workspace(mgr._h, ctypes.byref(args), ctypes.byref(need)),
                where)
    handle, context = _on_stream(stream, device)
    workspace = lse = None
    with context:
        if out is None:
            out = torch.empty((tokens, args.q_heads, dim), dtype=dtype, device=q.device)
        if return_lse:
            lse = torch.empty((tokens, args.q_heads), dtype=torch.float32, device=q.device)
            args.lse = lse.data_ptr()
        if need.value > 0:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=q.device)
            args.workspace, args.workspace_bytes = workspace.data_ptr(), need.value
    args.out_token_stride, args.out_head_stride = _rows(out, "out", device, dtype, q.shape)
    args.out = out.data_ptr()
    _capi.check(lib.kvx_manager_attend(mgr._h, ctypes.byref(args), handle), where)
    return (out, lse) if return_lse else out
