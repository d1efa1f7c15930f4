"""Operators that fill and read the paged KV pool (libkvx's attention kernels).

``norm_rope`` is the RMS norm of query and key heads and the position rotation
in one pass. ``append_kv`` and ``attend`` are methods of ``KVCacheManager``, over
pools of the tensors' type, float8 or 4 bits with their scales;
their argument handling is here. The three are a step's work around the cache:

    q, _ = norm_rope(q, None, positions, inv_freq, q_weight=wq)
    mgr.append_kv(2 * i, 2 * i + 1, k, v, tables, lengths, inv_freq=inv_freq, k_weight=wk)
    out = mgr.attend(2 * i, 2 * i + 1, q, tables, lengths)

They are serving operators with no derivatives: tensors that require gradients
are refused while gradients are recorded, and so are dual tensors of forward-mode
differentiation. Calls are enqueued on
``stream`` (default: torch's current stream), allocate their outputs and
workspace from torch's allocator on that stream, and can be captured into a
graph. This module only passes pointers; the checks behind it are libkvx's.
"""
import contextlib
import ctypes
import struct
from typing import Tuple

from . import _capi
from .kv_cache_manager import _stream_ptr

# A call's arguments are packed in one go (setting a ctypes structure field by
# field costs a decode step more than its kernel takes).
_CACHE, _BATCH = "5q4i", "QqqQQq"
_NORM_ROPE = struct.Struct("2iq4i4Q8q2Q2i2Qfi")
_APPEND_KV = struct.Struct(_CACHE + _BATCH + "q2i2Q4qQ2i2Qfi")
_ATTEND = struct.Struct(_CACHE + _BATCH + "q2i2Q4q3Q2ifiQq")
for _pack, _args in ((_NORM_ROPE, _capi.NormRopeArgs), (_APPEND_KV, _capi.AppendKvArgs),
                     (_ATTEND, _capi.AttendArgs)):
    assert _pack.size == ctypes.sizeof(_args)

_TYPES = {}
_torch = _forward_ad = None
_FP4 = None  # torch's 4-bit type, where it has one


def _current_stream(device):
    return _torch.cuda.current_stream(device).cuda_stream


def _load_torch():
    global _torch, _forward_ad, _current_stream, _FP4
    if _torch is None:
        import torch
        from torch.autograd import forward_ad
        _forward_ad = forward_ad
        # The handle alone, without a Stream object around it, where torch has it.
        _current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _current_stream)
        _TYPES.update({torch.bfloat16: _capi.BF16, torch.float16: _capi.F16,
                       torch.float32: _capi.F32, torch.float8_e4m3fn: _capi.E4M3})
        _FP4 = getattr(torch, "float4_e2m1fn_x2", None)
        if _FP4 is not None:
            _TYPES[_FP4] = _capi.FP4
        _torch = torch
    return _torch


def _off_device(t, what, device):
    """Why a tensor is not on the device."""
    if not getattr(t, "is_cuda", False):
        return f"{what} must be a tensor on a HIP device, got {getattr(t, 'device', t)}"
    return f"{what} is on device {t.device.index}, expected device {device}"


def _on_device(t, device):
    return getattr(t, "is_cuda", False) and (t.device.index or 0) == device


def _refuse_gradients(t, what):
    if t.requires_grad and _torch.is_grad_enabled():
        raise ValueError(f"{what} requires gradients: there is no backward pass")
    # Outside of a dual level (-1) no tensor has a tangent to look for.
    if (getattr(_forward_ad, "_current_level", 0) >= 0
            and _forward_ad.unpack_dual(t).tangent is not None):
        raise ValueError(f"{what} has a tangent: there is no forward-mode derivative")


def _rows(t, what, device, dtype=None, shape=None):
    """Checks a [tokens, heads, head_dim] tensor whose last dimension is
    contiguous; returns its address and (token, head) strides."""
    if not _on_device(t, device):
        raise ValueError(_off_device(t, what, device))
    got = t.shape
    if len(got) != 3:
        raise ValueError(f"{what} must be [tokens, heads, head_dim], got {tuple(got)}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{what} must be {dtype}, got {t.dtype}")
    if shape is not None and got != shape:
        raise ValueError(f"{what} must be {tuple(shape)}, got {tuple(got)}")
    _refuse_gradients(t, what)
    token, head, last = t.stride()
    if last != 1 and got[2] != 1:
        raise ValueError(f"{what} must be contiguous in its last dimension")
    return t.data_ptr(), token, head


def _vector(t, what, device, dtypes, n):
    """Checks a contiguous tensor of n elements; returns its address."""
    if not _on_device(t, device):
        raise ValueError(_off_device(t, what, device))
    if t.shape != (n,) or (n > 1 and not t.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous tensor of {n} elements, "
                         f"got {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise ValueError(f"{what} must be one of {', '.join(str(d) for d in dtypes)}, "
                         f"got {t.dtype}")
    return t.data_ptr()


def _weight(t, what, device, dtype, n):
    """(address, type) of a norm's weight."""
    if t is None:
        return 0, 0
    ptr = _vector(t, what, device, (dtype, _torch.float32), n)
    _refuse_gradients(t, what)
    return ptr, _TYPES[t.dtype]


def _rotation(device, inv_freq, positions, tokens, head_dim):
    """(rotary_dim, inv_freq address, positions address, positions are int64)."""
    if inv_freq is None:
        return 0, 0, 0, 0
    n = inv_freq.shape[0] if len(inv_freq.shape) == 1 else -1
    if not 1 <= 2 * n <= head_dim:
        raise ValueError(f"inv_freq must have 1 to {head_dim // 2} elements, "
                         f"got {tuple(inv_freq.shape)}")
    at = _vector(inv_freq, "inv_freq", device, (_torch.float32,), n)
    _refuse_gradients(inv_freq, "inv_freq")
    if positions is None:
        return 2 * n, at, 0, 0
    where = _vector(positions, "positions", device, (_torch.int64, _torch.int32), tokens)
    return 2 * n, at, where, int(positions.dtype == _torch.int64)


@contextlib.contextmanager
def _torch_stream(stream, device):
    if isinstance(stream, _torch.cuda.Stream):
        use = stream
    else:
        ptr = _stream_ptr(stream)
        use = (_torch.cuda.ExternalStream(ptr, device=device) if ptr
               else _torch.cuda.default_stream(device))
    with _torch.cuda.stream(use):
        yield


def _empty(stream, device, shape, dtype):
    """A new tensor from torch's allocator on the call's stream."""
    if stream is None:
        return _torch.empty(shape, dtype=dtype, device=device)
    with _torch_stream(stream, device.index or 0):
        return _torch.empty(shape, dtype=dtype, device=device)


def _result(out, what, like, device, stream):
    """(tensor, address, token stride, head stride) of a result shaped like
    `like`: `out`, or a new one."""
    if out is None:
        _, heads, dim = like.shape
        out = _empty(stream, like.device, like.shape, like.dtype)
        return out, out.data_ptr(), heads * dim, dim
    return (out,) + _rows(out, what, device, like.dtype, like.shape)


def norm_rope(q, k, positions, inv_freq, *, q_weight=None, k_weight=None, eps: float = 1e-6,
              interleaved: bool = False, out_q=None, out_k=None, stream=None) -> Tuple:
    """RMS norm and position rotation of every head of ``q`` and ``k``.

    Args:
      q, k: [tokens, heads, head_dim] of bf16, fp16 or fp32, head_dim up to
        256; any strides but a contiguous last dimension (parts of a fused
        projection). ``k`` may be None.
      positions: int32 or int64 [tokens].
      inv_freq: fp32 [rotary_dim / 2] with rotary_dim <= head_dim; the angle of
        pair i is position * inv_freq[i], exact for positions up to 2^53 before its
        cos and sin are taken in fp32. Dimensions from rotary_dim on are not rotated. None: norm only.
      q_weight, k_weight: [head_dim], of the rows' type or fp32; None: no norm.
      interleaved: pairs are (2i, 2i + 1) instead of (i, i + rotary_dim / 2).
      out_q, out_k: results; the input itself, or apart from the inputs.
        Default: new contiguous tensors.
    Returns (q, k) results, k's None without ``k``.
    """
    torch = _torch or _load_torch()
    if not getattr(q, "is_cuda", False):
        raise ValueError(_off_device(q, "q", 0))
    device = q.device.index or 0
    dtype = q.dtype
    if dtype not in (torch.bfloat16, torch.float16, torch.float32):
        raise ValueError(f"q must be bfloat16, float16 or float32, got {dtype}")
    q_at, q_token, q_head = _rows(q, "q", device)
    shape = q.shape
    tokens, q_heads, dim = shape
    if inv_freq is not None and positions is None:
        raise ValueError("positions are needed with inv_freq")
    k_at = k_token = k_head = k_heads = 0
    if k is not None:
        k_heads = k.shape[1] if len(k.shape) == 3 else 0
        k_at, k_token, k_head = _rows(k, "k", device, dtype, (tokens, k_heads, dim)
                                      if len(k.shape) == 3 else None)
    elif out_k is not None:
        raise ValueError("out_k without k")
    qw_at, qw_type = _weight(q_weight, "q_weight", device, dtype, dim)
    kw_at, kw_type = _weight(k_weight, "k_weight", device, dtype, dim)
    if qw_at and kw_at and qw_type != kw_type:
        raise ValueError("q_weight and k_weight must have the same dtype")
    rotary, inv_at, pos_at, pos_64 = _rotation(device, inv_freq, positions, tokens, dim)
    out_q, qo_at, qo_token, qo_head = _result(out_q, "out_q", q, device, stream)
    ko_at = ko_token = ko_head = 0
    if k is not None:
        out_k, ko_at, ko_token, ko_head = _result(out_k, "out_k", k, device, stream)
    args = _capi.NormRopeArgs.from_buffer_copy(_NORM_ROPE.pack(
        device, _TYPES[dtype], tokens, q_heads, k_heads, dim, rotary, q_at, k_at, qo_at, ko_at,
        q_token, q_head, k_token, k_head, qo_token, qo_head, ko_token, ko_head, qw_at, kw_at,
        qw_type if qw_at else kw_type, pos_64, pos_at, inv_at, eps, interleaved))
    handle = _current_stream(device) if stream is None else _stream_ptr(stream)
    rc = _capi.load().kvx_norm_rope(args, handle)
    if rc:
        _capi.check(rc, "norm_rope")
    return out_q, out_k


def _check_scales(layers, tables, shard_idx, kind, fp4_shape):
    """Checks the types of scale tables, and the shape of a 4-bit cache's (the
    library checks bytes, which bytes in another order would have too)."""
    for layer in tables:
        t = layers[layer][shard_idx]
        if kind == _torch.float8_e4m3fn:
            if t.dtype != _torch.float32:
                raise ValueError("scale tables must be float32")
        elif t.dtype != _torch.float8_e8m0fnu or tuple(t.shape[1:]) != fp4_shape:
            raise ValueError(f"scale tables must be float8_e8m0fnu [blocks, heads, tokens, "
                             f"head_dim / 32] ({fp4_shape}), got {t.dtype} {tuple(t.shape[1:])}")


def _describe_cache(mgr, k_layer, v_layer, shard_idx, dtype):
    """Two of the manager's storages as the fields of kvx_paged_cache; without
    v_layer the keys' alone, without dtype of any type."""
    torch = _torch
    if mgr._device is None:
        raise _capi.KvxError(9, "needs a device-backed KVCacheManagerBase", "KVCacheManager")
    layers = mgr._tensors
    n = mgr.num_kv_layers
    shapes = []
    if v_layer is None:
        v_layer = k_layer
    if dtype is None:
        allowed = "bfloat16, float16"
        types = (torch.bfloat16, torch.float16)
    else:
        allowed, types = dtype, (dtype,)
    for layer in (k_layer, v_layer):
        if not 0 <= layer < n or not 0 <= shard_idx < len(layers[layer]):
            raise _capi.KvxError(11, "layer or shard index out of range", "KVCacheManager")
        t = layers[layer][shard_idx]
        if len(t.shape) != 4:
            raise ValueError("the cache's storages must be [blocks, tokens, heads, head_dim] "
                             "tensors (in 4 bits [blocks, heads, tokens, head_dim / 2]), "
                             f"got {tuple(t.shape)}")
        if t.dtype not in types + (torch.float8_e4m3fn, _FP4):
            raise ValueError(f"the cache must be {allowed}, float8_e4m3fn or float4_e2m1fn_x2, "
                             f"got {t.dtype}")
        shapes.append((t.dtype,) + tuple(t.shape[1:]))
    if shapes[0] != shapes[1]:
        raise ValueError("the key and value storages must have the same type and block shape")
    kind, block_tokens, heads, head_dim = shapes[0]
    if kind == _FP4:
        heads, block_tokens, head_dim = block_tokens, heads, 2 * head_dim
    k_scales = v_scales = 0
    if kind in (torch.float8_e4m3fn, _FP4):
        # Scale tables follow the KV storages, one a storage; other side tables may
        # follow them.
        if len(layers) < 2 * n:
            raise ValueError(f"a {str(kind)[6:]} cache needs one scale table a KV storage "
                             f"({n}), got {len(layers) - n}")
        _check_scales(layers, (n + k_layer, n + v_layer), shard_idx, kind,
                      (heads, block_tokens, head_dim // 32))
        k_scales, v_scales = n + k_layer, n + v_layer
    return (k_layer, v_layer, shard_idx, k_scales, v_scales, _TYPES[kind], block_tokens, heads,
            head_dim)


def _cache(mgr, k_layer, v_layer, shard_idx, dtype):
    """_describe_cache, kept: a manager's storages do not change."""
    try:
        return mgr._paged_caches[k_layer, v_layer, shard_idx, dtype]
    except AttributeError:
        mgr._paged_caches = {}
    except KeyError:
        pass
    found = _describe_cache(mgr, k_layer, v_layer, shard_idx, dtype)
    mgr._paged_caches[k_layer, v_layer, shard_idx, dtype] = found
    return found


def _tables(device, tables):
    """(address, row stride, width) of block tables."""
    if not _on_device(tables, device):
        raise ValueError(_off_device(tables, "tables", device))
    shape = tables.shape
    if len(shape) != 2 or tables.dtype != _torch.int32:
        raise ValueError(f"tables must be an int32 [sequences, blocks] tensor, got "
                         f"{tables.dtype} {tuple(shape)}")
    row, last = tables.stride()
    if last != 1 and shape[1] > 1:
        raise ValueError("tables must be contiguous in their last dimension")
    return tables.data_ptr(), row, shape[1]


def _batch(device, tables, lengths, starts, tokens):
    """The fields of kvx_paged_batch."""
    tables_at, row, width = _tables(device, tables)
    n = tables.shape[0]
    lengths_at = _vector(lengths, "lengths", device, (_torch.int32,), n)
    starts_at = 0
    if starts is not None:
        starts_at = _vector(starts, "starts", device, (_torch.int32,), n + 1)
    elif tokens != n:
        raise ValueError(f"without starts there is one token a sequence: {tokens} tokens, "
                         f"{n} sequences")
    return tables_at, row, width, lengths_at, starts_at, n


def append_kv(mgr, k_layer, v_layer, k, v, tables, lengths, *, starts, inv_freq, positions,
              k_weight, eps, interleaved, shard_idx, stream) -> None:
    _torch or _load_torch()
    device = mgr._device or 0
    k_at, k_token, k_head = _rows(k, "k", device)
    dtype = k.dtype
    cache = _cache(mgr, k_layer, v_layer, shard_idx, dtype)
    tokens, dim = k.shape[0], cache[8]
    shape = (tokens, cache[7], dim)
    if k.shape != shape:
        raise ValueError(f"k must be {shape}, got {tuple(k.shape)}")
    v_at, v_token, v_head = _rows(v, "v", device, dtype, shape)
    batch = _batch(device, tables, lengths, starts, tokens)
    if positions is not None and inv_freq is None:
        raise ValueError("positions without inv_freq")
    rotary, inv_at, pos_at, pos_64 = _rotation(device, inv_freq, positions, tokens, dim)
    w_at, w_type = _weight(k_weight, "k_weight", device, dtype, dim)
    args = _capi.AppendKvArgs.from_buffer_copy(_APPEND_KV.pack(
        *cache, *batch, tokens, _TYPES[dtype], rotary, k_at, v_at, k_token, k_head, v_token, v_head,
        w_at, w_type, pos_64, pos_at, inv_at, eps, interleaved))
    handle = _current_stream(device) if stream is None else _stream_ptr(stream)
    rc = _capi.load().kvx_manager_append_kv(mgr._h, args, handle)
    if rc:
        _capi.check(rc, "KVCacheManager append_kv")


def attend(mgr, k_layer, v_layer, q, tables, lengths, *, starts, group_starts, prefix_lengths,
           scale, causal, out, return_lse, shard_idx, stream):
    torch = _torch or _load_torch()
    device = mgr._device or 0
    q_at, q_token, q_head = _rows(q, "q", device)
    dtype = q.dtype
    cache = _cache(mgr, k_layer, v_layer, shard_idx, dtype)
    shape = q.shape
    tokens, q_heads, dim = shape
    if dim != cache[8]:
        raise ValueError(f"q must have head_dim {cache[8]}, got {dim}")
    batch = _batch(device, tables, lengths, starts, tokens)
    if (group_starts is None) != (prefix_lengths is None):
        raise ValueError("group_starts and prefix_lengths go together")
    groups = groups_at = prefix_at = 0
    if group_starts is not None:
        groups = prefix_lengths.shape[0] if len(prefix_lengths.shape) == 1 else -1
        prefix_at = _vector(prefix_lengths, "prefix_lengths", device, (torch.int32,), groups)
        groups_at = _vector(group_starts, "group_starts", device, (torch.int32,), groups + 1)
    scale = dim ** -0.5 if scale is None else scale
    lib = _capi.load()
    where = "KVCacheManager attend"
    args = _capi.AttendArgs.from_buffer_copy(_ATTEND.pack(
        *cache, *batch, tokens, _TYPES[dtype], q_heads, q_at, 0, q_token, q_head, 0, 0, 0, groups_at,
        prefix_at, groups, not causal, scale, 0, 0, 0))
    need = ctypes.c_int64()
    rc = lib.kvx_manager_attend_workspace(mgr._h, args, need)
    if rc:
        _capi.check(rc, where)
    out, args.out, args.out_token_stride, args.out_head_stride = _result(out, "out", q, device,
                                                                         stream)
    if return_lse:
        lse = _empty(stream, q.device, shape[:2], torch.float32)
        args.lse = lse.data_ptr()
    if need.value:
        workspace = _empty(stream, q.device, need.value, torch.uint8)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need.value
    handle = _current_stream(device) if stream is None else _stream_ptr(stream)
    rc = lib.kvx_manager_attend(mgr._h, args, handle)
    if rc:
        _capi.check(rc, where)
    return (out, lse) if return_lse else out
