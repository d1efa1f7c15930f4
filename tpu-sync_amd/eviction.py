"""Operators that make the paged KV cache shorter: what attention each cached token
got, which tokens stay within a budget, and their move to the front of their
sequences. A served loop weighs its steps and cuts sequences when they have grown;
every layer is cut from the same lengths, and the new ones hold for all of them after
that:

    for i in range(layers):  # a step
        out, lse = mgr.attend(2 * i, 2 * i + 1, q, tables, lengths, return_lse=True)
        mgr.weigh(2 * i, q, tables, lengths, lse, weights[i])

    for i in range(layers):  # now and then
        cut = mgr.evict(2 * i, 2 * i + 1, weights[i], tables, lengths, 2048, recent=256)
    lengths = cut

Streams, memory, graphs and gradients are as in ``paged_attention``.
"""
import ctypes
import operator
import struct
from typing import Tuple

from . import _capi, paged_attention as base
from .kv_cache_manager import _stream_ptr

_WEIGH = struct.Struct(base._CACHE + base._BATCH + "q2iQ2q2QqQi2fiQqQ")
_CHOOSE = struct.Struct("4iqQ" + base._BATCH + "3Q2q")
_COMPACT = struct.Struct(base._CACHE + "Q3qQ4qQq")
for _pack, _args in ((_WEIGH, _capi.WeighArgs), (_CHOOSE, _capi.ChooseKeptArgs),
                     (_COMPACT, _capi.CompactArgs)):
    assert _pack.size == ctypes.sizeof(_args)


def _weights(t, device, blocks=None, heads=None, block_tokens=None):
    """Checks a table [blocks, heads, tokens] of weights; returns its address and
    number of blocks."""
    torch = base._torch
    if not base._on_device(t, device):
        raise ValueError(base._off_device(t, "weights", device))
    if t.dtype != torch.float32 or len(t.shape) != 3 or not t.is_contiguous():
        raise ValueError("weights must be a contiguous float32 [blocks, heads, tokens] tensor, "
                         f"got {t.dtype} {tuple(t.shape)}")
    base._refuse_gradients(t, "weights")
    if heads is not None and (tuple(t.shape[1:]) != (heads, block_tokens) or t.shape[0] < blocks):
        raise ValueError(f"weights must be [{blocks}, {heads}, {block_tokens}] as the cache, "
                         f"got {tuple(t.shape)}")
    return t.data_ptr(), t.shape[0]


def _positions(t, what, device, sequences):
    if t is None:
        return 0
    return base._vector(t, what, device, (base._torch.int32,), sequences)


def _count(value, what):
    try:
        value = None if isinstance(value, bool) else operator.index(value)
    except TypeError:
        value = None
    if value is None:
        raise ValueError(f"{what} must be an int")
    if not 0 <= value <= 1 << 30:
        raise ValueError(f"{what} must be 0..2^30, got {value}")
    return value


def weigh(mgr, k_layer, q, tables, lengths, lse, weights, *, starts, begins, weighed, decay, scale,
          causal, shard_idx, stream) -> None:
    torch = base._torch or base._load_torch()
    device = mgr._device or 0
    q_at, q_token, q_head = base._rows(q, "q", device)
    cache = base._cache(mgr, k_layer, None, shard_idx, q.dtype)
    tokens, q_heads, dim = q.shape
    if dim != cache[8]:
        raise ValueError(f"q must have head_dim {cache[8]}, got {dim}")
    batch = base._batch(device, tables, lengths, starts, tokens)
    if not base._on_device(lse, device):
        raise ValueError(base._off_device(lse, "lse", device))
    if lse.dtype != torch.float32 or lse.shape != q.shape[:2] or not lse.is_contiguous():
        raise ValueError(f"lse must be a contiguous float32 {tuple(q.shape[:2])} tensor, got "
                         f"{lse.dtype} {tuple(lse.shape)}")
    base._refuse_gradients(lse, "lse")
    blocks = mgr._tensors[k_layer][shard_idx].shape[0]
    weights_at, table_blocks = _weights(weights, device, blocks, cache[7], cache[6])
    args = _capi.WeighArgs.from_buffer_copy(_WEIGH.pack(
        *cache, *batch, tokens, base._TYPES[q.dtype], q_heads, q_at, q_token, q_head,
        lse.data_ptr(), weights_at, table_blocks, _positions(begins, "begins", device, batch[5]),
        not causal, dim ** -0.5 if scale is None else scale, decay, 0, 0, 0,
        _positions(weighed, "weighed", device, batch[5])))
    lib = _capi.load()
    if starts is not None or q_heads > 32 * cache[7]:  # single tokens need no workspace
        need = ctypes.c_int64()
        rc = lib.kvx_manager_weigh_workspace(mgr._h, args, need)
        if rc:
            _capi.check(rc, "KVCacheManager weigh")
        if need.value:
            workspace = base._empty(stream, q.device, need.value, torch.uint8)
            args.workspace, args.workspace_bytes = workspace.data_ptr(), need.value
    handle = base._current_stream(device) if stream is None else _stream_ptr(stream)
    rc = lib.kvx_manager_weigh(mgr._h, args, handle)
    if rc:
        _capi.check(rc, "KVCacheManager weigh")


def choose_kept(weights, tables, lengths, budget: int, *, recent: int = 0, begins=None,
                stream=None) -> Tuple:
    """The tokens of every sequence and key head that stay within ``budget``.

    Of a sequence that holds more, the first ``begins[s]`` tokens stay (a shared
    prefix, or the ones that every query attends to), the last ``recent`` ones,
    and of the others those with the largest weights, the earlier one where two
    are equal. (NaN counts as less than any number.) Where they do not all fit,
    the first ones go before the recent ones. Tokens that have not been weighed
    should be among the recent ones: their entries are another token's.

    Args:
      weights: float32 [blocks, heads, tokens], as ``KVCacheManager.weigh`` keeps.
      tables, lengths: int32 [sequences, blocks] and [sequences], as in
        ``KVCacheManager.attend``.
      begins: int32 [sequences]; None: 0.
    Returns (kept, lengths): int32 [sequences, heads, budget] positions,
    ascending, -1 behind the tokens of a shorter sequence, and int32 [sequences],
    what each one holds then.
    """
    torch = base._torch or base._load_torch()
    if not getattr(weights, "is_cuda", False):
        raise ValueError(base._off_device(weights, "weights", 0))
    device = weights.device.index or 0
    weights_at, blocks = _weights(weights, device)
    _, heads, block_tokens = weights.shape
    base._tables(device, tables)
    sequences = tables.shape[0]
    batch = base._batch(device, tables, lengths, None, sequences)
    budget, recent = _count(budget, "budget"), _count(recent, "recent")
    begins_at = _positions(begins, "begins", device, sequences)
    kept = base._empty(stream, weights.device, (sequences, heads, budget), torch.int32)
    cut = base._empty(stream, weights.device, (sequences,), torch.int32)
    args = _capi.ChooseKeptArgs.from_buffer_copy(_CHOOSE.pack(
        device, heads, block_tokens, 0, blocks, weights_at, *batch, begins_at, kept.data_ptr(),
        cut.data_ptr(), budget, recent))
    handle = base._current_stream(device) if stream is None else _stream_ptr(stream)
    rc = _capi.load().kvx_choose_kept(args, handle)
    if rc:
        _capi.check(rc, "choose_kept")
    return kept, cut


def compact(mgr, k_layer, v_layer, kept, tables, *, weights, shard_idx, stream) -> None:
    torch = base._torch or base._load_torch()
    device = mgr._device or 0
    cache = base._cache(mgr, k_layer, v_layer, shard_idx, None)
    if not base._on_device(kept, device):
        raise ValueError(base._off_device(kept, "kept", device))
    if kept.dtype != torch.int32 or len(kept.shape) != 3 or kept.shape[1] != cache[7]:
        raise ValueError(f"kept must be an int32 [sequences, {cache[7]}, budget] tensor, got "
                         f"{kept.dtype} {tuple(kept.shape)}")
    sequences, _, budget = kept.shape
    tables_at, row, width = base._tables(device, tables)
    if tables.shape[0] != sequences:
        raise ValueError(f"tables must have {sequences} sequences, got {tables.shape[0]}")
    weights_at = blocks = 0
    if weights is not None:
        blocks = mgr._tensors[k_layer][shard_idx].shape[0]
        weights_at, blocks = _weights(weights, device, blocks, cache[7], cache[6])
    args = _capi.CompactArgs.from_buffer_copy(_COMPACT.pack(
        *cache, tables_at, row, width, sequences, kept.data_ptr(), *kept.stride(), budget, weights_at,
        blocks))
    handle = base._current_stream(device) if stream is None else _stream_ptr(stream)
    rc = _capi.load().kvx_manager_compact(mgr._h, args, handle)
    if rc:
        _capi.check(rc, "KVCacheManager compact")
