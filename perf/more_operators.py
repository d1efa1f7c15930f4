"""The operators that make the paged KV cache smaller, timed at the sizes of a
served model's steps:

* ``append``: keys (normed and rotated on the way) and values of new tokens into
  a pool held in 4 bits (e2m1 codes, one power-of-two scale for 32 neighbouring
  dimensions of a token's head);
* ``attend``: causal attention of a batch over such a pool, one query a sequence
  or many, with or without a prefix that all its sequences share;
* ``weigh``: the attention weight that each cached token got in a step, added to
  a table of what it got before (pools of 16, 8 and 4 bits);
* ``choose``: which tokens of every sequence and key head stay within a budget;
* ``compact``: the kept tokens moved to the front of their sequence, in place.

A case's ``mix`` seeds its lengths, so one case always has the same ones.
"""
import math
import random

import torch

own = False

FP8_MAX = 448.0  # largest e4m3 value
FP4_MAX = 6.0    # largest e2m1 value
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # One decode step of 64 sequences of a Llama-3-8B layer's heads. Launch latency.
        dict(name="append_decode", family="append", sequences=64, tokens=64, heads=8, dim=128,
             block=16, cache="fp4", dtype="bf16", norm=False, longest=4096, mix=1),
        # Prefill chunks of 12 sequences, keys normed and rotated on the way.
        dict(name="append_prefill", family="append", sequences=12, tokens=16384, heads=8, dim=128,
             block=16, cache="fp4", dtype="bf16", norm=True, longest=8192, mix=2),
        # One sequence's decode step: latency.
        dict(name="attend_one", family="attend", sequences=1, tokens=1, q_heads=32, k_heads=8,
             dim=128, block=16, cache="fp4", dtype="bf16", longest=901, shortest=901, prefix=0,
             mix=3),
        # A decode step of 64 sequences of very different lengths: HBM.
        dict(name="attend_decode", family="attend", sequences=64, tokens=64, q_heads=32,
             k_heads=8, dim=128, block=16, cache="fp4", dtype="bf16", longest=16384, shortest=65,
             prefix=0, mix=4),
        # Prefill chunks of 5 sequences against what they hold already: matrix products.
        dict(name="attend_prefill", family="attend", sequences=5, tokens=4099, q_heads=32,
             k_heads=8, dim=128, block=16, cache="fp4", dtype="bf16", longest=12000,
             shortest=2000, prefix=0, mix=5),
        # What each token of 64 sequences got in a decode step, 16-bit pool.
        dict(name="weigh_decode", family="weigh", sequences=64, tokens=64, q_heads=32, k_heads=8,
             dim=128, block=16, cache="same", dtype="bf16", longest=8192, shortest=65, prefix=0,
             decay=1.0, mix=6),
        # The same on one rank of a Llama-3-70B over 8 GPUs (8 query heads on one), 4-bit pool.
        dict(name="weigh_decode_fp4", family="weigh", sequences=128, tokens=128, q_heads=8,
             k_heads=1, dim=128, block=32, cache="fp4", dtype="bf16", longest=16384,
             shortest=300, prefix=0, decay=0.95, mix=7),
        # Prefill chunks: every key against all later queries.
        dict(name="weigh_prefill", family="weigh", sequences=3, tokens=2051, q_heads=32,
             k_heads=8, dim=128, block=16, cache="same", dtype="bf16", longest=9000,
             shortest=1500, prefix=0, decay=1.0, mix=8),
        # One sequence cut to 1024 tokens: latency.
        dict(name="choose_one", family="choose", sequences=1, k_heads=8, block=16, longest=5000,
             shortest=5000, budget=1024, recent=128, prefix=4, mix=9),
        # 64 long sequences cut to 2048 tokens behind a system prompt.
        dict(name="choose_many", family="choose", sequences=64, k_heads=8, block=16,
             longest=16384, shortest=1000, budget=2048, recent=256, prefix=37, mix=10),
        # The rows of 64 such sequences, 16-bit pool.
        dict(name="compact_bf16", family="compact", sequences=64, k_heads=8, dim=128, block=16,
             cache="same", dtype="bf16", longest=8192, shortest=1000, budget=2048, recent=256,
             prefix=0, mix=11),
        # e4m3 pool: rows of blocks with different scales meet in one block.
        dict(name="compact_fp8", family="compact", sequences=24, k_heads=8, dim=128, block=32,
             cache="fp8", dtype="bf16", longest=8192, shortest=3000, budget=3000, recent=64,
             prefix=16, mix=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw_heads(rng):
    k_heads = rng.choice([1, 1, 2, 4, 8, 8])
    return k_heads * rng.choice([1, 2, 4, 4, 5, 8, 16]), k_heads


def _draw_append(rng):
    heads, dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 96, 128, 128, 256])
    sequences = _log_int(rng, 1, 256)
    most = max(2, 16384 * 8 * 128 // (heads * dim) // sequences)
    tokens = sequences if rng.random() < 0.4 else sequences * _log_int(rng, 1, min(4096, most))
    longest = _log_int(rng, 300, 8192)
    while longest > 300 and sequences * longest * heads * dim > 64 * 4096 * 8 * 128:
        longest //= 2
    return dict(family="append", sequences=sequences, tokens=tokens, heads=heads, dim=dim,
                block=rng.choice([8, 16, 16, 32, 64]), cache="fp4",
                dtype=rng.choice(["bf16", "fp16"]), norm=rng.random() < 0.4, longest=longest,
                mix=rng.randrange(1 << 20))


def _draw_step(rng, dims, most_products):
    """Sizes of a batch of queries over a pool."""
    q_heads, k_heads = _draw_heads(rng)
    dim, kind = rng.choice(dims), rng.choice(["one", "one", "some", "many"])
    longest = _log_int(rng, 16, 16384)
    # No more keys and values than the largest decode case holds, and no more
    # products than the prefill case.
    most = max(1, 64 * 4000 * 8 * 128 // (longest * k_heads * dim))
    sequences = _log_int(rng, 1, min(256, most))
    tokens = sequences
    if kind != "one":
        each = _log_int(rng, 2, 16 if kind == "some" else 1024)
        while each > 1 and sequences * each * (longest + 2 * each) * q_heads * dim > most_products:
            each //= 2
        tokens = sequences * each
    prefix = 0
    if kind == "one" and rng.random() < 0.4:
        prefix, longest = _log_int(rng, 64, 16384), min(longest, 1000)
        while prefix > 64 and sequences * prefix * k_heads * dim > 64 * 8000 * 8 * 128:
            prefix //= 2
    return dict(sequences=sequences, tokens=tokens, q_heads=q_heads, k_heads=k_heads, dim=dim,
                block=rng.choice([8, 16, 16, 32, 64]), dtype=rng.choice(["bf16", "fp16"]),
                longest=longest, shortest=rng.randint(1, longest), prefix=prefix,
                mix=rng.randrange(1 << 20))


def _draw_attend(rng):
    case = _draw_step(rng, [64, 96, 128, 128, 256], 4099 * 7000 * 32 * 128)
    return dict(family="attend", cache="fp4", **case)


def _draw_weigh(rng):
    cache = rng.choice(["same", "fp8", "fp4"])
    dims = [64, 96, 128, 256] if cache == "fp4" else [64, 80, 96, 128, 128, 256]
    case = _draw_step(rng, dims, 2051 * 5500 * 32 * 128)
    return dict(family="weigh", cache=cache, decay=rng.choice([0.0, 0.9, 1.0]), **case)


def _draw_cut(rng, most):
    """Sizes of sequences cut to a budget; `most` tokens of all heads."""
    k_heads = rng.choice([1, 1, 2, 4, 8, 8])
    longest = _log_int(rng, 16, 16384)
    sequences = _log_int(rng, 1, max(1, min(256, most // (longest * k_heads))))
    budget = _log_int(rng, 4, longest)
    return dict(sequences=sequences, k_heads=k_heads, block=rng.choice([8, 16, 16, 32, 64]),
                longest=longest, shortest=rng.randint(1, longest), budget=budget,
                recent=rng.choice([0, 1, budget // 8, budget // 2]),
                prefix=rng.choice([0, 0, 4, min(budget // 4, 300)]), mix=rng.randrange(1 << 20))


def _draw_choose(rng):
    return dict(family="choose", **_draw_cut(rng, 64 * 8000 * 8))


def _draw_compact(rng):
    dim, cache = rng.choice([64, 96, 128, 128, 256]), rng.choice(["same", "fp8", "fp4"])
    return dict(family="compact", dim=dim, cache=cache, dtype=rng.choice(["bf16", "fp16"]),
                **_draw_cut(rng, 64 * 4000 * 8 * 128 // dim))


def draw(rng):
    return rng.choice([_draw_append, _draw_attend, _draw_attend, _draw_weigh, _draw_weigh,
                       _draw_choose, _draw_compact])(rng)


def _split(rng, total, parts):
    """`parts` counts of at least 1 that add up to `total`."""
    weights = [rng.random() + 0.2 for _ in range(parts)]
    counts = [1 + int((total - parts) * w / sum(weights)) for w in weights]
    counts[0] += total - sum(counts)
    return counts


def _batch(case):
    """(new tokens, length with them) of every sequence; the prefix is part of
    the length."""
    rng = random.Random(case["mix"])
    new = _split(rng, case.get("tokens", case["sequences"]), case["sequences"])
    lo, hi = case.get("shortest", 0), case["longest"]
    prefix = case.get("prefix", 0)
    return new, [prefix + n + rng.randint(lo, hi) for n in new]


def _inverse_frequencies(rotary):
    return (500000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float().cuda()


def _randn(gen, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return x.mul_(scale).to(dtype)


def _tables(case, seed, lengths, shared):
    """Block tables over a pool whose free ids come in a worked-in allocator's
    order; the first `shared` blocks are the same for every sequence."""
    block = case["block"]
    counts = [(n + block - 1) // block - shared for n in lengths]
    ids = list(range(shared + sum(counts) + 7))
    random.Random(seed).shuffle(ids)
    first, at, rows = ids[:shared], shared, []
    for c in counts:
        rows.append(first + ids[at:at + c])
        at += c
    width = max(map(len, rows))
    table = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32)
    return table.cuda(), len(ids)


# -- the 4-bit format ------------------------------------------------------------------------------

def _fp4_scale_bits(amax, dtype):
    """Exponent (plus 127) of the smallest power of two s with amax <= 7 s: 6 is
    the largest code, and 7 is what rounds to it. Bounded, so that 6 s is finite."""
    bits = (amax.view(torch.int32) + 0x1fffff >> 23) - 2
    return bits.clamp(2, 140 if dtype == torch.float16 else 252)


def _fp4_codes(x, scale):
    """e2m1 codes of x / scale, nearest even."""
    y = (x / scale).abs().clamp_max(FP4_MAX)
    low, mid, high = (y * 2).round(), y.round() + 2, (y / 2).round() + 4
    code = torch.where(y < 2, low, torch.where(y < 4, mid, high)).to(torch.uint8)
    return code + (torch.signbit(x).to(torch.uint8) << 3)


def _fp4_pack(x, dtype):
    """fp32 rows [..., D] as (codes [..., D / 2] in bytes, scales [..., D / 32])."""
    groups = x.unflatten(-1, (-1, 32))
    bits = _fp4_scale_bits(groups.abs().amax(-1), dtype)
    codes = _fp4_codes(groups, (bits << 23).view(torch.float32)[..., None]).flatten(-2)
    return codes[..., 0::2] + (codes[..., 1::2] << 4), bits.to(torch.uint8)


def _fp4_table(dtype):
    """The two values of every byte."""
    one = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device="cuda")
    one = torch.cat((one, -one))
    byte = torch.arange(256, device="cuda")
    return torch.stack((one[byte % 16], one[byte // 16]), -1).to(dtype)


def _fp4_values(codes):
    """Values of the codes, before their scales, as e4m3 (which has them all)."""
    pairs = _fp4_table(torch.float8_e4m3fn).view(torch.int16)[:, 0]
    found = pairs.index_select(0, codes.view(torch.uint8).flatten().int())
    return found.view(torch.float8_e4m3fn).view(*codes.shape[:-1], -1)


def _fp4_rows(codes, scales):
    """Codes and scales of rows, in 32 bits."""
    pairs = _fp4_table(torch.float32).index_select(0, codes.view(torch.uint8).flatten().int())
    x = pairs.view(*codes.shape[:-1], -1, 32)
    return (x * scales.float()[..., None]).flatten(-2)


def _cache(case, gen, blocks, heads):
    """One storage of the pool and, where it has them, its scales."""
    block, dim = case["block"], case["dim"]
    if case["cache"] == "fp4":
        x = torch.randn((blocks, heads, block, dim), generator=gen, device="cuda")
        codes, scales = _fp4_pack(x, DTYPES[case["dtype"]])
        return codes.view(torch.float4_e2m1fn_x2), scales.view(torch.float8_e8m0fnu)
    shape = (blocks, block, heads, dim)
    if case["cache"] != "fp8":
        return _randn(gen, shape, DTYPES[case["dtype"]]), None
    scales = torch.rand(blocks, heads, generator=gen, device="cuda") * 0.004 + 0.004
    values = torch.randn(shape, generator=gen, device="cuda").div_(scales[:, None, :, None])
    return values.clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scales


def _manager(state):
    from __graft_entry__ import load_package
    kvx = load_package()
    scales = [s for s in (state["k_scales"], state["v_scales"]) if s is not None]
    return kvx.KVCacheManager([state["k_cache"], state["v_cache"]], host_blocks_to_allocate=1,
                              scale_tables=scales)


def _prepare_pool(case, gen, seed, heads, shared=0):
    new, lengths = _batch(case)
    tables, blocks = _tables(case, seed, lengths, shared)
    starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    state = dict(case=case, tables=tables, starts=starts, most=max(new),
                 lengths=torch.tensor(lengths, dtype=torch.int32).cuda())
    if case["family"] != "choose":
        state["k_cache"], state["k_scales"] = _cache(case, gen, blocks, heads)
        state["v_cache"], state["v_scales"] = _cache(case, gen, blocks, heads)
        if own:
            state["manager"] = _manager(state)
    elif own:
        from __graft_entry__ import load_package
        state["kvx"] = load_package()
    if case.get("prefix") and case["family"] != "attend":
        state["begins"] = torch.full((case["sequences"],), case["prefix"], dtype=torch.int32,
                                     device="cuda")
    if case["family"] in ("weigh", "choose", "compact"):
        # What tokens got so far: a few got most of it, some nothing at all.
        got = torch.randn((blocks, heads, case["block"]), generator=gen, device="cuda")
        got = got.mul_(1.5).exp_()
        state["weights"] = got.where(got > 0.3, 0.0)
    return state


def _prepare_append(case, gen, seed):
    T, H, D, dtype = case["tokens"], case["heads"], case["dim"], DTYPES[case["dtype"]]
    state = _prepare_pool(case, gen, seed, H)
    # k and v lie behind four query heads a key head in the fused projection.
    fused = _randn(gen, (T, 6 * H, D), dtype)
    state.update(k=fused[:, 4 * H:5 * H], v=fused[:, 5 * H:],
                 inv_freq=_inverse_frequencies(D),
                 k_weight=1 + _randn(gen, (D,), dtype, 0.1) if case["norm"] else None)
    return state


def _prepare_attend(case, gen, seed):
    shared = case["prefix"] // case["block"]
    state = _prepare_pool(case, gen, seed, case["k_heads"], shared)
    state["q"] = _randn(gen, (case["tokens"], case["q_heads"], case["dim"]),
                        DTYPES[case["dtype"]], 1.3)
    state["scale"] = case["dim"] ** -0.5
    if case["prefix"]:
        state["group_starts"] = torch.tensor([0, case["sequences"]], dtype=torch.int32).cuda()
        state["prefix_lengths"] = torch.tensor([shared * case["block"]], dtype=torch.int32).cuda()
    return state


def _prepare_weigh(case, gen, seed):
    state = _prepare_pool(case, gen, seed, case["k_heads"])
    shape = (case["tokens"], case["q_heads"])
    state["q"] = _randn(gen, shape + (case["dim"],), DTYPES[case["dtype"]], 1.3)
    state["scale"] = case["dim"] ** -0.5
    # The log of a sum of exponentials of such scores over what each query sees.
    new, lengths = _batch(case)
    seen = torch.cat([torch.arange(m - n + 1, m + 1) for n, m in zip(new, lengths)])
    state["lse"] = (seen.double().log() + 0.845).float().cuda()[:, None] + _randn(
        gen, shape, torch.float32, 0.1)
    return state


def _prepare_compact(case, gen, seed):
    state = _prepare_pool(case, gen, seed, case["k_heads"])
    state["kept"], _ = _plain_choose(state)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"append": _prepare_append, "attend": _prepare_attend, "weigh": _prepare_weigh,
            "choose": lambda *a: _prepare_pool(*a, case["k_heads"]),
            "compact": _prepare_compact}[case["family"]](case, gen, seed)


# -- the framework's calls -------------------------------------------------------------------------

def _own_append(s):
    case = s["case"]
    s["manager"].append_kv(0, 1, s["k"], s["v"], s["tables"], s["lengths"],
                           starts=None if case["tokens"] == case["sequences"] else s["starts"],
                           inv_freq=s["inv_freq"], k_weight=s["k_weight"], eps=1e-6)
    return _pool(s)


def _own_attend(s):
    case = s["case"]
    more = {}
    if case["tokens"] != case["sequences"]:
        more = dict(starts=s["starts"])
    if case["prefix"]:
        more.update(group_starts=s["group_starts"], prefix_lengths=s["prefix_lengths"])
    return s["manager"].attend(0, 1, s["q"], s["tables"], s["lengths"], scale=s["scale"], **more)


def _own_weigh(s):
    case = s["case"]
    s["manager"].weigh(0, s["q"], s["tables"], s["lengths"], s["lse"], s["weights"],
                       starts=None if case["tokens"] == case["sequences"] else s["starts"],
                       begins=s.get("begins"), decay=case["decay"], scale=s["scale"])
    return s["weights"]


def _own_choose(s):
    case = s["case"]
    return s["kvx"].choose_kept(s["weights"], s["tables"], s["lengths"], case["budget"],
                                recent=case["recent"], begins=s.get("begins"))


def _own_compact(s):
    s["manager"].compact(0, 1, s["kept"], s["tables"], weights=s["weights"])
    return _pool(s) + [s["weights"]]


def _pool(s):
    """The storages and their scales; 4-bit codes as the values they stand for."""
    found = [t for t in (s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"]) if t is not None]
    return [_fp4_values(t) if t.dtype == torch.float4_e2m1fn_x2 else t for t in found]


# -- the plain forms -------------------------------------------------------------------------------

def _plain_norm(x, weight):
    x = x.float()
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()


def _plain_rotate(x, positions, inv_freq):
    angle = (positions.double()[:, None] * inv_freq.double())[:, None]  # far positions need 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    half = inv_freq.numel()
    u, v = x[..., :half], x[..., half:2 * half]
    return torch.cat((u * cos - v * sin, v * cos + u * sin, x[..., 2 * half:]), -1)


def _plain_sequences(s):
    """Sequence and place in it of every new token."""
    starts = s["starts"].long()
    token = torch.arange(s["case"]["tokens"], device="cuda")
    sequence = (token[:, None] >= starts[None, 1:]).sum(1)
    return sequence, token - starts[sequence]


def _plain_append(s):
    starts, lengths, B = s["starts"].long(), s["lengths"].long(), s["case"]["block"]
    sequence, place = _plain_sequences(s)
    position = lengths[sequence] - (starts[sequence + 1] - starts[sequence]) + place
    block, slot = s["tables"][sequence, position // B].long(), position % B
    key = _plain_rotate(_plain_norm(s["k"], s["k_weight"]), position, s["inv_freq"])
    _plain_store(s["k_cache"], s["k_scales"], key, block, slot, s["k"].dtype)
    _plain_store(s["v_cache"], s["v_scales"], s["v"].float(), block, slot, s["v"].dtype)
    return _pool(s)


def _plain_store(cache, scales, x, block, slot, dtype):
    codes, bits = _fp4_pack(x.contiguous(), dtype)
    cache.view(torch.uint8).transpose(1, 2)[block, slot] = codes
    scales.view(torch.uint8).transpose(1, 2)[block, slot] = bits


def _plain_read(cache, scales, blocks):
    """Blocks [..., n] of a storage as [..., kv head, token, dim] in 32 bits."""
    if cache.dtype == torch.float4_e2m1fn_x2:
        codes = cache.view(torch.uint8)[blocks.long()]
        x = _fp4_rows(codes, scales.view(torch.uint8)[blocks.long()].view(torch.float8_e8m0fnu))
        return x.transpose(-4, -3).flatten(-3, -2).contiguous()
    x = cache[blocks.long()].float()
    if scales is not None:
        x = x * scales[blocks.long()][..., None, :, None]
    return x.flatten(-4, -3).transpose(-3, -2).contiguous()


def _plain_rows(s):
    """Scaled queries by sequence and key head, padded to the longest run
    [S, Hk, most * G, D], and where each query's rows are."""
    case = s["case"]
    S, Hk, D, most = case["sequences"], case["k_heads"], case["dim"], s["most"]
    G = case["q_heads"] // Hk
    sequence, place = _plain_sequences(s)
    rows = torch.zeros(S, most, Hk, G, D, device="cuda")
    rows[sequence, place] = (s["q"].float() * s["scale"]).view(-1, Hk, G, D)
    return rows.transpose(1, 2).reshape(S, Hk, most * G, D), sequence, place


def _plain_hidden(s, first, count):
    """Which of the positions first + [0, count) each query may not see:
    [S, 1, most * G, count]."""
    G = s["case"]["q_heads"] // s["case"]["k_heads"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    place = torch.arange(s["most"], device="cuda")
    last = (lengths - starts[1:] + starts[:-1])[:, None] + place  # position of each query
    j = torch.arange(count, device="cuda") + first
    hidden = j[None, None] > torch.minimum(last, lengths[:, None] - 1)[..., None]
    return hidden.repeat_interleave(G, 1)[:, None]


def _plain_attend(s):
    case = s["case"]
    S, Hk, D, B, most = (case["sequences"], case["k_heads"], case["dim"], case["block"], s["most"])
    G, shared = case["q_heads"] // Hk, case["prefix"] // case["block"]
    rows, sequence, place = _plain_rows(s)
    keys = _plain_read(s["k_cache"], s["k_scales"], s["tables"][:, shared:])
    values = _plain_read(s["v_cache"], s["v_scales"], s["tables"][:, shared:])
    scores = torch.matmul(rows, keys.transpose(-1, -2).contiguous())
    scores = scores.masked_fill_(_plain_hidden(s, shared * B, keys.shape[2]), -math.inf)
    if shared:
        # Every sequence's rows against the shared blocks at once.
        first_keys = _plain_read(s["k_cache"], s["k_scales"], s["tables"][0, :shared])
        first_values = _plain_read(s["v_cache"], s["v_scales"], s["tables"][0, :shared])
        together = rows.transpose(0, 1).reshape(Hk, S * most * G, D)
        ahead = torch.matmul(together, first_keys.transpose(-1, -2).contiguous())
        ahead = ahead.view(Hk, S, most * G, -1).transpose(0, 1)
        top = torch.maximum(scores.amax(-1, keepdim=True), ahead.amax(-1, keepdim=True))
        scores, ahead = (scores - top).exp(), (ahead - top).exp()
        total = scores.sum(-1, keepdim=True) + ahead.sum(-1, keepdim=True)
        flat = ahead.transpose(0, 1).reshape(Hk, S * most * G, -1)
        more = torch.matmul(flat, first_values).view(Hk, S, most * G, D).transpose(0, 1)
        out = (torch.matmul(scores, values) + more) / total
    else:
        scores = (scores - scores.amax(-1, keepdim=True)).exp_()
        out = torch.matmul(scores, values) / scores.sum(-1, keepdim=True)
    out = out.view(S, Hk, most, G, D).transpose(1, 2)[sequence, place]
    return out.reshape(-1, case["q_heads"], D).to(s["q"].dtype)


def _plain_places(s, width):
    """Block and slot of positions [0, width) of every sequence, [S, width]."""
    j = torch.arange(width, device="cuda")
    return s["tables"].long()[:, j // s["case"]["block"]], (j % s["case"]["block"]).expand(
        s["tables"].shape[0], -1)


def _plain_weigh(s):
    case = s["case"]
    S, Hk, G, most = (case["sequences"], case["k_heads"],
                      case["q_heads"] // case["k_heads"], s["most"])
    rows, sequence, place = _plain_rows(s)
    lse = torch.full((S, most, Hk, G), math.inf, device="cuda")
    lse[sequence, place] = s["lse"].view(-1, Hk, G)
    lse = lse.transpose(1, 2).reshape(S, Hk, most * G, 1)
    keys = _plain_read(s["k_cache"], s["k_scales"], s["tables"])
    scores = torch.matmul(rows, keys.transpose(-1, -2).contiguous())
    scores = scores.masked_fill_(_plain_hidden(s, 0, keys.shape[2]), -math.inf)
    got = scores.sub_(lse).exp_().sum(2).transpose(1, 2)  # [S, width, Hk]
    block, slot = _plain_places(s, keys.shape[2])
    lengths, j = s["lengths"].long()[:, None], torch.arange(keys.shape[2], device="cuda")
    old = lengths - (s["starts"][1:] - s["starts"][:-1]).long()[:, None]
    before = s["weights"][block, :, slot] * case["decay"]
    got = got + torch.where((j < old)[..., None], before, 0.0)
    mine = j < lengths
    if "begins" in s:
        mine = mine & (j >= s["begins"][:, None])
    block, slot = block[mine], slot[mine]
    s["weights"][block, :, slot] = got[mine]
    return s["weights"]


def _plain_choose(s):
    case, lengths = s["case"], s["lengths"].long()
    S, Hk, budget = case["sequences"], case["k_heads"], case["budget"]
    width = s["tables"].shape[1] * case["block"]
    block, slot = _plain_places(s, width)
    w = s["weights"][block, :, slot].transpose(1, 2)  # [S, Hk, width]
    j = torch.arange(width, device="cuda")
    first = torch.minimum(s["begins"].long(), lengths) if "begins" in s else lengths * 0
    first = first.clamp_max(budget)
    recent = (budget - first).clamp_max(case["recent"])
    held = (j < first[:, None]) | (j >= (lengths - recent)[:, None]) | (lengths <= budget)[:, None]
    there = (j < lengths[:, None])[:, None]
    rank = torch.where(held[:, None], math.inf, w).where(there, -math.inf)
    order = rank.sort(dim=-1, descending=True, stable=True).indices[..., :budget]
    inside = torch.arange(order.shape[-1], device="cuda") < lengths.clamp_max(budget)[:, None, None]
    kept = order.where(inside, width).sort(-1).values
    kept = torch.where(kept < width, kept, -1).int()
    if kept.shape[-1] < budget:
        kept = torch.cat((kept, kept.new_full((S, Hk, budget - kept.shape[-1]), -1)), -1)
    return kept, lengths.clamp_max(budget).int()


def _plain_move_fp8(s, cache, scales, block, slot, to, to_slot, head, moves):
    """Rows of blocks with different scales: the block that they go to gets the
    largest of their scales, and their codes are stored again under it."""
    B, n = s["case"]["block"], block.shape[-1]
    old = torch.where(moves[1], scales[block, head], 0.0)
    wide = torch.nn.functional.pad(old, (0, -n % B)).unflatten(-1, (-1, B))
    new = wide.amax(-1).repeat_interleave(B, -1)[..., :n]
    # Blocks whose rows all stay keep their scale.
    some = torch.nn.functional.pad(moves[0], (0, -n % B)).unflatten(-1, (-1, B)).any(-1)
    some = some.repeat_interleave(B, -1)[..., :n] & moves[1]
    ratio = torch.where(new > 0, old / new, 1.0)
    rows = cache[block, slot, head].float() * ratio[..., None]
    cache[to[some], to_slot[some], head[some]] = rows[some].to(cache.dtype)
    scales[to[some], head[some]] = new[some]


def _plain_move(cache, block, slot, to, to_slot, head, moves):
    """Rows of a storage [blocks, heads, tokens, ...] to their places."""
    rows = cache[block, head, slot]
    cache[to[moves], head[moves], to_slot[moves]] = rows[moves]


def _plain_compact(s):
    case, kept = s["case"], s["kept"].long()
    S, Hk, n = kept.shape
    there = kept >= 0
    tables = s["tables"].long()[:, None].expand(-1, Hk, -1)
    source = kept.clamp_min(0)
    block, slot = tables.gather(2, source // case["block"]), source % case["block"]
    place = torch.arange(n, device="cuda").expand(S, Hk, n)
    inside = (place // case["block"]).clamp_max(tables.shape[2] - 1)
    to, to_slot = tables.gather(2, inside), place % case["block"]
    head = torch.arange(Hk, device="cuda")[None, :, None].expand(S, Hk, n)
    moved = there & (source != place)
    at = (block, slot, to, to_slot, head)
    for cache, scales in ((s["k_cache"], s["k_scales"]), (s["v_cache"], s["v_scales"])):
        if case["cache"] == "fp8":
            _plain_move_fp8(s, cache, scales, *at, (moved, there))
        elif case["cache"] == "fp4":
            _plain_move(cache.view(torch.uint8), *at, moved)
            _plain_move(scales.view(torch.uint8), *at, moved)
        else:
            _plain_move(cache.transpose(1, 2), *at, moved)
    _plain_move(s["weights"], *at, moved)
    return _pool(s) + [s["weights"]]


def run(state):
    if own:
        return {"append": _own_append, "attend": _own_attend, "weigh": _own_weigh,
                "choose": _own_choose, "compact": _own_compact}[state["case"]["family"]](state)
    return {"append": _plain_append, "attend": _plain_attend, "weigh": _plain_weigh,
            "choose": _plain_choose, "compact": _plain_compact}[state["case"]["family"]](state)


# -- 64 bits, from the definitions -----------------------------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_fp4(x, dtype):
    """(values before the scale, scales) of rows [..., D]."""
    groups = x.unflatten(-1, (-1, 32))
    largest = groups.abs().amax(-1)
    low, high = -125, (13 if dtype == torch.float16 else 125)
    exponent = torch.ceil(torch.log2(largest / 7)).nan_to_num(low, low, low).clamp(low, high)
    exponent = exponent + (largest > 7 * 2.0 ** exponent).double()  # where the logarithm was rounded
    exponent = exponent - (largest <= 3.5 * 2.0 ** exponent).double()
    scale = 2.0 ** exponent.clamp(low, high)
    y = groups / scale[..., None]
    values = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    # A value in the middle between two goes to the one whose last bit is 0.
    middles, i = (values[1:] + values[:-1]) / 2, torch.zeros_like(y)
    for n, m in enumerate(middles.tolist()):
        i += (y.abs() > m) if n % 2 == 0 else (y.abs() >= m)
    return (values[i.long()] * torch.where(torch.signbit(y), -1.0, 1.0)).flatten(-2), scale


def _exact_decode(cache):
    b = cache.view(torch.uint8).long()
    both = torch.stack((b & 15, b >> 4), -1).flatten(-2)
    values = torch.tensor(_E2M1, dtype=torch.float64, device=b.device)
    return values[both & 7] * (1 - 2 * (both >> 3)).double()


def _exact_keys(x, weight, positions, inv_freq):
    """Norm and rotation as a complex product."""
    y = x.double()
    if weight is not None:
        y = y / ((y ** 2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * weight.double()
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"),
                       torch.outer(positions.double(), inv_freq.double()))[:, None]
    half = inv_freq.numel()
    pairs = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
    return torch.cat((pairs.real, pairs.imag, y[..., 2 * half:]), -1)


def _exact_append(case, s):
    new, lengths = _batch(case)
    B, table, blocks, slots, positions = case["block"], s["tables"].tolist(), [], [], []
    for i, (n, m) in enumerate(zip(new, lengths)):
        for p in range(m - n, m):
            blocks.append(table[i][p // B])
            slots.append(p % B)
            positions.append(p)
    b, t = torch.tensor(blocks).cuda(), torch.tensor(slots).cuda()
    key = _exact_keys(s["k"], s["k_weight"], torch.tensor(positions).cuda(), s["inv_freq"])
    outs, tables = [], []
    for cache, scales, x in ((s["k_cache"], s["k_scales"], key),
                             (s["v_cache"], s["v_scales"], s["v"].double())):
        values, sizes = _exact_fp4(x, s["k"].dtype)
        pool, table = _exact_decode(cache), scales.double()
        for h in range(case["heads"]):
            pool[b, h, t] = values[:, h]
            table[b, h, t] = sizes[:, h]
        outs.append(pool)
        tables.append(table)
    return outs + tables


def _exact_sequence(case, s, cache, scales, i, length):
    """Tokens [0, length) of sequence i, [length, heads, dim] in 64 bits."""
    B = case["block"]
    ids = s["tables"][i, :(length + B - 1) // B].long()
    if case["cache"] == "fp4":
        sizes = 2.0 ** (scales.view(torch.uint8)[ids].double() - 127)
        x = _exact_decode(cache.view(torch.uint8)[ids]) * sizes.repeat_interleave(32, -1)
        return x.transpose(1, 2).flatten(0, 1)[:length]
    x = cache[ids].double()
    if scales is not None:
        x = x * scales[ids].double()[:, None, :, None]
    return x.flatten(0, 1)[:length]


def _exact_attend(case, s):
    new, lengths = _batch(case)
    G, begin, outs = case["q_heads"] // case["k_heads"], 0, []
    for i, n in enumerate(new):
        k = _exact_sequence(case, s, s["k_cache"], s["k_scales"], i, lengths[i])
        v = _exact_sequence(case, s, s["v_cache"], s["v_scales"], i, lengths[i])
        q = s["q"][begin:begin + n].double()
        seen = (torch.arange(lengths[i], device="cuda")[None]
                <= torch.arange(lengths[i] - n, lengths[i], device="cuda")[:, None])
        heads = []
        for h in range(case["q_heads"]):
            weight = q[:, h] @ k[:, h // G].t().contiguous() * s["scale"]
            weight = torch.softmax(weight.masked_fill(~seen, -math.inf), -1)
            heads.append(weight @ v[:, h // G])
        outs.append(torch.stack(heads, 1))
        begin += n
    return torch.cat(outs)


def _exact_weigh(case, s):
    new, lengths = _batch(case)
    G, B, begin = case["q_heads"] // case["k_heads"], case["block"], 0
    table = s["weights"].double()
    for i, (n, m) in enumerate(zip(new, lengths)):
        k = _exact_sequence(case, s, s["k_cache"], s["k_scales"], i, m)
        q, lse = s["q"][begin:begin + n].double(), s["lse"][begin:begin + n].double()
        seen = (torch.arange(m, device="cuda")[None]
                <= torch.arange(m - n, m, device="cuda")[:, None])
        p = torch.arange(case["prefix"], m, device="cuda")
        b, t = s["tables"][i].long()[p // B], p % B
        for h in range(case["k_heads"]):
            got = torch.zeros(m, dtype=torch.float64, device="cuda")
            for g in range(h * G, h * G + G):
                score = q[:, g] @ k[:, h].t().contiguous() * s["scale"] - lse[:, g:g + 1]
                got += torch.where(seen, score.exp(), 0.0).sum(0)
            before = table[b, h, t] * case["decay"]
            table[b, h, t] = got[case["prefix"]:] + torch.where(p < m - n, before, 0.0)
        begin += n
    return table


def _exact_compact(case, s):
    kept, tables, B = s["kept"].tolist(), s["tables"].tolist(), case["block"]
    source, target, rows = [], [], []  # (block, slot, head), and number of the block written
    for i, of_head in enumerate(kept):
        for h, places in enumerate(of_head):
            first = next((p for p, k in enumerate(places) if k != p), len(places))
            for p, k in enumerate(places):
                if k >= 0 and p // B >= first // B:
                    source.append((tables[i][k // B], k % B, h))
                    target.append((tables[i][p // B], p % B, h))
    if not source:
        source = target = [(0, 0, 0)]
    (b, t, h), (c, u, _) = (torch.tensor(x, device="cuda").t() for x in (source, target))
    moved = [s["weights"].double()]
    moved[0][c, h, u] = s["weights"].double()[b, h, t]
    pools, scale_tables = [], []
    for cache, scales in ((s["k_cache"], s["k_scales"]), (s["v_cache"], s["v_scales"])):
        if case["cache"] == "fp4":
            pool, old = _exact_decode(cache), scales.double()
            table = old.clone()
            table[c, h, u] = old[b, h, t]
            pool[c, h, u] = _exact_decode(cache)[b, h, t]
        elif case["cache"] == "fp8":
            old, pool = scales.double(), cache.double()
            at = c * old.shape[1] + h
            table = old.clone().flatten()
            largest = torch.zeros_like(table).scatter_reduce_(0, at, old[b, h], "amax")
            table[at] = largest[at]
            table = table.view_as(old)
            again = pool[b, t, h] * (old[b, h] / table[c, h])[:, None]
            pool[c, u, h] = again.to(torch.float8_e4m3fn).double()
        else:
            pool, table = cache.double(), None
            pool[c, u, h] = cache.double()[b, t, h]
        pools.append(pool)
        if table is not None:
            scale_tables.append(table)
    return pools + scale_tables + moved


def exact(case, seed):
    if case["family"] == "choose":
        return None  # whole numbers
    return {"append": _exact_append, "attend": _exact_attend, "weigh": _exact_weigh,
            "compact": _exact_compact}[case["family"]](case, prepare(case, seed))


# -- what a pass cannot do without -----------------------------------------------------------------

def _row_bytes(case):
    """Bytes of one token's head in a storage, a block's scale shared out."""
    D = case["dim"]
    return {"same": 2 * D, "fp8": D + 4 / case["block"], "fp4": D // 2 + D // 32}[case["cache"]]


def work(case):
    new, lengths = _batch(case)
    B, prefix = case["block"], case.get("prefix", 0)
    if case["family"] == "append":
        values = 2 * case["tokens"] * case["heads"] * case["dim"]
        touched = sum((m - 1) // B - (m - n) // B + 1 for n, m in zip(new, lengths))
        held = 2 * case["tokens"] * case["heads"] * _row_bytes(case)
        return {"bytes": values * 2 + held + 4 * touched, "flops": 6 * values}
    H = case["k_heads"]
    if case["family"] in ("choose", "compact"):
        first = min(prefix, case["budget"])
        recent = min(case["recent"], case["budget"] - first)
        cut = [m for m in lengths if m > case["budget"]]
        if case["family"] == "choose":
            read = sum(m - first - recent for m in cut) * H
            return {"bytes": 4 * (read + len(lengths) * (case["budget"] * H + 1)), "flops": read}
        rows = len(cut) * (case["budget"] - first) * H
        each = 2 * (2 * _row_bytes(case) + 4) + 4
        return {"bytes": max(rows, 1) * each + 4 * sum(lengths) // B, "flops": 0}
    D, T = case["dim"], case["tokens"]
    seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, lengths))
    if case["family"] == "weigh":
        keys = sum(lengths)
        table = sum(m - min(prefix, m) for m in lengths) * H * (4 if case["decay"] == 0 else 8)
        return {"bytes": keys * H * _row_bytes(case) + table + 4 * (keys // B)
                         + T * case["q_heads"] * (2 * D + 4),
                "flops": 2 * seen * case["q_heads"] * D}
    keys = prefix + sum(m - prefix for m in lengths)
    return {"bytes": 2 * keys * H * _row_bytes(case) + 4 * (keys // B)
                     + 4 * T * case["q_heads"] * D,
            "flops": 4 * seen * case["q_heads"] * D}
