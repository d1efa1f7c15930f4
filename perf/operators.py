"""The operators that fill and read the paged KV pool, timed at the sizes of a
served model's steps:

* ``norm_rope``: RMS norm of every query and key head and the position
  rotation, in one pass;
* ``append``: keys (normed and rotated on the way) and values of new tokens
  into the blocks of the pool, quantised per (block, head) in an e4m3 pool;
* ``attend``: causal attention of a batch over the pool, one query a sequence
  or many, with or without a prefix that all its sequences share.

A case's ``mix`` seeds its lengths, so one case always has the same ones.
"""
import math
import random

import torch

own = False

FP8_MAX = 448.0  # largest e4m3 value
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One decode step of 64 sequences: heads of a Llama-3-8B layer. Launch latency.
        dict(name="norm_rope_decode", family="norm_rope", tokens=64, q_heads=32, k_heads=8,
             dim=128, rotary=128, dtype="bf16", norm=True, interleaved=False, far=120000),
        # Prefill of 8192 tokens of the same layer, q and k views of one fused projection.
        dict(name="norm_rope_prefill", family="norm_rope", tokens=8192, q_heads=32, k_heads=8,
             dim=128, rotary=128, dtype="bf16", norm=True, interleaved=False, far=32000),
        # Rotation of neighbouring pairs of part of an 80-wide head, no norm, odd count.
        dict(name="norm_rope_partial", family="norm_rope", tokens=4001, q_heads=16, k_heads=16,
             dim=80, rotary=32, dtype="fp16", norm=False, interleaved=True, far=5000),
        # The new token of each of 64 sequences into 16-token blocks.
        dict(name="append_decode", family="append", sequences=64, tokens=64, heads=8, dim=128,
             block=16, cache="same", dtype="bf16", norm=False, longest=4096, mix=1),
        # Prefill chunks of 12 sequences, keys normed and rotated on the way.
        dict(name="append_prefill", family="append", sequences=12, tokens=16384, heads=8, dim=128,
             block=16, cache="same", dtype="bf16", norm=True, longest=8192, mix=2),
        # The decode step of an e4m3 pool: the block's scale may grow.
        dict(name="append_fp8_decode", family="append", sequences=96, tokens=96, heads=8, dim=128,
             block=16, cache="fp8", dtype="bf16", norm=False, longest=4096, mix=3),
        # Prefill chunks into an e4m3 pool.
        dict(name="append_fp8_prefill", family="append", sequences=9, tokens=8201, heads=8,
             dim=128, block=32, cache="fp8", dtype="bf16", norm=False, longest=6000, mix=4),
        # One sequence's decode step: latency.
        dict(name="attend_one", family="attend", sequences=1, tokens=1, q_heads=32, k_heads=8,
             dim=128, block=16, cache="same", dtype="bf16", longest=700, shortest=700, prefix=0,
             mix=5),
        # A decode step of 64 sequences of very different lengths: HBM.
        dict(name="attend_decode", family="attend", sequences=64, tokens=64, q_heads=32,
             k_heads=8, dim=128, block=16, cache="same", dtype="bf16", longest=8192, shortest=65,
             prefix=0, mix=6),
        # One rank of a Llama-3-70B over 8 GPUs (8 query heads on one KV head), e4m3 pool.
        dict(name="attend_decode_fp8", family="attend", sequences=128, tokens=128, q_heads=8,
             k_heads=1, dim=128, block=32, cache="fp8", dtype="bf16", longest=16384,
             shortest=300, prefix=0, mix=7),
        # 128 sequences on one long prompt, each with a few hundred tokens of its own.
        dict(name="attend_shared_prefix", family="attend", sequences=128, tokens=128, q_heads=32,
             k_heads=8, dim=128, block=16, cache="same", dtype="bf16", longest=700, shortest=33,
             prefix=16000, mix=8),
        # Prefill chunks of 5 sequences against what they hold already: matrix products.
        dict(name="attend_prefill", family="attend", sequences=5, tokens=4099, q_heads=32,
             k_heads=8, dim=128, block=16, cache="same", dtype="bf16", longest=12000,
             shortest=2000, prefix=0, mix=9),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _draw_heads(rng):
    k_heads = rng.choice([1, 1, 2, 4, 8, 8])
    return k_heads * rng.choice([1, 2, 4, 4, 5, 8, 16]), k_heads


def _draw_norm_rope(rng):
    q_heads, k_heads = _draw_heads(rng)
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    most = max(1, 8192 * 40 * 128 // ((q_heads + k_heads) * dim))
    return dict(family="norm_rope", tokens=_log_int(rng, 1, min(16384, most)), q_heads=q_heads,
                k_heads=k_heads, dim=dim, rotary=rng.choice([dim, dim, dim // 2]),
                dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]), norm=rng.random() < 0.6,
                interleaved=rng.random() < 0.3, far=_log_int(rng, 1000, 1000000))


def _draw_append(rng):
    heads, dim = rng.choice([1, 2, 4, 8, 8]), rng.choice([64, 80, 96, 128, 128, 256])
    sequences = _log_int(rng, 1, 256)
    most = max(2, 16384 * 8 * 128 // (heads * dim) // sequences)
    tokens = sequences if rng.random() < 0.4 else sequences * _log_int(rng, 1, min(4096, most))
    return dict(family="append", sequences=sequences, tokens=tokens, heads=heads, dim=dim,
                block=rng.choice([8, 16, 16, 32, 64]),
                cache=rng.choice(["same", "same", "fp8"]), dtype=rng.choice(["bf16", "fp16"]),
                norm=rng.random() < 0.4, longest=_log_int(rng, 500, 8192),
                mix=rng.randrange(1 << 20))


def _draw_attend(rng):
    q_heads, k_heads = _draw_heads(rng)
    dim, kind = rng.choice([64, 80, 96, 128, 128, 256]), rng.choice(["one", "one", "some", "many"])
    longest = _log_int(rng, 16, 16384)
    # No more keys and values than the largest decode case holds, and no more
    # products than the prefill case.
    most = max(1, 64 * 4000 * 8 * 128 // (longest * k_heads * dim))
    sequences = _log_int(rng, 1, min(256, most))
    tokens = sequences
    if kind != "one":
        each = _log_int(rng, 2, 16 if kind == "some" else 1024)
        while each > 1 and (sequences * each * (longest + 2 * each) * q_heads * dim
                            > 4099 * 7000 * 32 * 128):
            each //= 2
        tokens = sequences * each
    prefix = 0
    if kind == "one" and rng.random() < 0.4:
        prefix, longest = _log_int(rng, 64, 16384), min(longest, 1000)
    return dict(family="attend", sequences=sequences, tokens=tokens, q_heads=q_heads,
                k_heads=k_heads, dim=dim, block=rng.choice([8, 16, 16, 32, 64]),
                cache=rng.choice(["same", "same", "fp8"]), dtype=rng.choice(["bf16", "fp16"]),
                longest=longest, shortest=rng.randint(1, longest), prefix=prefix,
                mix=rng.randrange(1 << 20))


def draw(rng):
    return {"norm_rope": _draw_norm_rope, "append": _draw_append,
            "attend": _draw_attend}[rng.choice(["norm_rope", "append", "append", "attend",
                                                "attend", "attend"])](rng)


def _split(rng, total, parts):
    """`parts` counts of at least 1 that add up to `total`."""
    weights = [rng.random() + 0.2 for _ in range(parts)]
    counts = [1 + int((total - parts) * w / sum(weights)) for w in weights]
    counts[0] += total - sum(counts)
    return counts


def _batch(case):
    """(new tokens, length with them) of every sequence; the shared prefix is
    part of the length."""
    rng = random.Random(case["mix"])
    new = _split(rng, case["tokens"], case["sequences"])
    lo, hi = case.get("shortest", 0), case["longest"]
    prefix = case.get("prefix", 0)
    return new, [prefix + n + rng.randint(lo, hi) for n in new]


def _inverse_frequencies(rotary):
    return (500000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float().cuda()


def _randn(gen, shape, dtype, scale=1.0):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    return x.mul_(scale).to(dtype)


def _cache(case, gen, blocks, heads, empty=False):
    """One storage of the pool and, in e4m3, its scales."""
    shape = (blocks, case["block"], heads, case["dim"])
    if case["cache"] != "fp8":
        return _randn(gen, shape, DTYPES[case["dtype"]]), None
    scales = torch.rand(blocks, heads, generator=gen, device="cuda") * 0.004 + 0.004
    values = torch.randn(shape, generator=gen, device="cuda").div_(scales[:, None, :, None])
    return values.clamp_(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scales


def _tables(case, seed, lengths):
    """Block tables over a pool whose free ids come in a worked-in allocator's
    order; the blocks of a shared prefix are the same for every sequence."""
    block, prefix = case["block"], case.get("prefix", 0)
    shared = prefix // block
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


def _manager(state):
    from __graft_entry__ import load_package
    kvx = load_package()
    scales = [s for s in (state["k_scales"], state["v_scales"]) if s is not None]
    return kvx.KVCacheManager([state["k_cache"], state["v_cache"]], host_blocks_to_allocate=1,
                              scale_tables=scales)


def _prepare_norm_rope(case, gen, seed):
    del seed
    T, Hq, Hk, D = case["tokens"], case["q_heads"], case["k_heads"], case["dim"]
    dtype = DTYPES[case["dtype"]]
    # q and k are parts of the fused projection's output (q, k and v side by side).
    fused = _randn(gen, (T, Hq + 2 * Hk, D), dtype, 1.5)
    state = dict(case=case, q=fused[:, :Hq], k=fused[:, Hq:Hq + Hk],
                 positions=torch.randint(0, case["far"], (T,), generator=gen, device="cuda"),
                 inv_freq=_inverse_frequencies(case["rotary"]), q_weight=None, k_weight=None)
    if case["norm"]:
        state["q_weight"] = 1 + _randn(gen, (D,), dtype, 0.1)
        state["k_weight"] = 1 + _randn(gen, (D,), dtype, 0.1)
    if own:
        from __graft_entry__ import load_package
        state["kvx"] = load_package()
    return state


def _prepare_pool(case, gen, seed, heads):
    new, lengths = _batch(case)
    tables, blocks = _tables(case, seed, lengths)
    k_cache, k_scales = _cache(case, gen, blocks, heads)
    v_cache, v_scales = _cache(case, gen, blocks, heads)
    starts = torch.tensor([0] + new, dtype=torch.int32).cumsum(0, dtype=torch.int32).cuda()
    state = dict(case=case, tables=tables, k_cache=k_cache, v_cache=v_cache, k_scales=k_scales,
                 v_scales=v_scales, lengths=torch.tensor(lengths, dtype=torch.int32).cuda(),
                 starts=starts)
    if own:
        state["manager"] = _manager(state)
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
    state = _prepare_pool(case, gen, seed, case["k_heads"])
    state["q"] = _randn(gen, (case["tokens"], case["q_heads"], case["dim"]),
                        DTYPES[case["dtype"]], 1.3)
    state["scale"] = case["dim"] ** -0.5
    if case["prefix"]:
        state["group_starts"] = torch.tensor([0, case["sequences"]], dtype=torch.int32).cuda()
        whole = case["prefix"] // case["block"] * case["block"]
        state["prefix_lengths"] = torch.tensor([whole], dtype=torch.int32).cuda()
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return {"norm_rope": _prepare_norm_rope, "append": _prepare_append,
            "attend": _prepare_attend}[case["family"]](case, gen, seed)


# -- the framework's calls ------------------------------------------------------------------------

def _own_norm_rope(s):
    return s["kvx"].norm_rope(s["q"], s["k"], s["positions"], s["inv_freq"],
                              q_weight=s["q_weight"], k_weight=s["k_weight"], eps=1e-6,
                              interleaved=s["case"]["interleaved"])


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


def _pool(s):
    return [t for t in (s["k_cache"], s["v_cache"], s["k_scales"], s["v_scales"]) if t is not None]


# -- the plain forms ------------------------------------------------------------------------------

def _plain_norm(x, weight):
    x = x.float()
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.float()


def _plain_rotate(x, positions, inv_freq, interleaved):
    angle = (positions.double()[:, None] * inv_freq.double())[:, None]  # far positions need 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    half = inv_freq.numel()
    out = x.clone()
    if interleaved:
        u, v = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = u * cos - v * sin, v * cos + u * sin
    else:
        u, v = x[..., :half], x[..., half:2 * half]
        out[..., :half], out[..., half:2 * half] = u * cos - v * sin, v * cos + u * sin
    return out


def _plain_norm_rope(s):
    inter = s["case"]["interleaved"]
    return tuple(_plain_rotate(_plain_norm(x, w), s["positions"], s["inv_freq"], inter).to(x.dtype)
                 for x, w in ((s["q"], s["q_weight"]), (s["k"], s["k_weight"])))


def _plain_places(s):
    """Position, block and slot of every new token, and its sequence."""
    starts, lengths = s["starts"].long(), s["lengths"].long()
    token = torch.arange(s["case"]["tokens"], device="cuda")
    sequence = (token[:, None] >= starts[None, 1:]).sum(1)
    position = lengths[sequence] - starts[sequence + 1] + token
    block = s["tables"][sequence, position // s["case"]["block"]].long()
    return sequence, position, block, position % s["case"]["block"]


def _plain_store_fp8(s, cache, scales, x, block, slot):
    """x into an e4m3 storage: a block's scale is the largest of its new
    values' and, where it holds earlier tokens, its present one."""
    starts, lengths = s["starts"].long(), s["lengths"].long()
    first = lengths - (starts[1:] - starts[:-1])  # position of each sequence's first new token
    begun = s["tables"].long().gather(1, (first // s["case"]["block"])[:, None])[:, 0]
    earlier = first % s["case"]["block"]  # tokens that the block holds already
    old = torch.zeros_like(scales)
    old[begun] = torch.where(earlier[:, None] > 0, scales[begun], torch.zeros_like(scales[begun]))
    index = block[:, None].expand(-1, x.shape[1])
    new = old.scatter_reduce(0, index, x.abs().amax(-1) / FP8_MAX, "amax")
    # Earlier tokens keep their values under the larger scale.
    ratio = torch.where(new[begun] > 0, old[begun] / new[begun], torch.ones_like(new[begun]))
    kept = cache[begun].float()
    slots = torch.arange(s["case"]["block"], device="cuda")
    mine = (slots[None] < earlier[:, None])[:, :, None, None]
    moved = torch.where(mine, kept * ratio[:, None, :, None], kept)
    cache[begun] = moved.to(torch.float8_e4m3fn)
    inverse = torch.where(new > 0, 1 / new, torch.zeros_like(new))
    values = (x * inverse[block][:, :, None]).clamp(-FP8_MAX, FP8_MAX)
    cache[block, slot] = values.to(torch.float8_e4m3fn)
    scales[block] = new[block]


def _plain_append(s):
    sequence, position, block, slot = _plain_places(s)
    key = _plain_rotate(_plain_norm(s["k"], s["k_weight"]), position, s["inv_freq"], False)
    if s["k_scales"] is not None:
        _plain_store_fp8(s, s["k_cache"], s["k_scales"], key, block, slot)
        _plain_store_fp8(s, s["v_cache"], s["v_scales"], s["v"].float(), block, slot)
    else:
        s["k_cache"][block, slot] = key.to(s["k_cache"].dtype)
        s["v_cache"][block, slot] = s["v"]
    return _pool(s)


def _plain_read(cache, scales, blocks):
    """Blocks [..., n] of a storage as [..., kv head, token, dim] in 32 bits."""
    x = cache[blocks.long()].float()
    if scales is not None:
        x = x * scales[blocks.long()][..., None, :, None]
    x = x.flatten(-4, -3)
    return x.transpose(-3, -2).contiguous()


def _plain_attend(s):
    case, q = s["case"], s["q"].float() * s["scale"]
    S, Hk, D, B = case["sequences"], case["k_heads"], case["dim"], case["block"]
    G, shared = case["q_heads"] // Hk, case["prefix"] // case["block"]
    starts, lengths = s["starts"].long(), s["lengths"].long()
    new = starts[1:] - starts[:-1]
    token = torch.arange(case["tokens"], device="cuda")
    sequence = (token[:, None] >= starts[None, 1:]).sum(1)
    place = token - starts[sequence]
    # Queries by sequence, padded to the longest run: [S, Hk, most * G, D].
    most = max(_batch(case)[0])
    rows = torch.zeros(S, most, Hk, G, D, device="cuda")
    rows[sequence, place] = q.view(-1, Hk, G, D)
    rows = rows.transpose(1, 2).reshape(S, Hk, most * G, D)
    keys = _plain_read(s["k_cache"], s["k_scales"], s["tables"][:, shared:])
    values = _plain_read(s["v_cache"], s["v_scales"], s["tables"][:, shared:])
    scores = torch.matmul(rows, keys.transpose(-1, -2).contiguous())
    j = torch.arange(keys.shape[2], device="cuda") + shared * B
    last = (lengths - new)[:, None] + torch.arange(most, device="cuda")  # position of each query
    hidden = j[None, None] > torch.minimum(last, lengths[:, None] - 1)[..., None]
    hidden = hidden.repeat_interleave(G, 1)[:, None]
    scores = scores.masked_fill_(hidden, -math.inf)
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


def run(state):
    if own:
        return {"norm_rope": _own_norm_rope, "append": _own_append,
                "attend": _own_attend}[state["case"]["family"]](state)
    return {"norm_rope": _plain_norm_rope, "append": _plain_append,
            "attend": _plain_attend}[state["case"]["family"]](state)


# -- 64 bits, from the definitions ----------------------------------------------------------------

def _exact_rows(x, weight, positions, inv_freq, interleaved):
    """Norm and rotation as a complex product."""
    y = x.double()
    if weight is not None:
        y = y / ((y ** 2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * weight.double()
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device="cuda"),
                       torch.outer(positions.double(), inv_freq.double()))[:, None]
    half = inv_freq.numel()
    part = y[..., :2 * half]
    if interleaved:
        pairs = torch.view_as_complex(part.unflatten(-1, (half, 2)).contiguous())
        turned = torch.view_as_real(pairs * turn).flatten(-2)
    else:
        pairs = torch.complex(part[..., :half].contiguous(), part[..., half:].contiguous()) * turn
        turned = torch.cat((pairs.real, pairs.imag), -1)
    return torch.cat((turned, y[..., 2 * half:]), -1)


def _exact_append(case, s):
    new, lengths = _batch(case)
    B, at = case["block"], []
    for i, n in enumerate(new):
        at += [(i, lengths[i] - n + j) for j in range(n)]
    positions = torch.tensor([p for _, p in at], device="cuda")
    key = _exact_rows(s["k"], s["k_weight"], positions, s["inv_freq"], False)
    outs, scale_outs = [], []
    for cache, scales, x in ((s["k_cache"], s["k_scales"], key),
                             (s["v_cache"], s["v_scales"], s["v"].double())):
        pool = cache.double()
        table = scales.double() if scales is not None else None
        begin = 0
        for i, n in enumerate(new):
            p = lengths[i] - n
            done = 0
            while done < n:
                b = int(s["host_tables"][i][(p + done) // B])
                slot = (p + done) % B
                many = min(B - slot, n - done)
                rows = x[begin + done:begin + done + many]
                if table is not None:
                    old = table[b] if slot else torch.zeros_like(table[b])
                    size = torch.maximum(old, rows.abs().amax((0, 2)) / FP8_MAX)
                    if slot:
                        pool[b, :slot] = (pool[b, :slot] * (old / size)[:, None]).to(
                            torch.float8_e4m3fn).double()
                    table[b] = size
                    rows = (rows / size[:, None]).clamp(-FP8_MAX, FP8_MAX)
                    rows = rows.to(torch.float8_e4m3fn).double()
                pool[b, slot:slot + many] = rows
                done += many
            begin += n
        outs.append(pool)
        if table is not None:
            scale_outs.append(table)
    return outs + scale_outs


def _exact_attend(case, s):
    new, lengths = _batch(case)
    B, Hk = case["block"], case["k_heads"]
    G, begin, outs = case["q_heads"] // Hk, 0, []
    for i, n in enumerate(new):
        ids = s["tables"][i, :(lengths[i] + B - 1) // B].long()
        k, v = s["k_cache"][ids].double(), s["v_cache"][ids].double()
        if s["k_scales"] is not None:
            k = k * s["k_scales"][ids].double()[:, None, :, None]
            v = v * s["v_scales"][ids].double()[:, None, :, None]
        k, v = (x.flatten(0, 1)[:lengths[i]] for x in (k, v))
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


def exact(case, seed):
    s = prepare(case, seed)
    if case["family"] == "norm_rope":
        return tuple(_exact_rows(s[n], s[n + "_weight"], s["positions"], s["inv_freq"],
                                 case["interleaved"]) for n in ("q", "k"))
    if case["family"] == "append":
        s["host_tables"] = s["tables"].tolist()
        return _exact_append(case, s)
    return _exact_attend(case, s)


# -- what a pass cannot do without ----------------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    held = 1 if case.get("cache") == "fp8" else size
    T, D, B = case["tokens"], case["dim"], case.get("block", 1)
    if case["family"] == "norm_rope":
        values = T * (case["q_heads"] + case["k_heads"]) * D
        return {"bytes": 2 * values * size + 8 * T, "flops": 10 * values}
    new, lengths = _batch(case)
    if case["family"] == "append":
        values = 2 * T * case["heads"] * D
        touched = sum((m - 1) // B - (m - n) // B + 1 for n, m in zip(new, lengths))
        scales = 2 * 8 * touched * case["heads"] if held == 1 else 0
        return {"bytes": values * (size + held) + scales + 4 * touched, "flops": 6 * values}
    keys = case["prefix"] + sum(m - case["prefix"] for m in lengths)
    seen = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, lengths))
    scales = 2 * 4 * case["k_heads"] * (keys // B) if held == 1 else 0
    return {"bytes": 2 * keys * case["k_heads"] * D * held + scales + 4 * (keys // B)
                     + 2 * T * case["q_heads"] * D * size,
            "flops": 4 * seen * case["q_heads"] * D}
