"""Plain 64-bit forms of the operators that fill and read the paged pool, on the
CPU, and how far a result in fewer bits may be from them."""
import torch

FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
U32 = 2.0 ** -24  # half a step of fp32, relative


def half(dtype):
    """Half a step of a rounding to `dtype`, relative to the value."""
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance of the smallest values."""
    return {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150,
            FP8: 2.0 ** -10}[dtype]


def rotate(y, positions, inv_freq, interleaved=False):
    if inv_freq is None:
        return y
    a = positions.double().cpu()[:, None, None] * inv_freq.double().cpu()[None, None]
    n, out = inv_freq.numel(), y.clone()
    if interleaved:
        u, v = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
        out[..., 0:2 * n:2], out[..., 1:2 * n:2] = u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()
    else:
        u, v = y[..., :n], y[..., n:2 * n]
        out[..., :n], out[..., n:2 * n] = u * a.cos() - v * a.sin(), v * a.cos() + u * a.sin()
    return out


def norm_rope(x, weight, positions, inv_freq, eps=1e-6, interleaved=False):
    """(result, bound of the error before the last rounding). In fp32: a mean
    of D squares (D + 2 half steps), a root, a reciprocal and two products (6),
    then an angle good to 2^-25 turns (2 pi 2^-25 < 4 half steps), cos and sin
    (4 each) and three roundings: D + 32 half steps of each of the pair's
    magnitudes bound them."""
    y = x.double().cpu()
    if weight is not None:
        y = y * weight.double().cpu() / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    out = rotate(y, positions, inv_freq, interleaved)
    size = y.abs()
    if inv_freq is not None:
        n, other = inv_freq.numel(), torch.zeros_like(size)
        if interleaved:
            other[..., 0:2 * n:2], other[..., 1:2 * n:2] = size[..., 1:2 * n:2], size[..., 0:2 * n:2]
        else:
            other[..., :n], other[..., n:2 * n] = size[..., n:2 * n], size[..., :n]
        size = size + other
    return out, size * ((x.shape[-1] + 32) * U32)


def assert_rounded(got, want, slack, dtype):
    """got: want + at most slack, rounded to dtype (half a step of the value)."""
    got, room = got.double().cpu(), (want.abs() + slack) * half(dtype) + slack + tiny(dtype)
    off = (got - want).abs()
    bad = ~(off <= room)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((off / room.clamp_min(1e-300)).max())} of its bound")


def places(starts, lengths, tokens, sequences):
    """[(token, sequence, position)] of a call's tokens."""
    out = []
    for s in range(sequences):
        first, end = (s, s + 1) if starts is None else (starts[s], starts[s + 1])
        out += [(t, s, lengths[s] - end + t) for t in range(first, min(end, tokens))]
    return out


def gather(cache, scales, table, length):
    """Tokens [0, length) of a sequence, dequantised, [length, heads, dim]."""
    block = cache.shape[1]
    rows = []
    for j in range((length + block - 1) // block):
        x = cache[table[j]].double()
        if scales is not None:
            x = x * scales[table[j]].double()[None, :, None]
        rows.append(x)
    if not rows:
        return cache[:0].double().reshape(0, *cache.shape[2:])
    return torch.cat(rows)[:length]


def attend(q, k, v, visible, scale, dtype, product):
    """Attention of q [n, Hq, D] over k, v [L, Hk, D]; row i sees the tokens
    where visible[i]. Returns (out, lse, slack). The error before the last
    rounding: scores are sums of D products (exact in 32 bits each) scaled and
    moved into an exponent of 2, D + 8 half steps of sum |q k| scale, plus 64
    of 1 for the exponent's own size and the exponential; exponentials are
    rounded to `product` (half a step each) and summed with the values, L + 64
    half steps in fp32. All of it weighs with the attention of |v|; below the
    16-bit type's range an exponential is off by tiny(product), and the sum of
    exponentials is at least 2^-8 of its largest."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out = torch.zeros(n, heads, dim, dtype=torch.float64)
    slack = torch.zeros_like(out)
    lse = torch.full((n, heads), float("-inf"), dtype=torch.float64)
    for h in range(heads if len(k) else 0):
        keys, values = k[:, h // group], v[:, h // group]
        s = q[:, h].double() @ keys.t() * scale
        s = s.masked_fill(~visible, float("-inf"))
        some = visible.any(-1)
        lse[:, h] = torch.logsumexp(s, -1)
        w = torch.softmax(s, -1)
        w[~some] = 0
        w = torch.where(visible, w, torch.zeros_like(w))
        clean = torch.where(visible.any(0)[:, None], values, torch.zeros_like(values))
        out[:, h] = w @ clean
        size = q[:, h].double().abs() @ keys.nan_to_num(0, 0, 0).abs().t() * scale
        size = torch.where(visible, size, torch.zeros_like(size)).amax(-1, keepdim=True)
        rel = (2 * (dim + 8) * size + len(keys) + 128) * U32 + half(product)
        slack[:, h] = rel * (w @ clean.abs()) + tiny(product) * 256 * (
            clean.abs().sum(0, keepdim=True) if product == torch.float16 else 0)
    return out, lse, slack
