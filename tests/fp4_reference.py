"""The 4-bit pool's format on the CPU, from its definition: e2m1 codes [blocks,
heads, tokens, dim / 2] with one e8m0 scale for 32 dimensions [blocks, heads,
tokens, dim / 32]."""
import torch

FP4, E8M0 = torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
CODES = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6],
                     dtype=torch.float64)
LEAST, MOST = -125, {torch.bfloat16: 125, torch.float16: 13}  # exponents of scales


def raw(t):
    return t.view(torch.uint8).cpu()


def values(codes):
    """What the codes stand for, before their scales."""
    b = raw(codes).long()
    return CODES[torch.stack((b & 15, b >> 4), -1).flatten(-2)]


def scale_values(scales):
    e = raw(scales).double()
    return torch.where(e == 255, torch.tensor(float("nan"), dtype=torch.float64), 2.0 ** (e - 127))


def decode(codes, scales):
    return values(codes) * scale_values(scales).repeat_interleave(32, -1)


def scale_code(largest, dtype):
    """e8m0 code of a group whose largest finite magnitude is given (64 bits)."""
    code = torch.full(largest.shape, LEAST + 127, dtype=torch.int64)
    for e in range(LEAST + 1, MOST[dtype] + 1):
        code += (largest > 7 * 2.0 ** (e - 1)).long()
    return code


def half_step(size):
    """Half the distance between the codes around a magnitude (in scales)."""
    return torch.where(size <= 2, 0.25, torch.where(size <= 4, 0.5, 1.0)).double()


def encode(x, dtype):
    """(codes, scale codes) of rows [..., D] in bytes: the nearest, even ones in
    the middle."""
    groups = x.double().cpu().unflatten(-1, (-1, 32))
    size = groups.abs()
    finite = torch.where(size < float("inf"), size, 0.0).nan_to_num(0)
    code = scale_code(finite.amax(-1), dtype)
    y = size / (2.0 ** (code - 127).double())[..., None]
    middles = (CODES[1:8] + CODES[:7]) / 2
    found = torch.zeros(y.shape, dtype=torch.int64)
    for i, m in enumerate(middles.tolist()):  # the middle above an odd code goes up
        found += ((y > m) if i % 2 == 0 else (y >= m)).long()
    found += torch.signbit(groups).long() * 8
    found = found.flatten(-2)
    code = torch.where(groups.isnan().any(-1), 255, code)
    return (found[..., 0::2] + 16 * found[..., 1::2]).to(torch.uint8), code.to(torch.uint8)


def storage(x, dtype, device):
    """A 4-bit storage and its scales of values [blocks, heads, tokens, dim]."""
    codes, scales = encode(x, dtype)
    return codes.to(device).view(FP4), scales.to(device).view(E8M0)


def gather(codes, scales, table, length):
    """Tokens [0, length) of a sequence, [length, heads, dim] in 64 bits."""
    block = codes.shape[2]
    ids = torch.tensor(table[:(length + block - 1) // block], dtype=torch.long)
    if not len(ids):
        return torch.zeros(0, codes.shape[1], codes.shape[3] * 2, dtype=torch.float64)
    x = decode(raw(codes)[ids], raw(scales)[ids])
    return x.transpose(1, 2).flatten(0, 1)[:length]
