"""GPU: norm and rotation of query and key heads against the 64-bit form."""
import decimal

import pytest

torch = pytest.importorskip("torch")

import paged_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def freqs(n, cuda):
    return (10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))).float().to(cuda)


def check(got, x, weight, positions, inv_freq, eps=1e-6, interleaved=False):
    want, slack = ref.norm_rope(x, weight, positions, inv_freq, eps, interleaved)
    ref.assert_rounded(got, want, slack, x.dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("tokens,hq,hk,dim,rotary,norm,inter", [
    (1, 1, 1, 128, 128, True, False), (3, 32, 8, 128, 128, True, False),
    (65, 5, 1, 64, 64, False, False), (7, 4, 2, 80, 32, False, True),
    (33, 8, 8, 96, 96, True, True), (5, 2, 1, 256, 128, True, False),
    (9, 3, 3, 20, 6, True, False), (4, 2, 2, 33, 32, True, True), (2, 1, 1, 1, 0, True, False),
    (11, 2, 1, 128, 0, True, False), (1500, 3, 1, 64, 48, True, False),
    (2, 2, 2, 200, 200, True, False), (1, 70, 1, 136, 136, True, True)])
def test_against_64_bits(kvx, cuda, dtype, tokens, hq, hk, dim, rotary, norm, inter):
    gen = torch.Generator(device=cuda).manual_seed(tokens * 1000 + dim)
    fused = torch.randn(tokens, hq + 2 * hk, dim, device=cuda, generator=gen).to(dtype)
    q, k = fused[:, :hq], fused[:, hq:hq + hk]
    before = fused.clone()
    positions = torch.randint(0, 100000, (tokens,), device=cuda, generator=gen)
    inv_freq = freqs(rotary // 2, cuda) if rotary else None
    wq = wk = None
    if norm:
        wq = torch.randn(dim, device=cuda, generator=gen).to(dtype)
        wk = torch.randn(dim, device=cuda, generator=gen).to(dtype)
    gq, gk = kvx.norm_rope(q, k, positions, inv_freq, q_weight=wq, k_weight=wk, eps=1e-5,
                           interleaved=inter)
    assert gq.shape == q.shape and gk.dtype == dtype and gk.is_contiguous()
    check(gq, q, wq, positions, inv_freq, 1e-5, inter)
    check(gk, k, wk, positions, inv_freq, 1e-5, inter)
    assert torch.equal(fused, before)


def test_strides_weights_and_position_types(kvx, cuda):
    x = torch.randn(6, 3, 128, device=cuda).to(BF16)
    heads_first = x.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(6 * 3 * 128 + 1, dtype=BF16, device=cuda)[1:].view(6, 3, 128)
    odd.copy_(x)
    wide = torch.zeros(6, 3, 131, dtype=BF16, device=cuda)[..., :128]
    wide.copy_(x)
    w = torch.randn(128, device=cuda)  # fp32 weight of bf16 rows
    pos = torch.tensor([0, 1, 2**31 - 1, 77, 5, 131071], dtype=torch.int32, device=cuda)
    inv = freqs(64, cuda)
    base, _ = kvx.norm_rope(x, None, pos, inv, q_weight=w)
    check(base, x, w, pos, inv)
    for y in (heads_first, odd, wide):
        got, none = kvx.norm_rope(y, None, pos, inv, q_weight=w)
        assert none is None
        check(got, x, w, pos, inv)
    out = torch.full((6, 3, 256), 7.0, dtype=BF16, device=cuda)
    kvx.norm_rope(x, None, pos, inv, q_weight=w, out_q=out[..., :128])
    assert torch.equal(out[..., :128], base) and bool((out[..., 128:] == 7).all())
    expanded = x[:, :1].expand(6, 3, 128)
    got, _ = kvx.norm_rope(expanded, None, pos, inv)
    check(got, expanded, None, pos, inv)
    far = torch.tensor([2**40 + 3, 10**15, 0, 1, 2**53, 12], dtype=torch.int64, device=cuda)
    got, _ = kvx.norm_rope(x.float(), None, far, inv)
    # 64 bits do not hold these products: the reference takes the angles, reduced
    # by whole turns, from 60 decimal digits.
    with decimal.localcontext() as ctx:
        ctx.prec = 60
        turn = 2 * decimal.Decimal("3.14159265358979323846264338327950288419716939937510582097494")
        angles = torch.tensor([[float(decimal.Decimal(p) * decimal.Decimal(f) % turn)
                                for f in inv.double().tolist()] for p in far.tolist()],
                              dtype=torch.float64)
    y = x.double().cpu()
    u, v, c, s = y[..., :64], y[..., 64:], angles.cos()[:, None], angles.sin()[:, None]
    want = torch.cat((u * c - v * s, v * c + u * s), -1)
    _, slack = ref.norm_rope(x.float(), None, far, inv)
    ref.assert_rounded(got, want, slack, F32)


def test_in_place_and_split_over_workgroups(kvx, cuda):
    fused = torch.randn(40, 12, 128, device=cuda).to(F16)
    pos = torch.arange(40, device=cuda)
    inv, w = freqs(64, cuda), torch.randn(128, device=cuda).to(F16)
    want_q, want_k = kvx.norm_rope(fused[:, :8], fused[:, 8:10], pos, inv, q_weight=w, k_weight=w)
    v = fused[:, 10:].clone()
    q, k = fused[:, :8], fused[:, 8:10]
    rq, rk = kvx.norm_rope(q, k, pos, inv, q_weight=w, k_weight=w, out_q=q, out_k=k)
    assert rq is q and rk is k
    assert torch.equal(q, want_q) and torch.equal(k, want_k) and torch.equal(fused[:, 10:], v)


def test_values_that_are_not_finite_stay_in_their_row(kvx, cuda):
    x = torch.randn(4, 2, 128, device=cuda)
    x[1, 0, 3], x[2, 1, 70] = float("nan"), float("inf")
    pos = torch.arange(4, device=cuda)
    got, _ = kvx.norm_rope(x, None, pos, freqs(64, cuda), q_weight=torch.ones(128, device=cuda))
    bad = ~torch.isfinite(got).all(-1)
    assert bad.tolist() == [[False, False], [True, False], [False, True], [False, False]]
    zero = torch.zeros(2, 1, 64, device=cuda)
    got, _ = kvx.norm_rope(zero, None, pos[:2], freqs(32, cuda),
                           q_weight=torch.ones(64, device=cuda), eps=1e-6)
    assert bool((got == 0).all())


def test_no_tokens_and_another_stream(kvx, cuda):
    empty = torch.empty(0, 4, 64, device=cuda)
    got, _ = kvx.norm_rope(empty, None, torch.empty(0, dtype=torch.int64, device=cuda),
                           freqs(32, cuda))
    assert got.shape == (0, 4, 64)
    x = torch.randn(300, 8, 128, device=cuda).to(BF16)
    pos, inv = torch.arange(300, device=cuda), freqs(64, cuda)
    want, _ = kvx.norm_rope(x, None, pos, inv)
    side = torch.cuda.Stream(cuda)
    torch.cuda.synchronize()
    for stream in (side, side.cuda_stream):
        got, _ = kvx.norm_rope(x, None, pos, inv, stream=stream)
        side.synchronize()
        assert torch.equal(got, want)
