"""Attention over the 8-bit cache where the sizes of its values differ from block to block, by more than fp32's range of
exponents if need be: blocks of any size in any order within one warp's and one CTA's share, blocks at the ends of the range,
blocks of zeros beside small values, and recent tokens beside complete blocks."""
import pytest
import torch

from helpers import randn
from oracle import quantized as OQ

pytestmark = pytest.mark.gpu


def expect_close(got, q, k, v, start):
    """got [S,Hq,D] against 64 bits, relative to the values' own size. Per output element, with u half a step of the type:
    its own rounding u; every weight rounded to the type u; scores in fp32 over D products, e = 2 (D + 8) 2^-24 times the largest
    (an error of a score is a factor exp(e), in numerator and denominator); the score plus log2 of the value scale (at
    most 150) rounded three times, 3 * 150 * 2^-24 * ln 2 < 2^-15; exponentials and sums 2^-18. A weight is a multiple of 2^-24 after
    the factor of at least 2^7 that the largest weight in its row starts from: 2^-32 of the largest term at most, for every token."""
    length, dtype = k.shape[0], q.dtype
    kk, vv = OQ.held(k, length), OQ.held(v, length)
    want, scale, largest = OQ.attention(q, kk, vv, start)
    u = torch.finfo(dtype).eps / 2
    e = 2 * (q.shape[2] + 8) * 2.0 ** -24 * largest + 2.0 ** -15 + 2.0 ** -18
    most = vv.abs().amax(dim=2)                                            # [H,T]: a token's terms are at most p * most
    for j in range(0, length - length % 64, 64):
        most[:, j:j + 64] = vv[:, j:j + 64].abs().amax(dim=(1, 2))[:, None]
    group = q.shape[1] // kk.shape[0]
    scores = torch.einsum('shd,htd->hst', q.double(), kk.repeat_interleave(group, dim=0)) * q.shape[2] ** -0.5
    late = torch.arange(length)[None] > start + torch.arange(q.shape[0])[:, None]
    p = torch.softmax(scores.masked_fill(late, float('-inf')), dim=-1)
    term = (p * most.repeat_interleave(group, dim=0)[:, None]).amax(dim=-1).transpose(0, 1)[..., None]      # [S,Hq,1]
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    bound = u * want.abs() + (u + e) * (scale + want.abs()) * 1.01 + length * 2.0 ** -32 * term + step
    assert torch.isfinite(got).all()
    excess = ((got.double().cpu() - want).abs() - bound) / want.abs().amax().clamp_min(1e-300)
    assert float(excess.max()) <= 0, float(excess.max())


def attend(sizes, s, d, dtype, batch, tail=0, seed=5, peak=None):
    """A cache of the blocks whose values have these sizes (and `tail` tokens of the last size), for `batch` sequences of the
    same tokens: enough of them leave a sequence in one piece, so that a warp (a CTA) meets all kinds of blocks."""
    from qwen3_triton.inference import quantized as Q
    t = 64 * len(sizes) if not tail else 64 * (len(sizes) - 1) + tail
    k = randn((t, 1, d), seed) * 0.2
    v = randn((t, 1, d), seed + 1).clamp(-3, 3) + 0.5                       # a mean that sums do not lose
    for j, size in enumerate(sizes):
        v[64 * j:64 * j + 64] *= size
    q = randn((s, 4, d), seed + 2)
    if peak is not None:                                                   # one token takes `peak` times the weight of another
        q[..., 0], k[..., 0] = 1.0, 0.0
        k[t - s, 0, 0] = torch.log(torch.tensor(peak)) * d ** 0.5
    k, v, q = k.to(dtype), v.to(dtype), q.to(dtype)
    assert torch.isfinite(v).all()
    cache = Q.QuantizedCache(batch, 1, t, d, dtype=dtype)
    Q.append(k.cuda().expand(batch, t, 1, d).contiguous(), v.cuda().expand(batch, t, 1, d).contiguous(), cache, 0)
    out = Q.attention(q.cuda().expand(batch, s, 4, d).contiguous(), cache, t - s)
    assert torch.equal(out, out[:1].expand_as(out))
    expect_close(out[0], q, k, v, t - s)


@pytest.mark.parametrize('s,d', [(1, 128), (3, 64), (40, 128), (90, 64)])
@pytest.mark.parametrize('sizes', [(1.0, 1e-36), (1e-36, 1.0), (1e20, 1e-18), (1e-18, 1e20), (1e20, 1e-30), (1e-30, 1e20), (1e37, 1e-37),
                                   (1e37, 1.0, 1e-37), (1e-37, 1e-20, 1e-3, 1e14, 1e37)])
@pytest.mark.parametrize('batch', [1, 160])
def test_value_scales_of_any_ratio_in_any_order(sizes, s, d, batch):
    g = torch.Generator().manual_seed(len(sizes))
    order = [sizes[i] for i in torch.randint(0, len(sizes), (24,), generator=g).tolist()]
    attend(list(sizes) + order + list(sizes[::-1]), s, d, torch.bfloat16, batch)


@pytest.mark.parametrize('s', [1, 3, 40])
@pytest.mark.parametrize('size', [1e-38, 1e-36, 1e-34, 1e-30, 9e37])
@pytest.mark.parametrize('blocks,batch', [(1, 1), (2, 1), (30, 1), (30, 160), (600, 1)])
def test_values_at_the_ends_of_the_range(size, s, blocks, batch):
    """All values tiny, or so large that a sum of two is not finite: in one piece, joined pieces and merged pieces."""
    attend([size] * blocks, s, 128, torch.bfloat16, batch)


@pytest.mark.parametrize('dtype,size', [(torch.bfloat16, 1e-3), (torch.bfloat16, 1e-5), (torch.bfloat16, 1e-6), (torch.bfloat16, 1e-20),
                                        (torch.float16, 1e-3), (torch.float16, 1e-5), (torch.float16, 1e-6)])
@pytest.mark.parametrize('s', [1, 3, 40])
@pytest.mark.parametrize('tail', [0, 50])
@pytest.mark.parametrize('batch', [1, 160])
def test_blocks_of_zeros_beside_small_values(dtype, s, size, tail, batch):
    attend([size, 0.0, size, size, 0.0, 0.0, size], s, 64, dtype, batch, tail)
    attend([size, 0.0, size, 0.0], s, 64, dtype, batch, tail)               # the zeros last


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('s', [1, 3, 40])
@pytest.mark.parametrize('size', [1.0, 1e-2, 1e-4, 1e-6])
def test_small_values_of_complete_blocks_beside_a_heavy_recent_token(dtype, s, size):
    """Half of the weight on a recent token: what the 64 of the block beside it hold must keep its digits."""
    attend([size, size], s, 128, dtype, 1, 50, peak=100.0)
    attend([size] * 6, s, 128, dtype, 1, 50, peak=300.0)
