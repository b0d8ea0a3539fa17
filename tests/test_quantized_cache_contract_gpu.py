"""What the 8-bit cache promises around the edges of its contract: appends that it refuses, stepping back more than once, padded
calls at the end of the cache, caches much longer than their sequences, and where each byte lies."""
import pytest
import torch

from helpers import randn
from oracle import quantized as OQ
from test_quantized_cache_gpu import expect_attention, expect_read, lengths, make, tokens

pytestmark = pytest.mark.gpu


def part(x, first, last):
    return x[:, first:last].contiguous().cuda()


def reported():
    """Whether the status names missing tokens, and nothing else."""
    from qwen3_triton import _abi
    status = _abi.read_status()
    assert status in (0, _abi.STATUS_CACHE_RECENT)
    return status != 0


def test_a_refused_append_to_an_incomplete_block_leaves_the_sequence_alone():
    """A gap: the block's earlier tokens are not all there. What was held stays; the length that the call was to reach is reported."""
    from qwen3_triton.inference import quantized as Q
    dtype, h, d, t = torch.bfloat16, 2, 64, 400
    k, v = tokens(2, t, h, d, dtype, 21)
    cache = make(2, h, t, d, dtype)
    Q.append(part(k, 0, 300), part(v, 0, 300), cache, 0)
    buffers = (cache.keys, cache.values, cache.key_scales, cache.value_scales, cache.recent_keys, cache.recent_values, cache.marks)
    before = [x.clone() for x in buffers]
    for start, n in [(310, 1), (301, 19), (100, 3), (330, 50)]:              # in the block, to its end, an older block, the next one
        n = min(n, 63 - start % 64)
        Q.append(part(k, start, start + n), part(v, start, start + n), cache, start)
        assert reported()
        assert all(torch.equal(x, y) for x, y in zip(before, buffers)), start
        Q.read(cache, start + n)
        assert reported()
        for s in (1, 40):
            Q.attention(randn((2, s, 4, d), 1, dtype).cuda(), cache, start + n - s)
            assert reported()
    for i in range(2):
        expect_read(Q.read(cache, 300)[0][i], k[i], 300)
    Q.append(part(k, 300, 400), part(v, 300, 400), cache, 300)
    for i in range(2):
        expect_read(Q.read(cache, 400)[1][i], v[i], 400)
    assert not reported()


@pytest.mark.parametrize('start,n', [(100, 28), (100, 29), (100, 92), (100, 93), (100, 200), (70, 250)])
@pytest.mark.parametrize('ragged', [False, True])
def test_a_refused_append_that_completes_its_block_is_reported_until_it_is_written_anew(start, n, ragged):
    from qwen3_triton.inference import quantized as Q
    dtype, h, d, t = torch.float16, 1, 128, 700
    k, v = tokens(2, t, h, d, dtype, 23)
    cache = make(2, h, t, d, dtype)
    Q.append(part(k, 0, 600), part(v, 0, 600), cache, 0)
    end = start + n
    where = lengths(start, start) if ragged else start
    Q.append(part(k, start, end), part(v, start, end), cache, where)         # blocks 8 and 9 are held, not block 1
    assert reported()

    def all_report():
        seen = []
        for s in (1, 40):
            Q.attention(randn((2, s, 2, d), 1, dtype).cuda(), cache, end - s)
            seen.append(reported())
        Q.read(cache, end)
        seen.append(reported())
        Q.read(cache, end, 64, 5)
        seen.append(reported())
        return seen

    assert all(all_report())
    Q.append(part(k, end, end + 70), part(v, end, end + 70), cache, end)     # more tokens do not make it right
    assert reported()
    end += 70
    assert all(all_report())
    Q.append(part(k, 110, 120), part(v, 110, 120), cache, 110)               # nor does another step back into the block
    assert reported()
    Q.read(cache, 64)                                                        # what lies before it is untouched
    assert not reported()
    expect_read(Q.read(cache, 64)[1][0], v[0], 64)
    Q.attention(randn((2, 1, 2, d), 1, dtype).cuda(), cache, 63)
    assert not reported()
    Q.append(part(k, 64, end), part(v, 64, end), cache, 64)                  # the block anew
    assert not any(all_report())
    for i in range(2):
        expect_read(Q.read(cache, end)[0][i], k[i], end)
        expect_read(Q.read(cache, end)[1][i], v[i], end)
    Q.append(part(k, end, end + 5), part(v, end, end + 5), cache, end)
    assert not reported()
    expect_read(Q.read(cache, end + 5)[1][1], v[1], end + 5)


def test_a_new_sequence_in_the_place_of_a_refused_one():
    from qwen3_triton.inference import quantized as Q
    dtype, h, d, t = torch.bfloat16, 1, 64, 400
    k, v = tokens(1, t, h, d, dtype, 25)
    for n in (1, 64, 65, 300):
        cache = make(1, h, t, d, dtype)
        Q.append(part(k, 0, 300), part(v, 0, 300), cache, 0)
        Q.append(part(k, 100, 300), part(v, 100, 300), cache, 100)
        assert reported()
        Q.append(part(k, 0, n), part(v, 0, n), cache, 0)
        assert not reported()
        q = randn((1, 1, 2, d), 26, dtype)
        expect_attention(Q.attention(q.cuda(), cache, n - 1)[0], q[0], k[0, :n], v[0, :n], n - 1, dtype)
        expect_read(Q.read(cache, n)[0][0], k[0], n)
        assert not reported()
        Q.append(part(k, n, n + 70), part(v, n, n + 70), cache, n)
        expect_read(Q.read(cache, n + 70)[0][0], k[0], n + 70)
        assert not reported()


@pytest.mark.parametrize('s', [3, 50])
@pytest.mark.parametrize('where', ['host', 'device'])
def test_padding_may_reach_beyond_the_capacity(s, where):
    """The last chunk of a sequence, padded to the size of the others: its real tokens fit, its padding does not."""
    from qwen3_triton import _abi
    from qwen3_triton.inference import quantized as Q
    dtype, b, h, hq, d, cap = torch.bfloat16, 2, 2, 4, 64, 150
    k, v = tokens(b, cap + s, h, d, dtype, 31)
    q = randn((b, s, hq, d), 32, dtype)
    start, counts = cap - 2, (2, 1)
    cache = make(b, h, cap, d, dtype)
    Q.append(part(k, 0, start), part(v, 0, start), cache, 0)
    at = lengths(start, start) if where == 'device' else start
    Q.append(part(k, start, start + s), part(v, start, start + s), cache, at, lengths(*counts))
    out = Q.attention(q.cuda(), cache, at, lengths(*counts))
    for i, n in enumerate(counts):
        expect_attention(out[i, :n], q[i, :n], k[i, :start + n], v[i, :start + n], start, dtype)
        assert not out[i, n:].any()
        expect_read(Q.read(cache, lengths(*(start + c for c in counts)), 0, cap)[0][i], k[i], start + n)
    Q.append(part(k, 0, s), part(v, 0, s), cache, cap, lengths(0, 0))         # a full cache, and nothing new
    assert not Q.attention(q.cuda(), cache, cap, lengths(0, 0)).any()
    assert _abi.read_status() == 0
    Q.append(part(k, 0, s), part(v, 0, s), cache, cap - 1, lengths(1, 2))     # the second one does not fit
    assert _abi.read_status() == _abi.STATUS_CACHE_RANGE
    with pytest.raises(ValueError):
        Q.append(part(k, 0, s), part(v, 0, s), cache, cap + 1, lengths(0, 0))
    for call in (lambda: Q.append(part(k, 0, s), part(v, 0, s), cache, cap - s + 1), lambda: Q.attention(q.cuda(), cache, cap - s + 1)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('total', [100, 128, 150, 192, 200, 333, 340])
def test_the_recent_tokens_do_not_depend_on_the_cuts(dtype, total):
    """The last 128 tokens as given, one slot for each, whatever the calls were: token by token, at once, and pieces that start and
    end in the same and in different slots, before and behind one another."""
    from qwen3_triton.inference import quantized as Q
    h, d = 2, 64
    k, v = tokens(1, total, h, d, dtype, 40 + total)
    k[0, total - 70, 0, 5], v[0, total - 3, 1, 7] = float('nan'), float('inf')               # held as 0, with a mark
    pieces = [[total], [1] * total, [50, total - 50], [30, 40, total - 70], [10, total - 30, 20], [60, total - 64, 4]]
    want = [torch.zeros(1, h, 2, 64 * d, dtype=dtype), torch.zeros(1, h, 2, 64 * d, dtype=dtype)]
    for t in range(max(0, total - 128), total):
        row = t % 64
        key = [((row // 8) * (d // 64) + x // 64) * 512 + (row % 8) * 64 + x % 64 for x in range(d)]
        value = [x * 64 + ((row // 2) % 4) * 16 + (row // 8) * 2 + row % 2 for x in range(d)]
        for buffer, x, places in ((want[0], k, key), (want[1], v, value)):
            buffer[0, :, t // 64 % 2, places] = torch.where(torch.isfinite(x[0, t]), x[0, t], torch.zeros_like(x[0, t]))
    for cut in pieces:
        cache, at = make(1, h, total, d, dtype), 0
        for n in cut:
            Q.append(part(k, at, at + n), part(v, at, at + n), cache, at)
            at += n
        assert at == total
        assert torch.equal(cache.recent_keys.cpu(), want[0]) and torch.equal(cache.recent_values.cpu(), want[1]), cut
    assert not reported()


def test_steps_back_in_a_row():
    """What a sequence may go back to after it has gone back: the block it is in, and the one before only if it came from there."""
    from qwen3_triton.inference import quantized as Q
    dtype, h, d, t = torch.bfloat16, 2, 64, 400

    def check(steps, refused=()):
        cache, now = make(1, h, t, d, dtype), [torch.zeros(1, t, h, d, dtype=dtype) for _ in range(2)]
        for i, (start, n) in enumerate(steps):
            k, v = tokens(1, n, h, d, dtype, 60 + i)
            Q.append(k.cuda(), v.cuda(), cache, start)
            assert reported() == (i in refused), (steps, i)
            if i in refused:
                return
            for x, new in zip(now, (k, v)):
                x[:, start:start + n] = new
            end = start + n
            expect_read(Q.read(cache, end)[0][0], now[0][0], end)
            expect_read(Q.read(cache, end)[1][0], now[1][0], end)
            for s in (1, min(end, 30)):
                q = randn((1, s, 4, d), 90 + i, dtype)
                expect_attention(Q.attention(q.cuda(), cache, end - s)[0], q[0], now[0][0, :end], now[1][0, :end], end - s, dtype)
            assert not reported(), (steps, i)

    check([(0, 200), (195, 3), (193, 1), (150, 2), (140, 5)])            # down within blocks 3 and 2
    check([(0, 200), (130, 3), (131, 80), (190, 1)])                     # back to block 2, on into block 3: both are held again
    check([(0, 200), (130, 3), (100, 1)], refused=(2,))                  # block 1 was not held any more
    check([(0, 200), (128, 3), (100, 1)], refused=(2,))
    check([(0, 200), (64, 10), (30, 1)], refused=(2,))                   # nor block 0
    check([(0, 200), (64, 10), (70, 60), (100, 3)])                      # blocks 1 and 2
    check([(0, 200), (64, 10), (0, 30), (20, 100), (64, 1), (10, 3)])    # 64 lies in block 1, the last one: 0 stays held
    check([(0, 200), (64, 10), (0, 30), (20, 100), (10, 3), (12, 60), (71, 1), (64, 3), (40, 90)])
    check([(0, 128), (127, 1), (64, 64), (127, 1), (128, 1), (100, 1)])  # ends and starts on the boundaries


@pytest.mark.parametrize('d', [64, 128])
def test_where_each_byte_lies(d):
    """The order of csrc/quantized_cache.cuh on real buffers: integers that are their own quantised form (largest magnitude 127)."""
    from qwen3_triton.inference import quantized as Q
    g = torch.Generator().manual_seed(3)
    b, h, t = 2, 2, 150
    k, v = (torch.randint(-126, 127, (b, t, h, d), generator=g) for _ in range(2))
    for x in (k, v):
        x[:, 5::64, :, 3] = 127
    cache = make(b, h, t, d, torch.bfloat16)
    Q.append(k.bfloat16().cuda(), v.bfloat16().cuda(), cache, 0)
    row, dim = torch.arange(64)[:, None], torch.arange(d)[None]
    key = (row // 8 * (d // 64) + dim // 64) * 512 + row % 8 * 64 + dim % 64
    value = dim * 64 + row // 2 % 4 * 16 + row // 8 * 2 + row % 2
    for got, scales, x, place in ((cache.keys, cache.key_scales, k, key), (cache.values, cache.value_scales, v, value)):
        blocks = x[:, :128].transpose(1, 2).reshape(b, h, 2, 64, d)
        want = torch.empty(b, h, 2, 64 * d, dtype=torch.uint8)
        want[..., place.reshape(-1)] = (blocks + 128).to(torch.uint8).reshape(b, h, 2, 64 * d)
        assert torch.equal(got[:, :, :2].cpu(), want)
        assert torch.equal(scales[:, :, :2].cpu(), torch.ones(b, h, 2))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('held', [0, 1, 64, 100, 128])
def test_tokens_that_were_never_appended_are_reported_on_block_boundaries_too(dtype, held):
    from qwen3_triton.inference import quantized as Q
    h, d, t = 1, 64, 600
    k, v = tokens(1, t, h, d, dtype, 70)
    cache = make(1, h, t, d, dtype)
    if held:
        Q.append(part(k, 0, held), part(v, 0, held), cache, 0)
    cache.keys.fill_(7), cache.values.fill_(9), cache.key_scales.fill_(1), cache.value_scales.fill_(1)     # finite, whatever is read
    if held:
        Q.append(part(k, 0, held), part(v, 0, held), cache, 0)
    marks = cache.marks.clone()
    for end in (64, 192, 256):
        for call in (lambda: Q.read(cache, end), lambda: Q.read(cache, lengths(end), 0, end), lambda: Q.read(cache, end, end - 1),
                     lambda: Q.attention(randn((1, 1, 2, d), 1, dtype).cuda(), cache, end - 1),
                     lambda: Q.attention(randn((1, 40, 2, d), 1, dtype).cuda(), cache, end - 40)):
            call()
            assert reported() == (end > held), end
    Q.append(part(k, 192, 200), part(v, 192, 200), cache, 192)                # a gap before a block: nothing is written
    assert reported() and torch.equal(cache.marks, marks)
    Q.append(part(k, 192, 300), part(v, 192, 300), cache, 192)                # blocks beyond the gap: reported until it is filled
    assert reported()
    for s in (1, 40):
        Q.attention(randn((1, s, 2, d), 1, dtype).cuda(), cache, 300 - s)
        assert reported()
    Q.read(cache, 300, 256)
    assert reported()
    if held >= 64:
        expect_read(Q.read(cache, 64)[0][0], k[0], 64)                        # what was whole is whole
        assert not reported()
    Q.append(part(k, 300, 310), part(v, 300, 310), cache, 300)
    assert reported()
    first = held // 64 * 64                                                   # the ring holds blocks 3 and 4
    Q.append(part(k, first, 310), part(v, first, 310), cache, first)
    assert not reported()
    expect_read(Q.read(cache, 310)[0][0], k[0], 310)
    q = randn((1, 40, 2, d), 2, dtype)
    expect_attention(Q.attention(q.cuda(), cache, 270)[0], q[0], k[0, :310], v[0, :310], 270, dtype)
    assert not reported()


def test_a_gap_is_filled_from_where_the_sequence_ended():
    from qwen3_triton.inference import quantized as Q
    dtype, h, d = torch.bfloat16, 1, 64
    k, v = tokens(1, 300, h, d, dtype, 71)
    cache = make(1, h, 300, d, dtype)
    Q.append(part(k, 0, 100), part(v, 0, 100), cache, 0)
    Q.append(part(k, 128, 192), part(v, 128, 192), cache, 128)                # block 2; block 1 is held up to token 100
    assert reported()
    Q.read(cache, 192)
    assert reported()
    Q.append(part(k, 100, 200), part(v, 100, 200), cache, 100)
    assert not reported()
    expect_read(Q.read(cache, 200)[0][0], k[0], 200)
    expect_read(Q.read(cache, 200)[1][0], v[0], 200)
    assert not reported()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_every_quotient_of_significands_rounds_as_in_exact_arithmetic(dtype):
    """A block for every significand A of the largest magnitude, with all x = X 2^-k of the type below it: quotients 127 X 2^-k / A
    as near to a tie as they come (0.50000192 for X = 2047, k = 8, A = 2031), in whole numbers on the host's side."""
    from qwen3_triton.inference import quantized as Q
    bits, d = (8, 128) if dtype == torch.bfloat16 else (11, 128)
    low = 1 << (bits - 1)
    a = torch.arange(low, 2 * low, device='cuda')
    row, dim = torch.arange(64, device='cuda')[:, None], torch.arange(d, device='cuda')[None]
    places = ((row // 8 * (d // 64) + dim // 64) * 512 + row % 8 * 64 + dim % 64, dim * 64 + row // 2 % 4 * 16 + row // 8 * 2 + row % 2)
    cache = make(1, low, 64, d, dtype)
    given, wanted = [], []
    for first in (0, 1):                                                      # keys: k = 0..7, values: k = 1..8
        k = torch.arange(first, first + 8, device='cuda')[:, None]
        x = torch.arange(low, 2 * low, device='cuda')[None].expand(8, low)
        x, k = x.reshape(1, -1), k.expand(8, low).reshape(1, -1)              # [1, 8 low]
        over = a[:, None] << k                                                # the quotient is 127 x / over
        x = torch.where(x <= over, x, torch.zeros_like(x))
        whole = (254 * x + over) // (2 * over)
        whole -= (((254 * x + over) % (2 * over) == 0) & (whole % 2 == 1)).long()            # halves to even
        value = x.double() * torch.exp2(-k.double())
        sign = 1 - 2 * (torch.arange(x.shape[1], device='cuda') % 3 == 0).long()
        fill = torch.zeros(low, 64 * d, dtype=torch.float64, device='cuda')
        want = torch.zeros(low, 64 * d, dtype=torch.int64, device='cuda')
        n = min(x.shape[1], 64 * d - 1)
        fill[:, 1:n + 1], want[:, 1:n + 1] = (value * sign)[:, :n], (whole * sign)[:, :n]
        fill[:, 0], want[:, 0] = a.double(), 127
        given.append(fill.to(dtype).view(low, 64, d).transpose(0, 1)[None].contiguous())
        assert torch.equal(given[-1].double(), fill.view(low, 64, d).transpose(0, 1)[None])
        wanted.append(want)
    Q.append(*given, cache, 0)
    for got, want, place in zip((cache.keys, cache.values), wanted, places):
        assert torch.equal(got[0, :, 0][:, place.reshape(-1)].long() - 128, want)


def test_scores_far_from_zero_that_are_exact():
    """Scores of several thousand that fp32 holds exactly: equal ones average the values, and of two sizes the larger takes all."""
    from qwen3_triton.inference import quantized as Q
    for s in (1, 3, 40):
        for t, later in ((150, 0), (1000, 0), (150, 100), (1000, 700)):
            dtype, d = torch.bfloat16, 64
            k, v = torch.zeros(1, t, 1, d), randn((1, t, 1, d), 81)
            k[..., 0] = 127 * 64.0                                            # n = 127 with a scale of 64, and 8128 as given
            if later:
                k[:, later:, :, 0] = -127 * 64.0
            q = torch.zeros(1, s, 4, d)
            q[..., 0] = 4.0                                                   # scores of 4064, or -4064
            k, v, q = k.to(dtype), v.to(dtype), q.to(dtype)
            cache = make(1, 1, t, d, dtype)
            Q.append(k.cuda(), v.cuda(), cache, 0)
            out = Q.attention(q.cuda(), cache, t - s)[0].double().cpu()
            want, scale, _ = OQ.attention(q[0], OQ.held(k[0], t), OQ.held(v[0], t), t - s)
            # with scale * log2(e) in fp32 a score is off by 2^-23 of itself at most, 4064 * 1.45 * 2^-23 < 2^-10 in the exponent, the same
            # for equal scores; the weights' and the result's rounding as for any scores
            bound = 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9) * (scale + want.abs())
            assert float(((out - want).abs() - bound).max()) <= 0, (s, t, later)


@pytest.mark.parametrize('capacity', [1001, 5000, 300000])
def test_a_cache_much_longer_than_its_sequences(capacity):
    """With lengths on the device a call is cut for the whole capacity: most pieces then have no tokens."""
    from qwen3_triton.inference import quantized as Q
    dtype, b, h, hq, d = torch.bfloat16, 3, 2, 8, 128
    held = (1001, 64, 65)
    k, v = tokens(b, 1001, h, d, dtype, 91)
    cache = make(b, h, capacity, d, dtype)
    Q.append(k.cuda(), v.cuda(), cache, 0, lengths(*held))
    for s in (1, 4, 30):
        q = randn((b, s, hq, d), 92, dtype)
        out = Q.attention(q.cuda(), cache, lengths(*(n - s for n in held)))
        for i, n in enumerate(held):
            expect_attention(out[i], q[i], k[i, :n], v[i, :n], n - s, dtype)
    assert not reported()
