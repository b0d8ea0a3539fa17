"""The decode-time cache in 8 bits: tokens quantised as they are written, read back, and attended over.

Beside the 16-bit operators of kernels.py: `append` and `attention` take the same tensors with a QuantizedCache in
place of the two cache tensors. Per kv head, every complete block of 64 tokens is held as 8-bit integers with one scale
for its keys and one for its values (largest magnitude / 127, halves to even); the incomplete last block is held as
given. What a cache holds therefore depends on its tokens alone, not on how they were cut into calls. A block of which
an element is NaN or infinite reads back as NaN.

Lengths are Python ints (the same for every sequence) or int64 CUDA tensors [B], which the kernels read when they run:
a step captured into a CUDA graph follows them. Ints are checked here; what a tensor holds (with `count` also whether
start and count together fit) is checked on the device, where a violation leaves the sequence alone and shows in the
status word (_abi.raise_on_status).
"""
import ctypes
import operator

import torch

from .. import _abi

BLOCK = 64
_DTYPES = (torch.bfloat16, torch.float16)
_MOST_READ = 65535 * BLOCK - BLOCK


class QuantizedCache:
    """Buffers of a cache for `batch` sequences of up to `capacity` tokens: `heads` kv heads of `head_dim` 64 or 128, of
    a model in bfloat16 or float16. 1 byte per element, plus 4 bytes of scale per block and the last two blocks in 16
    bits. The integers lie in an order of the kernels' own: `read` gives the values. The buffers are made once and stay."""

    def __init__(self, batch, heads, capacity, head_dim, *, dtype=torch.bfloat16, device='cuda'):
        if min(batch, heads, capacity) < 1 or capacity > 2 ** 30 or batch * heads > 2 ** 24 or heads > 2 ** 16:
            raise ValueError('Expected positive sizes, at most 2**30 tokens and 2**24 (sequence, head) pairs')
        if head_dim not in (64, 128):
            raise ValueError('head_dim 64 or 128 required')
        if dtype not in _DTYPES:
            raise TypeError(f'unsupported dtype {dtype}; bfloat16 or float16 required')
        if torch.device(device).type != 'cuda':
            raise ValueError('A CUDA device is required; no fallback')
        self.batch, self.heads, self.capacity, self.head_dim, self.dtype = batch, heads, capacity, head_dim, dtype
        blocks = -(-capacity // BLOCK)
        payload, recent = (batch, heads, blocks, BLOCK * head_dim), (batch, heads, 2, BLOCK * head_dim)
        self.keys, self.values = (torch.empty(payload, dtype=torch.uint8, device=device) for _ in range(2))
        self.key_scales, self.value_scales = (torch.empty(payload[:3], dtype=torch.float32, device=device) for _ in range(2))
        # only complete blocks are read from the four above; what the ring does not hold yet meets weights of 0 and must be finite
        self.recent_keys, self.recent_values = torch.zeros((2, *recent), dtype=dtype, device=device)
        self.marks = torch.zeros((batch, heads, 2, 2, 4), dtype=torch.int32, device=device)
        self.device = self.keys.device
        # what every call passes, made once: the host struct with the buffers' addresses, and the device's status word
        self._struct = _abi.QuantizedCacheView(
            self.keys.data_ptr(), self.values.data_ptr(), self.key_scales.data_ptr(), self.value_scales.data_ptr(),
            self.recent_keys.data_ptr(), self.recent_values.data_ptr(), self.marks.data_ptr(),
            batch, heads, capacity, head_dim, _abi.dt(dtype))
        self._view = ctypes.addressof(self._struct)
        self._status = _abi.status_word(self.device).data_ptr()


def _elsewhere(cache):
    return torch._C._cuda_getDevice() != cache.device.index


def _launch(entry, cache, *args):
    """Call a C entry for a cache on the current device, on its current stream. (The raw handle: the stream object that
    torch.cuda.current_stream() makes costs more than the launch of a small kernel.)"""
    code = entry(cache._view, *args, cache._status, torch._C._cuda_getCurrentRawStream(cache.device.index))
    if code:
        _abi.check(code, entry.__name__)


def _length(value, cache, most, what):
    """(host number, device tensor or None) of a length: an int in [0, most] or an int64 CUDA tensor [B]."""
    if isinstance(value, torch.Tensor):
        if value.dtype != torch.int64 or value.shape != (cache.batch,):
            raise ValueError(f'{what}: an int or an int64 tensor of {cache.batch} lengths required')
        if value.device != cache.device or not value.is_contiguous():
            raise ValueError(f'{what}: a contiguous tensor on the device of the cache required')
        return 0, value
    number = operator.index(value)
    if not 0 <= number <= most:
        raise ValueError(f'{what} {number} does not fit the cache')
    return number, None


def _counts(count, cache):
    if count is None:
        return None
    if not isinstance(count, torch.Tensor):
        raise ValueError('count: None or an int64 tensor [B] required')
    return _length(count, cache, 0, 'count')[1]


def _check_tokens(tensors, cache):
    dtype, device = cache.dtype, cache.device
    if not all([t.is_cuda and t.dtype == dtype and t.device == device and t.is_contiguous() for t in tensors]):
        raise ValueError('Contiguous CUDA tensors of the type and on the device of the cache required; no fallback')


def append(k, v, cache, start, count=None):
    """Write the new k, v [B,S,H,D] into the cache after `start` tokens of each sequence. With `count` (int64 [B]) only
    the first count[b] of the S tokens are real; the rest is padding. A sequence may go back, by a `start` below its
    length, to any multiple of 64 or to any token of its last two blocks (once it has gone back to an earlier block, only of
    that one, until it begins the next). Any other start inside a block, and a start beyond the length (tokens are missing
    or no longer held as given), shows in _abi.raise_on_status: the sequence stays as it was if the block of `start` would
    have stayed incomplete; else other tokens stand in their place, and every call that reaches a block without its own
    reports so, until that is written anew. So does a read or attention over tokens that were never appended."""
    if k.ndim != 4 or k.shape != v.shape:
        raise ValueError('Expected k, v [B,S,H,D]')
    b, s, h, d = k.shape
    if b != cache.batch or h != cache.heads or d != cache.head_dim:
        raise ValueError('Expected k, v of the batch, heads and head_dim of the cache')
    if s < 1 or s > cache.capacity:
        raise ValueError('New tokens do not fit the cache')
    _check_tokens((k, v), cache)
    if _elsewhere(cache):
        with torch.cuda.device(cache.device):
            return append(k, v, cache, start, count)
    start, starts = _length(start, cache, cache.capacity - (s if count is None else 0), 'start')
    counts = _counts(count, cache)
    _launch(_abi.lib().q3_qcache_append, cache, k.data_ptr(), v.data_ptr(), s, start, _abi.ptr(starts), _abi.ptr(counts))


def read(cache, length, start=0, tokens=None):
    """(keys, values) [B,H,tokens,D] in the cache's type: tokens start .. start + tokens - 1 of sequences that hold
    `length` tokens, zero at and past the length. `tokens` may be left out where both are ints: up to the length."""
    held, lengths = _length(length, cache, cache.capacity, 'length')
    first, firsts = _length(start, cache, cache.capacity, 'start')
    if tokens is None:
        if lengths is not None or firsts is not None:
            raise ValueError('tokens is required with lengths on the device')
        tokens = held - first
    if not 0 <= tokens <= _MOST_READ:
        raise ValueError(f'Expected between 0 and {_MOST_READ} tokens')
    if _elsewhere(cache):
        with torch.cuda.device(cache.device):
            return read(cache, length, start, tokens)
    shape = (cache.batch, cache.heads, tokens, cache.head_dim)
    k, v = torch.empty(shape, dtype=cache.dtype, device=cache.device), torch.empty(shape, dtype=cache.dtype, device=cache.device)
    if tokens:
        _launch(_abi.lib().q3_qcache_read, cache, k.data_ptr(), v.data_ptr(), tokens, held, _abi.ptr(lengths), first, _abi.ptr(firsts))
    return k, v


def attention(q, cache, start, count=None):
    """q [B,S,Hq,D], the queries of the S newest tokens (already appended), against the cache, causal: the query of new
    token s sees tokens 0 .. start + s. Returns [B,S,Hq,D]; rows of padding (s >= count[b]) are zero."""
    if q.ndim != 4:
        raise ValueError('Expected q [B,S,Hq,D]')
    b, s, hq, d = q.shape
    if b != cache.batch or d != cache.head_dim or hq < 1 or hq % cache.heads:
        raise ValueError('Expected q of the batch and head_dim of the cache, its heads a multiple of the cache\'s')
    if s < 1 or s > cache.capacity:
        raise ValueError('Query does not match the cache')
    _check_tokens((q,), cache)
    if _elsewhere(cache):
        with torch.cuda.device(cache.device):
            return attention(q, cache, start, count)
    start, starts = _length(start, cache, cache.capacity - (s if count is None else 0), 'start')
    counts = _counts(count, cache)
    out = torch.empty_like(q)
    lib = _abi.lib()
    need = lib.q3_qcache_attention_workspace_bytes(cache._view, s, hq, start if starts is None else -1)
    ws = torch.empty(need, dtype=torch.uint8, device=cache.device) if need else None
    _launch(lib.q3_qcache_attention, cache, q.data_ptr(), out.data_ptr(), _abi.ptr(ws), need, s, hq, start, _abi.ptr(starts),
            _abi.ptr(counts), d ** -0.5)
    return out
