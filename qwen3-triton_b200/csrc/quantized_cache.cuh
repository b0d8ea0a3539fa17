// Layout of the 8-bit key/value cache and the device helpers its kernels share.
//
// Tokens are held in blocks of 64. A complete block of one (sequence, kv head) is 64 * D bytes of keys and as many of
// values, with one fp32 scale each; the last 128 tokens are also kept as they were given, in a ring of two
// blocks ("recent"), so that the incomplete block is exact and a block gets its scale from its own tokens,
// however the appends were cut (marks say what of it can be relied on: tokens of the last two blocks). Both forms store
// their elements in the order in which the tensor-core fragments of attention read them, so that a warp's loads are
// consecutive 16-byte pieces:
//   keys    [token / 8][dim / 64][token % 8][dim % 64]      lane (g, t) of a warp: token 8i + g, dims 64c + 16t .. +15
//   values  [dim][(token / 2) % 4][token / 8][token % 2]    lane (g, t): dim 8m + g, tokens 8i + 2t, 8i + 2t + 1, i = 0..7
// (the pair of tokens a lane holds of the value fragment is the pair of scores it holds of the score fragment).
// An integer n is stored as the byte n + 128: two bytes put below 0x64 in a byte permute are the fp16 numbers 1024 + byte,
// one packed subtraction of 1152 away from n.
#pragma once
#include "common.cuh"

namespace q3 {
namespace qc {

constexpr int kBlock = 64;   // tokens per block

__host__ __device__ constexpr int key_offset(int token, int dim, int D) {
  return ((token >> 3) * (D >> 6) + (dim >> 6)) * 512 + (token & 7) * 64 + (dim & 63);
}
__host__ __device__ constexpr int value_column(int token) { return ((token >> 1) & 3) * 16 + (token >> 3) * 2 + (token & 1); }
__host__ __device__ constexpr int value_offset(int token, int dim) { return dim * kBlock + value_column(token); }

// What the ring holds: slot (block % 2) of a (sequence, head) holds the first `fill` tokens of `block`. `bad` is 0, or 1 +
// the first of them that had a NaN or an infinity (those are stored as 0); `amax` is at least their largest magnitude, and at
// most 2^10 times as much (attention takes them to fp16 by a power of two). One mark for the keys and one for the values. A
// block that was completed without its earlier tokens has -fill: its length counts, its tokens cannot be relied on.
// `torn`, the same in all marks of a (sequence, head): 0, or 1 + the first complete block of which tokens were missing when it, or
// a later one, was completed; whoever reads it or what follows is told so, until it is written anew from its first token.
struct Mark {
  int block;
  short fill, bad;
  int torn;
  float amax;
};

struct Cache {
  uint8_t* payload[2];     // keys, values   [B, H, blocks, 64 * D], n + 128
  float* scales[2];        //                [B, H, blocks]
  void* recent[2];         //                [B, H, 2, 64 * D] in the model's type
  Mark* marks;             //                [B, H, 2 (keys, values), 2 (slots)]
  int64_t batch, heads, capacity, blocks;
};

inline Cache device_view(const q3_quantized_cache* c) {
  Cache d;
  d.payload[0] = (uint8_t*)c->keys; d.payload[1] = (uint8_t*)c->values;
  d.scales[0] = c->key_scales; d.scales[1] = c->value_scales;
  d.recent[0] = c->recent_keys; d.recent[1] = c->recent_values;
  d.marks = (Mark*)c->marks;
  d.batch = c->batch; d.heads = c->heads; d.capacity = c->capacity;
  d.blocks = cdiv(c->capacity, kBlock);
  return d;
}

inline int check_cache(const q3_quantized_cache* c) {
  if (!c || !c->keys || !c->values || !c->key_scales || !c->value_scales || !c->recent_keys || !c->recent_values || !c->marks)
    return Q3_ERR_ARG;
  if (c->dtype != Q3_BF16 && c->dtype != Q3_F16) return Q3_ERR_DTYPE;
  if (c->batch < 1 || c->heads < 1 || c->capacity < 1 || c->capacity > (int64_t)1 << 30 || (c->head_dim != 64 && c->head_dim != 128))
    return Q3_ERR_SHAPE;
  if (c->batch > (int64_t)1 << 24 || c->heads > (int64_t)1 << 16 || c->batch * c->heads > (int64_t)1 << 24) return Q3_ERR_SHAPE;
  if (!aligned16(c->keys) || !aligned16(c->values) || !aligned16(c->recent_keys) || !aligned16(c->recent_values) ||
      !aligned16(c->marks) || (reinterpret_cast<uintptr_t>(c->key_scales) & 3u) || (reinterpret_cast<uintptr_t>(c->value_scales) & 3u))
    return Q3_ERR_ALIGN;
  return Q3_OK;
}

#define Q3_DISPATCH_CACHE(C, T, D, ...)                                                                  \
  if ((C)->dtype == Q3_BF16) {                                                                           \
    using T = __nv_bfloat16;                                                                             \
    if ((C)->head_dim == 128) { constexpr int D = 128; __VA_ARGS__; } else { constexpr int D = 64; __VA_ARGS__; } \
  } else {                                                                                               \
    using T = __half;                                                                                    \
    if ((C)->head_dim == 128) { constexpr int D = 128; __VA_ARGS__; } else { constexpr int D = 64; __VA_ARGS__; } \
  }

#ifdef __CUDACC__
// Where a sequence stands: `start` tokens held before the call and `count` new ones. The values come from the host
// (the same for every sequence) or from device arrays; ok is false for what does not fit the cache.
struct Span {
  int64_t start, count;
  bool ok;
};
__device__ __forceinline__ Span span_of(int64_t b, int64_t S, int64_t capacity, int64_t start, const int64_t* starts,
                                        const int64_t* counts) {
  Span s;
  s.start = starts ? starts[b] : start;
  s.count = counts ? counts[b] : S;
  s.ok = s.start >= 0 && s.start <= capacity && s.count >= 0 && s.count <= S && s.count <= capacity - s.start;
  return s;
}

template <typename T> __device__ __forceinline__ void pair_to_f32(uint32_t w, float& a, float& b);
template <> __device__ __forceinline__ void pair_to_f32<__nv_bfloat16>(uint32_t w, float& a, float& b) {
  a = __uint_as_float(w << 16);
  b = __uint_as_float(w & 0xffff0000u);
}
template <> __device__ __forceinline__ void pair_to_f32<__half>(uint32_t w, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  a = f.x;
  b = f.y;
}

// Tokens that the two marks of a (sequence, head) speak for: its length after the last append.
__device__ __forceinline__ int held_tokens(const Mark& a, const Mark& b) {
  return max(a.block < 0 ? 0 : a.block * kBlock + abs(a.fill), b.block < 0 ? 0 : b.block * kBlock + abs(b.fill));
}
// Whether the first `tokens` tokens are held, none of their blocks torn. (That the incomplete block of a shorter length is
// still among the recent ones is another question.)
__device__ __forceinline__ bool held_whole(const Mark* marks, int tokens) {
  const Mark a = marks[0], b = marks[1];
  return tokens <= held_tokens(a, b) && (a.torn == 0 || tokens <= (a.torn - 1) * kBlock);
}

// two fp32 in one register pair: one instruction for both
__device__ __forceinline__ uint64_t pack_f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
#endif

}  // namespace qc
}  // namespace q3
