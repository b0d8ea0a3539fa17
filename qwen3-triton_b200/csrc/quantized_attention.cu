// Attention over the 8-bit key/value cache.
//
// With k_t = ks * n_t and v_t = vs * w_t (n, w the integers of a block, ks, vs its scales), a row of the result is
//   sum_t 2^{s'_t} w_t / sum_t 2^{s'_t - log2 vs},   s'_t = (q . n_t) * ks * scale * log2(e) + log2(vs):
// the scale of the values is part of the exponent, so the weights that meet the integers lie in [0, 1] whatever the blocks'
// scales are, and numerator and denominator keep a running reference each (m, ml). Weights are rounded to fp16 after a
// factor of 2^15: 11 bits down to 2^-29 of the largest. Integers are exact in fp16; queries in bf16 are taken to fp16 by a
// power of two per row, and the incomplete block's tokens by one per block: their elements reach 2^15 where integers reach 127,
// so their weights have 8 bits less of that room, and one 2^-39 of the block's largest (2^-29 where the mark holds a larger one)
// counts as zero. Products accumulate in fp32.
// The denominator adds up the weights too, block by block, with vs taken out again. Where vs is below 2^-kFar of the largest so
// far and the block's largest weight below 2^-kFar, the block counts with a larger vs, such that this weight is 2^-kFar: in fp16
// its weights are zero with either, and its share of the denominator does not flush. The last factor 2^{m - ml} / sum reaches
// beyond fp32's exponents and is applied as two halves.
#include "quantized_cache.cuh"
#include "tcgen05.cuh"
#include <math_constants.h>
#include <type_traits>
#include <utility>

namespace q3 {
namespace qc {

struct AttendParams {
  Cache c;
  const void* q;
  void* out;
  float* part;             // [rows of out][splits][D], normalised within the split
  float* lse;              // [rows of out][splits], log2, up to a constant
  int64_t S, start;
  const int64_t* starts;
  const int64_t* counts;
  bool joined;             // the splits of a (sequence, head) are one cluster and join their results themselves
  int Hq, group, rows, tiles, splits;   // rows = S * group of one kv head; `tiles` of 256 where there are many
  float scale_log2;
  int* status;
};

constexpr float kFar = 64.f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// four bytes n + 128 -> two pairs of fp16 n
__device__ __forceinline__ void widen4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));    // 1152
  const __half2 x = __hsub2(*reinterpret_cast<const __half2*>(&a), bias), y = __hsub2(*reinterpret_cast<const __half2*>(&b), bias);
  lo = *reinterpret_cast<const uint32_t*>(&x);
  hi = *reinterpret_cast<const uint32_t*>(&y);
}
// a pair of 16-bit elements of the model's type, times a power of two, as fp16
template <typename T> __device__ __forceinline__ uint32_t to_half_pair(uint32_t w, float up);
template <> __device__ __forceinline__ uint32_t to_half_pair<__half>(uint32_t w, float) { return w; }
template <> __device__ __forceinline__ uint32_t to_half_pair<__nv_bfloat16>(uint32_t w, float up) {
  return pack_half(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
}
// the same of recent tokens: one that `up` does not speak for, because it is not counted in, must not become infinite - its
// weight of 0 would make NaN of it
template <typename T> __device__ __forceinline__ uint32_t recent_pair(uint32_t w, float up) {
  float a, b;
  pair_to_f32<T>(w, a, b);
  return pack_half(fminf(fmaxf(a * up, -65504.f), 65504.f), fminf(fmaxf(b * up, -65504.f), 65504.f));
}
// The power of two that takes magnitudes up to `amax` below 2^15, as far as fp32 holds it and its reciprocal: the largest for
// zeros. Recent tokens take it in both types: their weights then hold their size, as those of complete blocks hold their
// scale, and neither takes the other's digits. Queries take it in bf16 only: fp16 is what they are to become.
__device__ __forceinline__ float up_scale(float amax) {
  int e = 14 - ((int)(__float_as_uint(amax) >> 23) - 127);
  e = e > 126 ? 126 : (e < -126 ? -126 : e);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}
template <typename T> __device__ __forceinline__ float query_scale(float amax) { return up_scale(amax); }
template <> __device__ __forceinline__ float query_scale<__half>(float) { return 1.f; }

// Largest magnitude of the first `live` tokens of a ring slot, by the whole CTA: where fewer tokens are counted in than the
// slot's mark speaks for, its amax may be of others that dwarf them.
template <typename T, int D, bool V> __device__ __forceinline__ float live_amax(const T* ring, int live, float* red) {
  float m = 0.f;
#pragma unroll 1
  for (int at = threadIdx.x; at < kBlock * D; at += blockDim.x) {
    const int col = at & 63;
    const int token = V ? ((col >> 1) & 7) * 8 + (col >> 4) * 2 + (col & 1) : at / (512 * (D / 64)) * 8 + (at & 511) / 64;
    if (token < live) m = fmaxf(m, fabsf(to_f32<T>(ring[at])));
  }
  return block_max(m, red);
}
// A mark as `need` tokens see it.
template <typename T, int D> __device__ __forceinline__ void narrow_marks(Mark (&mark)[2], const Cache& c, int64_t bh, int block, int need, float* red) {
  const int64_t at = (bh * 2 + (block & 1)) * (kBlock * D);
  if (mark[0].fill != need) {
    mark[0].amax = live_amax<T, D, false>((const T*)c.recent[0] + at, need, red);
    mark[1].amax = live_amax<T, D, true>((const T*)c.recent[1] + at, need, red);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) mark[i].bad = mark[i].bad > 0 && mark[i].bad <= need;
}

__device__ __forceinline__ void mma_16816_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                              uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ float load_cluster(uint32_t cluster_addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(cluster_addr) : "memory");
  return v;
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Few query rows (decoding, drafted tokens): the cache is streamed once and the work is bound by HBM. One CTA takes the up to
// 8 * NT rows - new tokens x query heads - of one kv head, and every splits-th unit (block of 64 tokens) of the sequence; its
// four or eight warps take turns. A warp is on its own until the end: it brings whole blocks into its own ring of shared-memory slots
// by bulk copies (the layout puts a block's keys, and its values, in one piece), two or three of them in flight, and reads them back
// as tensor-core fragments without bank conflicts. Keys (and value columns) are the 16 rows of the MMA tile and the query rows
// its 8 columns, so a group of up to 8 query heads fills the tile: S^T = K Q^T, O^T = V^T P^T. Short sequences are a matter of
// latency: the first copies leave before anything else is looked up, and products that follow one another go to different
// accumulators. 32 query / 8 kv heads of 128 in bf16: 64 sequences of 8001 tokens 157 us (6.7 TB/s), 4 of 131001 160 us, one of
// 1501 9.5 us, of which a CTA needs 1 us until its copies have left and 1.5 us for its first block.
constexpr int ring_bytes(int warps) { return warps == 4 ? 24576 : 16384; }   // per warp

template <typename T, int D, int NT, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 8 / WARPS)
attention_split_kernel(const AttendParams p) {
  constexpr int kSplitWarps = WARPS, kRingBytes = ring_bytes(WARPS);
  constexpr int SLOT = kBlock * D, SLOTS = kRingBytes / SLOT, CH = D / 64, ROWS = 8 * NT;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kSplitWarps * SLOTS];
  __shared__ int abort_word;
  __shared__ float red[32];
  __shared__ float s_row[ROWS][D], s_sum[ROWS];                    // this CTA's rows, for the other CTAs of its cluster
  volatile int* abort_flag = &abort_word;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.x % p.splits, bh = blockIdx.x / p.splits;
  const int b = bh / (int)p.c.heads, kvh = bh - b * (int)p.c.heads;
  const uint32_t bar0 = tc::smem_u32(bars + warp * SLOTS), ring = tc::smem_u32(smem) + warp * kRingBytes;
  if (threadIdx.x == 0) *abort_flag = 0;
  if (lane == 0) {
    for (int i = 0; i < SLOTS; ++i) tc::mbar_init(bar0 + 8u * i, 1);
    tc::fence_barrier_init();
  }
  Span sp = span_of(b, p.S, p.c.capacity, p.start, p.starts, p.counts);
  const bool fits = sp.ok;
  if (!fits) sp.start = sp.count = 0;
  // tokens the rows see: up to the last real row's own
  const int start = (int)sp.start, count = (int)sp.count, end = start + count;      // a cache has at most 2^30 tokens
  const int seen = count > 0 ? end : 0, complete = end / kBlock;
  int full = (seen + kBlock - 1) / kBlock;
  bool tail = full > complete;
  if (tail) full = complete;
  // this warp's units: split + (warp + WARPS k) * splits
  const int first = split + warp * p.splits, stride = kSplitWarps * p.splits;
  const int mine = first < full ? (full - first + stride - 1) / stride : 0;
  const uint8_t* kbase = p.c.payload[0] + (int64_t)bh * p.c.blocks * SLOT;
  const uint8_t* vbase = p.c.payload[1] + (int64_t)bh * p.c.blocks * SLOT;
  const int items = 2 * mine;
  auto issue = [&](int n) {                                        // lane 0
    const uint32_t bar = bar0 + 8u * (n % SLOTS);
    tc::mbar_expect_tx(bar, SLOT);
    bulk_load(ring + (n % SLOTS) * SLOT, ((n & 1) ? vbase : kbase) + (int64_t)(first + (n >> 1) * stride) * SLOT, SLOT, bar);
  };
  if (lane == 0)
    for (int n = 0; n < (items < SLOTS ? items : SLOTS); ++n) issue(n);
  // everything else that has to be fetched, at once
  const float* kscale = p.c.scales[0] + (int64_t)bh * p.c.blocks;
  const float* vscale = p.c.scales[1] + (int64_t)bh * p.c.blocks;
  float ks = 0.f, vs = 1.f;
  if (mine > 0) { ks = kscale[first]; vs = vscale[first]; }
  Mark both[2] = {};                                               // of the keys, thread 0
  if (threadIdx.x == 0) { both[0] = p.c.marks[bh * 4]; both[1] = p.c.marks[bh * 4 + 1]; }
  Mark mark[2];
  if (tail) {
    mark[0] = p.c.marks[(bh * 2 + 0) * 2 + (complete & 1)];
    mark[1] = p.c.marks[(bh * 2 + 1) * 2 + (complete & 1)];
  }
  // query fragments: column g of n-tile nt is row 8 nt + g; its 16 dims 64c + 16t .. +15 feed four MMAs
  uint4 qv[NT][CH][2];
  int s_of[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = 8 * nt + g;
    s_of[nt] = r / p.group;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      qv[nt][c][0] = qv[nt][c][1] = make_uint4(0u, 0u, 0u, 0u);
      if (r < p.rows) {
        const T* src = (const T*)p.q + (((int64_t)b * p.S + s_of[nt]) * p.Hq + kvh * p.group + r - s_of[nt] * p.group) * D + 64 * c + 16 * t;
        qv[nt][c][0] = *reinterpret_cast<const uint4*>(src);
        qv[nt][c][1] = *reinterpret_cast<const uint4*>(src + 8);
      }
    }
  }
  __syncthreads();                                                 // abort_flag
  if (!fits && threadIdx.x == 0) flag_status(p.status, Q3_STATUS_CACHE_RANGE);
  if (threadIdx.x == 0 && !held_whole(both, seen)) flag_status(p.status, Q3_STATUS_CACHE_RECENT);
  if (tail) {
    const int need = end - complete * kBlock;
    if (mark[0].block != complete || mark[0].fill < need || mark[1].block != complete || mark[1].fill < need) {
      if (threadIdx.x == 0) flag_status(p.status, Q3_STATUS_CACHE_RECENT);
      tail = false;
    } else {
      narrow_marks<T, D>(mark, p.c, bh, complete, need, red);
    }
  }

  uint32_t qf[NT][CH][4][2];
  float rowf[NT][2];                                               // of rows 2t, 2t + 1: scale * log2(e) / query's power of two
  int visible[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float amax = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t w[4] = {qv[nt][c][i].x, qv[nt][c][i].y, qv[nt][c][i].z, qv[nt][c][i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)                                // only used for bf16
          amax = fmaxf(amax, fmaxf(__uint_as_float(w[e] << 16 & 0x7fffffffu), __uint_as_float(w[e] & 0x7fff0000u)));
      }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const float up = query_scale<T>(amax);
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        qf[nt][c][2 * i][0] = to_half_pair<T>(qv[nt][c][i].x, up);
        qf[nt][c][2 * i][1] = to_half_pair<T>(qv[nt][c][i].y, up);
        qf[nt][c][2 * i + 1][0] = to_half_pair<T>(qv[nt][c][i].z, up);
        qf[nt][c][2 * i + 1][1] = to_half_pair<T>(qv[nt][c][i].w, up);
      }
    const float f = p.scale_log2 / up;
    const int vis = 8 * nt + g < p.rows && s_of[nt] < count ? start + s_of[nt] + 1 : 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      rowf[nt][e] = __shfl_sync(0xffffffffu, f, (2 * t + e) * 4);
      visible[nt][e] = __shfl_sync(0xffffffffu, vis, (2 * t + e) * 4);
    }
  }
  // tokens that every row sees: no mask before them
  const int unmasked = ROWS <= p.rows && (ROWS - 1) / p.group < count ? start + 1 : 0;

  float m[NT][2], ml[NT][2], l[NT][2], o[NT][D / 16][4];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int e = 0; e < 2; ++e) { m[nt][e] = ml[nt][e] = -CUDART_INF_F; l[nt][e] = 0.f; }
#pragma unroll
    for (int i = 0; i < D / 16; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
  }
  float sc[NT][4][4];
  uint32_t pf[NT][8];
  bool ok = true;
  float top_lvs = -CUDART_INF_F;                                   // of the blocks so far

  // scores of 16 * IT tokens from `token` on -> weights in pf; o rescaled
  auto softmax = [&](auto it_count, int token, float ks, float vs) {
    constexpr int IT = decltype(it_count)::value;
    const float lvs = log2f(vs);
    const bool masked = token + 16 * IT > unmasked;
    top_lvs = fmaxf(top_lvs, lvs);
    const bool far = lvs < top_lvs - kFar;                         // only then can weights flush that count
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float alpha[2], ref[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float f = ks * rowf[nt][e];
        const int ahead = visible[nt][e] - token, limit = ahead - g;               // of these tokens, those that the row sees
        float mx = -CUDART_INF_F;
#pragma unroll
        for (int it = 0; it < IT; ++it)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float s = fmaf(sc[nt][it][2 * hf + e], f, lvs);
            if (masked && 16 * it + 8 * hf >= limit) s = -CUDART_INF_F;
            sc[nt][it][2 * hf + e] = s;
            mx = fmaxf(mx, s);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float nm = fmaxf(m[nt][e], mx);
        ref[e] = nm > -CUDART_INF_F ? nm : 0.f;
        float base = ref[e] - 15.f, d = ref[e] - lvs;
        if (far && mx > -CUDART_INF_F) {
          const float raise = fmaxf(ref[e] - kFar - mx, 0.f);      // of log2 vs
          base -= raise;
          d -= raise;
        }
        alpha[e] = exp2_fast(m[nt][e] - ref[e]);
        m[nt][e] = nm;
        float sum = 0.f;
#pragma unroll
        for (int it = 0; it < IT; ++it)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const float w = exp2_fast(sc[nt][it][2 * hf + e] - base);
            sc[nt][it][2 * hf + e] = w;
            sum += w;
          }
        if (ahead > 0) {                                           // the same in all lanes of a row
          const float nml = fmaxf(ml[nt][e], d);
          l[nt][e] = l[nt][e] * exp2_fast(ml[nt][e] - nml) + sum * exp2_fast(d - nml);
          ml[nt][e] = nml;
        }
      }
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        pf[nt][2 * it] = transpose_8x8(pack_half(sc[nt][it][0], sc[nt][it][1]));
        pf[nt][2 * it + 1] = transpose_8x8(pack_half(sc[nt][it][2], sc[nt][it][3]));
      }
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        o[nt][i][0] *= alpha[0]; o[nt][i][1] *= alpha[1]; o[nt][i][2] *= alpha[0]; o[nt][i][3] *= alpha[1];
      }
    }
  };
  auto clear_scores = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int it = 0; it < 4; ++it) sc[nt][it][0] = sc[nt][it][1] = sc[nt][it][2] = sc[nt][it][3] = 0.f;
  };
  // N fragments of a complete block: 16 bytes each per lane, of which word w holds two pairs
  auto word = [](const uint4& v, int w) { return w == 0 ? v.x : w == 1 ? v.y : w == 2 ? v.z : v.w; };
  auto keys8 = [&](uint32_t kt, int c) {                           // dims 64c .. +63 of the 64 tokens
    uint4 r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = lds16(kt + (i * CH + c) * 512 + lane * 16);
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int it = 0; it < 4; ++it) {                             // key groups 2 it, 2 it + 1
        uint32_t a0, a2, a1, a3;
        widen4(word(r[2 * it], w), a0, a2);
        widen4(word(r[2 * it + 1], w), a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816_f16(sc[nt][it], a0, a1, a2, a3, qf[nt][c][w][0], qf[nt][c][w][1]);
      }
  };
  auto values8 = [&](uint32_t vt, int m0) {                        // dims 16 m0 .. +63 of the 64 tokens
    uint4 r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = lds16(vt + (2 * m0 + i) * 512 + lane * 16);
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) {                                // dims 16 (m0 + i) .. +7, +8 .. +15
        uint32_t a0, a2, a1, a3;
        widen4(word(r[2 * i], w), a0, a2);
        widen4(word(r[2 * i + 1], w), a1, a3);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816_f16(o[nt][m0 + i], a0, a1, a2, a3, pf[nt][2 * w], pf[nt][2 * w + 1]);
      }
  };
  int taken = 0;                                                   // items waited for
  auto wait_item = [&]() {
    ok = ok && tc::mbar_wait(bar0 + 8u * (taken % SLOTS), (taken / SLOTS) & 1u, abort_flag);
    ok = __all_sync(0xffffffffu, ok);
    return ring + (taken % SLOTS) * SLOT;
  };
  auto release_item = [&]() {                                      // the slot has been read: its next item may land
    __syncwarp();
    if (lane == 0 && ok && taken + SLOTS < items) issue(taken + SLOTS);
    ++taken;
  };

  for (int k = 0; k < mine && ok; ++k) {
    const int j = first + k * stride;
    float ks_next = 0.f, vs_next = 1.f;
    if (k + 1 < mine) { ks_next = kscale[j + stride]; vs_next = vscale[j + stride]; }
    clear_scores();
    const uint32_t kt = wait_item();
    if (!ok) break;
#pragma unroll
    for (int c = 0; c < CH; ++c) keys8(kt, c);
    release_item();
    softmax(std::integral_constant<int, 4>(), j * kBlock, ks, vs);
    const uint32_t vt = wait_item();
    if (!ok) break;
#pragma unroll
    for (int m0 = 0; m0 < D / 16; m0 += 4) values8(vt, m0);
    release_item();
    ks = ks_next; vs = vs_next;
  }
  if (tail && full % p.splits == split && ok && warp < 4) {
    // The recent tokens: 16 for each of four warps, straight from memory (they have just been written and lie in L2).
    const int64_t ring_at = ((int64_t)bh * 2 + (complete & 1)) * SLOT;
    const T* kr = (const T*)p.c.recent[0] + ring_at;
    const T* vr = (const T*)p.c.recent[1] + ring_at;
    uint4 kw[CH][2][2];
    uint2 vw[D / 8];
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const T* src = kr + key_offset(16 * warp + 8 * u + g, 64 * c + 16 * t, D);
        kw[c][u][0] = *reinterpret_cast<const uint4*>(src);
        kw[c][u][1] = *reinterpret_cast<const uint4*>(src + 8);
      }
#pragma unroll
    for (int i = 0; i < D / 8; ++i) vw[i] = *reinterpret_cast<const uint2*>(vr + (8 * i + g) * kBlock + 16 * t + 4 * warp);
    const float kup = up_scale(mark[0].amax), vup = up_scale(mark[1].amax);
    clear_scores();
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint4 lo = kw[c][0][w >> 1], hi = kw[c][1][w >> 1];
        const uint32_t a0 = recent_pair<T>((w & 1) ? lo.z : lo.x, kup), a2 = recent_pair<T>((w & 1) ? lo.w : lo.y, kup);
        const uint32_t a1 = recent_pair<T>((w & 1) ? hi.z : hi.x, kup), a3 = recent_pair<T>((w & 1) ? hi.w : hi.y, kup);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_16816_f16(sc[nt][0], a0, a1, a2, a3, qf[nt][c][w][0], qf[nt][c][w][1]);
      }
    softmax(std::integral_constant<int, 1>(), complete * kBlock + 16 * warp, mark[0].bad ? CUDART_NAN_F : 1.f / kup,
            mark[1].bad ? CUDART_NAN_F : 1.f / vup);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      const uint32_t a0 = recent_pair<T>(vw[2 * i].x, vup), a2 = recent_pair<T>(vw[2 * i].y, vup);
      const uint32_t a1 = recent_pair<T>(vw[2 * i + 1].x, vup), a3 = recent_pair<T>(vw[2 * i + 1].y, vup);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma_16816_f16(o[nt][i], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
    }
  }
  if (!ok) {                                                       // nothing may still be landing when the CTA ends
    const int issued = taken + SLOTS < items ? taken + SLOTS : items;
    for (int n = taken; n < issued; ++n) tc::mbar_wait_drain(bar0 + 8u * (n % SLOTS), (n / SLOTS) & 1u);
  }
  __syncwarp();

  // this warp's rows, divided by their sums, and log2 of the sums, into its own ring
  constexpr int STRIDE = D + 4;
  float* s_part = reinterpret_cast<float*>(smem + warp * kRingBytes);          // [ROWS][D + 4]
  float* s_ref = reinterpret_cast<float*>(smem + warp * kRingBytes + ROWS * STRIDE * 4);     // log2 of the row's sum
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float sum = l[nt][e];
      sum += __shfl_xor_sync(0xffffffffu, sum, 4);
      sum += __shfl_xor_sync(0xffffffffu, sum, 8);
      sum += __shfl_xor_sync(0xffffffffu, sum, 16);
      const int r = 8 * nt + 2 * t + e;
      const float whole = ml[nt][e] + log2f(sum), half = sum == 0.f ? 0.f : exp2_fast(0.5f * (m[nt][e] - whole));
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        s_part[r * STRIDE + 16 * i + g] = o[nt][i][e] * half * half;
        s_part[r * STRIDE + 16 * i + 8 + g] = o[nt][i][2 + e] * half * half;
      }
      if (g == 0) s_ref[r] = sum == 0.f ? -CUDART_INF_F : whole;
    }
  __syncthreads();
  // rows shared out over the warps: the warps' results are weighted by their sums
  constexpr int CPL = D / 32;
  for (int r = warp; r < ROWS && r < p.rows; r += kSplitWarps) {
    // (the weights are divided by their sum before they are used: a sum of large rows may not be finite)
    float weight[kSplitWarps];
    float mx = -CUDART_INF_F, tot = 0.f, acc[CPL];
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      weight[w] = *reinterpret_cast<const float*>(smem + w * kRingBytes + ROWS * STRIDE * 4 + r * 4);
      mx = fmaxf(mx, weight[w]);
    }
    const float at = mx > -CUDART_INF_F ? mx : 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      weight[w] = exp2_fast(weight[w] - at);
      tot += weight[w];
    }
    const float inv = tot == 0.f ? 0.f : 1.f / tot;
#pragma unroll
    for (int c = 0; c < CPL; ++c) acc[c] = 0.f;
#pragma unroll
    for (int w = 0; w < kSplitWarps; ++w) {
      const float f = weight[w] * inv;
      const float* src = reinterpret_cast<const float*>(smem + w * kRingBytes) + r * STRIDE + lane;
#pragma unroll
      for (int c = 0; c < CPL; ++c) acc[c] = fmaf(f, src[32 * c], acc[c]);
    }
    const int s = r / p.group;
    const int64_t orow = ((int64_t)b * p.S + s) * p.Hq + kvh * p.group + r - s * p.group;
    if (p.joined) {
#pragma unroll
      for (int c = 0; c < CPL; ++c) s_row[r][lane + 32 * c] = acc[c];
      if (lane == 0) s_sum[r] = tot == 0.f ? -CUDART_INF_F : at + log2f(tot);
    } else if (p.splits == 1) {
#pragma unroll
      for (int c = 0; c < CPL; ++c) ((T*)p.out)[orow * D + lane + 32 * c] = from_f32<T>(acc[c]);
    } else {
      const int64_t at_part = orow * p.splits + split;
#pragma unroll
      for (int c = 0; c < CPL; ++c) p.part[at_part * D + lane + 32 * c] = acc[c];
      if (lane == 0) p.lse[at_part] = tot == 0.f ? -CUDART_INF_F : at + log2f(tot);
    }
  }
  if (p.joined) {
    // rows shared out over the CTAs of the cluster and their warps, each weighted by the sums of all splits
    tc::cluster_sync_all();
    for (int r = split + warp * p.splits; r < ROWS && r < p.rows; r += kSplitWarps * p.splits) {
      float sum = -CUDART_INF_F;
      if (lane < p.splits) sum = load_cluster(tc::mapa_u32(tc::smem_u32(&s_sum[r]), lane));
      const float mx = warp_max(sum), at = mx > -CUDART_INF_F ? mx : 0.f;
      const float part = exp2_fast(sum - at), tot = warp_sum(part), mine = tot == 0.f ? 0.f : part / tot;
      float acc[CPL];
#pragma unroll
      for (int c = 0; c < CPL; ++c) acc[c] = 0.f;
      for (int i = 0; i < p.splits; ++i) {
        const uint32_t src = tc::mapa_u32(tc::smem_u32(&s_row[r][lane]), i);
        const float w = __shfl_sync(0xffffffffu, mine, i);
#pragma unroll
        for (int c = 0; c < CPL; ++c) acc[c] = fmaf(w, load_cluster(src + 128 * c), acc[c]);
      }
      const int s = r / p.group;
      const int64_t orow = ((int64_t)b * p.S + s) * p.Hq + kvh * p.group + r - s * p.group;
#pragma unroll
      for (int c = 0; c < CPL; ++c) ((T*)p.out)[orow * D + lane + 32 * c] = from_f32<T>(acc[c]);
    }
    tc::cluster_sync_all();                                        // nobody leaves while its rows are read
  }
  if (threadIdx.x == 0 && *abort_flag) flag_status(p.status, Q3_STATUS_WAIT_TIMEOUT);
}

// Many query rows (prompts, chunks of prompts): bound by the tensor cores. One CTA takes 256 rows of one kv head as two
// tiles of 128 and walks the keys 128 (two blocks) at a time:
//   warps 0-3    widen: blocks come from global memory to registers one tile ahead (their order makes that coalesced) and go to
//                shared memory as fp16, 128-byte swizzled, as K [key][dim] and V^T [dim][key]: both K-major for the tensor
//                cores. About 12 instructions per 16 bytes, shared by 256 rows. Keys are placed in the order in which the values
//                are stored: weights and values agree without a shuffle. (Bulk copies to shared memory first cost 40 % more
//                shared-memory traffic there, and the products need most of that bandwidth.)
//   warps 4-11   softmax, one row per thread, the scores of a block at a time in registers: weights under a reference that trails
//                the row's maximum by less than 2^8 (fp16 weights have the room: they start at 2^7), back to tensor memory over
//                the scores they came from, as the A operand of the second product. Only when a row outgrows its reference are
//                the sums in tensor memory rescaled.
//   warps 12, 13 issue the products, one tile each: while one tile's weights are computed, the other tile's products run
// 32 query / 8 kv heads of 128 in bf16: 512 tokens over 32000 302 us (900 TFLOP/s; products alone 163 us at the measured rate), two
// prompts of 4096 332 us. Bound by the chain scores -> exponentials -> weights -> products of a tile, which has one place for scores
// and weights: about 4000 cycles per 256 x 128 against 2050 of products, and as many of shared memory (256 KB per step, operands
// read and widened tiles written, at 128 bytes a cycle). The exponentials of the two tiles take turns (when that was built, the
// first case took 297 us, at once 385). Some 20000 cycles per CTA pass before its first and after its last step.
// Registers move from the other warps to the softmax's: 128 threads x (120 + 56) + 256 x 168 = 512 x 128 at launch.
constexpr int kPromptThreads = 16 * 32;
constexpr int kPromptRows = 256;
constexpr float kGrow = 8.f, kLift = 7.f;

template <int D> constexpr int prompt_smem() { return 6 * 128 * D * 2 + 1024; }

// tcgen05 products and commit, to be executed by one elected lane. A product's descriptors are offsets from their operand's,
// added next to the instruction: kept ahead, a loop's worth of them does not fit the warp's registers.
template <int A, int B>
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tadd.s64 x, %1, %5;\n\tadd.s64 y, %2, %6;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate),
      "n"(A), "n"(B) : "memory");
}
template <int A, int B>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b32 x;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tadd.s32 x, %1, %5;\n\tadd.s64 y, %2, %6;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate),
      "n"(A), "n"(B) : "memory");
}
// steps of 16 of the contraction: operands K-major, in halves of 64 elements, HALF (16-byte units) apart
template <int HALF, int... K>
__device__ __forceinline__ void mma_ss_all(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, std::integer_sequence<int, K...>) {
  (mma_ss<(K >> 2) * HALF + (K & 3) * 2, (K >> 2) * HALF + (K & 3) * 2>(d, a, b, idesc, K > 0), ...);
}
template <int... K>
__device__ __forceinline__ void mma_ts_all(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate, std::integer_sequence<int, K...>) {
  (mma_ts<K * 8, K * 2>(d, a, b, idesc, accumulate || K > 0), ...);
}
// One lane of the warp, in the form from which the compiler knows that it is one: products then take their operands through
// the uniform registers without a detour (137 instead of 240 cycles per product beside three busy warps).
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}

template <typename T, int D>
__global__ void __launch_bounds__(kPromptThreads, 1)
attention_prompt_kernel(const AttendParams p, const uint32_t idesc_qk, const uint32_t idesc_pv) {
  constexpr int CH = D / 64, TILE = 128 * D * 2, BLOCK = kBlock * D, PIECES = BLOCK / 16 / 128;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[26];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_word;
  __shared__ float red[32];
  volatile int* abort_flag = &abort_word;
  const uint32_t base = (tc::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_s = base, k_s = base + 2 * TILE, v_s = base + 4 * TILE;
  const uint32_t bar0 = tc::smem_u32(bars);
  auto q_full = [&](int i) { return bar0 + 8u * i; };
  auto full = [&](int which, int s) { return bar0 + 8u * (2 + 2 * which + s); };      // which: keys, values
  auto empty = [&](int which, int s) { return bar0 + 8u * (6 + 2 * which + s); };
  auto s_full = [&](int i) { return bar0 + 8u * (10 + i); };
  auto p_full = [&](int i, int h) { return bar0 + 8u * (12 + 2 * i + h); };           // weights of block h of the pair
  auto done = [&](int i) { return bar0 + 8u * (16 + i); };
  auto turn = [&](int i, int q) { return bar0 + 8u * (18 + 4 * i + q); };            // the exponentials' of tile i, row quarter q
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  // the tiles with the most keys first
  const uint32_t bhs = (uint32_t)(p.c.batch * p.c.heads) * p.splits;
  const uint32_t from_last = blockIdx.x / bhs, rest = blockIdx.x - from_last * bhs;
  const int tile = p.tiles - 1 - (int)from_last, bh32 = rest / p.splits, split = rest - bh32 * p.splits;
  const int64_t bh = bh32, b = bh32 / (int)p.c.heads, kvh = bh32 - b * p.c.heads;
  Span sp = span_of(b, p.S, p.c.capacity, p.start, p.starts, p.counts);
  if (!sp.ok) {
    if (threadIdx.x == 0) flag_status(p.status, Q3_STATUS_CACHE_RANGE);
    sp.start = sp.count = 0;
  }
  const int start = (int)sp.start, end = (int)(sp.start + sp.count);           // a cache has at most 2^30 tokens
  const int complete = end / kBlock;
  if (blockIdx.x < bhs && split == 0 && threadIdx.x == 0 && sp.count > 0 && !held_whole(p.c.marks + bh * 4, end))
    flag_status(p.status, Q3_STATUS_CACHE_RECENT);
  const int row0 = tile * kPromptRows;
  const int real = (int)sp.count * p.group - row0;                 // rows of this CTA that are not padding
  const int here = real < kPromptRows ? real : kPromptRows;
  const int seen = here > 0 ? start + (row0 + here - 1) / p.group + 1 : 0;
  const int total = (seen + 127) / 128, per = (total + p.splits - 1) / p.splits;
  const int t0 = split * per, t1 = t0 + per < total ? t0 + per : total, n = t1 > t0 ? t1 - t0 : 0;
  const bool two = here > 128;
  const int wanted = (seen + kBlock - 1) / kBlock;                 // blocks
  const int whole = complete < wanted ? complete : wanted;         // of them, in 8 bits
  Mark mark[2];
  mark[0].block = -1;
  if (wanted > complete) {
    mark[0] = p.c.marks[(bh * 2 + 0) * 2 + (complete & 1)];
    mark[1] = p.c.marks[(bh * 2 + 1) * 2 + (complete & 1)];
    const int need = end - complete * kBlock;
    if (mark[0].block != complete || mark[0].fill < need || mark[1].block != complete || mark[1].fill < need) {
      if (threadIdx.x == 0) flag_status(p.status, Q3_STATUS_CACHE_RECENT);
      mark[0].block = -1;
    } else {
      narrow_marks<T, D>(mark, p.c, bh, complete, need, red);
    }
  }
  const bool tail = mark[0].block >= 0;

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(done(i), 1); for (int q = 0; q < 4; ++q) tc::mbar_init(turn(i, q), 1); tc::mbar_init(q_full(i), 4); tc::mbar_init(s_full(i), 1); tc::mbar_init(p_full(i, 0), 4); tc::mbar_init(p_full(i, 1), 4);
      for (int w = 0; w < 2; ++w) { tc::mbar_init(full(w, i), 4); tc::mbar_init(empty(w, i), two ? 2 : 1); }
    }
    tc::fence_barrier_init();
  }
  if (warp == 12) { tc::tmem_alloc(tc::smem_u32(&tmem_slot), 512); tc::tmem_relinquish(); }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;      // columns: scores / weights 0..127, 128..255; sums 256..383, 384..511

  if (warp < 4) {
    // ---------------------------------------------------------------- widen
    asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
    const int tid = threadIdx.x, g = (tid >> 2) & 7, t = tid & 3, upper = tid >> 5;
    const float lift[2] = {tail ? up_scale(mark[0].amax) : 1.f, tail ? up_scale(mark[1].amax) : 1.f};
    auto put = [&](uint32_t row_at, uint32_t x, const uint32_t (&w)[8]) {
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row_at + (((2 * t) ^ x) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(row_at + (((2 * t + 1) ^ x) << 4)), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
    };
    // The thread's piece u (128 u + tid) of a block: keys - (token / 8, dim / 64), token % 8, 16 dims: its row is the place of the
    // token, its 128-byte half dim / 64; values - dim / 8, dim % 8, 16 tokens: its row is the dim, its half the block. Two
    // 16-byte chunks each, XORed with the row's low bits.
    auto place = [&](int which, int h, int u, uint32_t& row_at, uint32_t& x) {
      const int up = u * 4 + upper;
      const int row = which ? up * 8 + g : h * 64 + ((g >> 1) & 3) * 16 + (up / CH) * 2 + (g & 1);
      x = row & 7;
      row_at = row * 128 + (which ? h * (D * 128) : (up % CH) * 16384);
    };
    uint4 kr[2][PIECES], vr[2][PIECES];
    auto fetch = [&](int which, uint4 (&r)[2][PIECES], int j) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int blk = 2 * (t0 + j) + h;
        if (j < n && blk < whole) {
          const uint4* src = reinterpret_cast<const uint4*>(p.c.payload[which] + (bh * p.c.blocks + blk) * BLOCK) + tid;
#pragma unroll
          for (int u = 0; u < PIECES; ++u) r[h][u] = __ldg(src + u * 128);
        }
      }
    };
    auto widen = [&](int which, const uint4 (&r)[2][PIECES], int j) -> bool {
      const int s = j & 1;
      const uint32_t buf = (which ? v_s : k_s) + s * TILE;
      if (!__all_sync(0xffffffffu, tc::mbar_wait(empty(which, s), ((j >> 1) & 1u) ^ 1u, abort_flag))) return false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int blk = 2 * (t0 + j) + h;
        if (blk < whole) {
#pragma unroll
          for (int u = 0; u < PIECES; ++u) {
            uint32_t w[8], row_at, x;
            widen4(r[h][u].x, w[0], w[1]); widen4(r[h][u].y, w[2], w[3]);
            widen4(r[h][u].z, w[4], w[5]); widen4(r[h][u].w, w[6], w[7]);
            place(which, h, u, row_at, x);
            put(buf + row_at, x, w);
          }
        } else {                                                   // recent tokens, or nothing
          const bool raw = tail && blk == complete;
          const T* ring = (const T*)p.c.recent[which] + (bh * 2 + (complete & 1)) * BLOCK;
#pragma unroll 1
          for (int u = 0; u < PIECES; ++u) {
            uint32_t w[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u}, row_at, x;
            if (raw) {
              const float up = lift[which];
              const uint4 a = *reinterpret_cast<const uint4*>(ring + (u * 128 + tid) * 16), e = *reinterpret_cast<const uint4*>(ring + (u * 128 + tid) * 16 + 8);
              w[0] = recent_pair<T>(a.x, up); w[1] = recent_pair<T>(a.y, up); w[2] = recent_pair<T>(a.z, up); w[3] = recent_pair<T>(a.w, up);
              w[4] = recent_pair<T>(e.x, up); w[5] = recent_pair<T>(e.y, up); w[6] = recent_pair<T>(e.z, up); w[7] = recent_pair<T>(e.w, up);
            }
            place(which, h, u, row_at, x);
            put(buf + row_at, x, w);
          }
        }
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(full(which, s));
      return true;
    };
    fetch(0, kr, 0);
    fetch(1, vr, 0);
    for (int j = 0; j < n; ++j) {
      if (!widen(0, kr, j)) break;
      fetch(0, kr, j + 1);
      if (!widen(1, vr, j)) break;
      fetch(1, vr, j + 1);
    }
  } else if (warp >= 12) {
    // ---------------------------------------------------------------- products
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int i = warp - 12;                                       // the tile: its products stay in order, the other's do not wait
    if (i < (two ? 2 : 1) && n > 0) {
      const uint32_t s_tmem = tmem + i * 128, o_tmem = tmem + 256 + i * 128;
      const uint64_t qd = tc::make_smem_desc(q_s + i * TILE, 0, 1024), kd = tc::make_smem_desc(k_s, 0, 1024), vd = tc::make_smem_desc(v_s, 0, 1024);
      bool ok = tc::mbar_wait(q_full(i), 0, abort_flag) && tc::mbar_wait(full(0, 0), 0, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      tc::tc_fence_after();
      if (ok && elect_one()) {
        mma_ss_all<(16384 >> 4)>(s_tmem, qd, kd, idesc_qk, std::make_integer_sequence<int, D / 16>());
        tc::mma_commit(s_full(i));
      }
      __syncwarp();
      // One commit per step: it also tells that the products before it are done - the previous sums, and with them the
      // buffers of keys and values that the softmax warps hand back (a commit costs as much as one product).
      for (int j = 0; j < n && ok; ++j) {
        const int s = j & 1, s1 = s ^ 1;
        ok = tc::mbar_wait(full(1, s), (j >> 1) & 1u, abort_flag) && (j + 1 == n || tc::mbar_wait(full(0, s1), ((j + 1) >> 1) & 1u, abort_flag)) &&
             tc::mbar_wait(p_full(i, 0), j & 1u, abort_flag);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc::tc_fence_after();
        if (elect_one()) mma_ts_all(o_tmem, s_tmem, vd + s * (TILE >> 4), idesc_pv, j > 0, std::make_integer_sequence<int, 4>());
        __syncwarp();
        ok = __all_sync(0xffffffffu, tc::mbar_wait(p_full(i, 1), j & 1u, abort_flag));
        if (!ok) break;
        tc::tc_fence_after();
        if (elect_one()) {
          mma_ts_all(o_tmem, s_tmem + 32, vd + s * (TILE >> 4) + (D * 128 >> 4), idesc_pv, true, std::make_integer_sequence<int, 4>());
          if (j + 1 < n) {
            mma_ss_all<(16384 >> 4)>(s_tmem, qd, kd + s1 * (TILE >> 4), idesc_qk, std::make_integer_sequence<int, D / 16>());
            tc::mma_commit(s_full(i));
          }
        }
        __syncwarp();
      }
      if (elect_one()) tc::mma_commit(done(i));
      __syncwarp();
      tc::mbar_wait_drain(done(i), 0);
    }
  } else {
    // ---------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int i = (warp - 4) >> 2, quarter = warp & 3;
    const int rt = quarter * 32 + lane, r = i * 128 + rt, row = row0 + r;   // row of the tile, of the CTA, of the kv head
    const bool mine = r < here;
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_addr = lanes + i * 128, o_addr = lanes + 256 + i * 128;
    const bool active = n > 0 && (i == 0 || two);
    bool ok = active;
    float rowf = 0.f, ref = -CUDART_INF_F, ml = -CUDART_INF_F, l = 0.f;
    int visible = 0;
    const int s_tok = row / p.group;
    if (active) {
      // the row's query into the swizzled tile, taken to fp16
      if (mine) visible = start + s_tok + 1;
      const T* src = (const T*)p.q + ((b * p.S + s_tok) * p.Hq + kvh * p.group + row % p.group) * D;
      uint4 qv[D / 8];
      float amax = 0.f;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        qv[c] = mine ? *reinterpret_cast<const uint4*>(src + c * 8) : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t w[4] = {qv[c].x, qv[c].y, qv[c].z, qv[c].w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          amax = fmaxf(amax, fmaxf(__uint_as_float(w[e] << 16 & 0x7fffffffu), __uint_as_float(w[e] & 0x7fff0000u)));
      }
      const float up = query_scale<T>(amax);
      rowf = p.scale_log2 / up;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        const uint32_t at = q_s + i * TILE + (c >> 3) * 16384 + rt * 128 + (((c & 7) ^ (rt & 7)) << 4);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(to_half_pair<T>(qv[c].x, up)), "r"(to_half_pair<T>(qv[c].y, up)),
                     "r"(to_half_pair<T>(qv[c].z, up)), "r"(to_half_pair<T>(qv[c].w, up)) : "memory");
      }
      tc::fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(q_full(i));
    }
    const float* kscale = p.c.scales[0] + bh * p.c.blocks;
    const float* vscale = p.c.scales[1] + bh * p.c.blocks;
    auto scales = [&](int j, float (&ks)[2], float (&vs)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int blk = 2 * j + h;
        ks[h] = vs[h] = 1.f;
        if (blk < whole) { ks[h] = __ldg(kscale + blk); vs[h] = __ldg(vscale + blk); }
        else if (tail && blk == complete) {
          ks[h] = mark[0].bad ? CUDART_NAN_F : 1.f / up_scale(mark[0].amax);
          vs[h] = mark[1].bad ? CUDART_NAN_F : 1.f / up_scale(mark[1].amax);
        }
      }
    };
    // without the recent tokens there is nothing from the incomplete block on
    if (!tail && visible > complete * kBlock) visible = complete * kBlock;
    float ks[2], vs[2], top_lvs = -CUDART_INF_F;
    if (active) scales(t0, ks, vs);
    for (int j = 0; j < n && ok; ++j) {
      const int ahead = visible - (t0 + j) * 128;
      const int limit = ahead < 0 ? 0 : (ahead < 128 ? ahead : 128);         // tokens of the tile that the row sees
      float f[2], lvs[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        lvs[h] = log2f(vs[h]);
        f[h] = ks[h] * rowf;
        if (f[h] < 1e-37f || limit <= h * 64) f[h] = 1e-37f;       // -inf times it stays -inf; NaN stays where the row sees it
      }
      top_lvs = fmaxf(top_lvs, fmaxf(lvs[0], lvs[1]));
      const bool far = fminf(lvs[0], lvs[1]) < top_lvs - kFar;     // only then can weights flush that count
      if (j + 1 < n) scales(t0 + j + 1, ks, vs);
      ok = __all_sync(0xffffffffu, tc::mbar_wait(s_full(i), j & 1u, abort_flag));
      if (!ok) break;
      tc::tc_fence_after();
      if (quarter == 0 && lane == 0) {                             // keys of this step and values of the last one have been used
        tc::mbar_arrive(empty(0, j & 1));
        if (j > 0) tc::mbar_arrive(empty(1, (j - 1) & 1));
      }
      if (__any_sync(0xffffffffu, limit < 128)) {                  // a tile that some row does not see to its end: -inf there
#pragma unroll 1
        for (int c0 = 0; c0 < 128; c0 += 32) {
          uint32_t e[32];
          tc::tmem_ld32(s_addr + c0, e);
          tc::tmem_ld_wait();
          const int left = limit - (c0 & 64) - ((c0 & 32) >> 3);
#pragma unroll
          for (int c = 0; c < 32; ++c)                             // the token of column c0 + c, less that of column c0
            if (((c >> 1) & 7) * 8 + (c >> 4) * 2 + (c & 1) >= left) e[c] = 0xff800000u;
          tc::tmem_st32(s_addr + c0, e);
        }
        tc::tmem_st_wait();
      }
      // The scores of one block at a time are in registers: the second block's are read for the maximum first, and once more
      // after the first block's weights (all 128 of them would not leave the other warps enough registers).
      uint32_t a[2][32];
      float top_of[2];
#pragma unroll
      for (int h = 1; h >= 0; --h) {
#pragma unroll
        for (int q = 0; q < 2; ++q) tc::tmem_ld32(s_addr + h * 64 + q * 32, a[q]);
        tc::tmem_ld_wait();
        float top[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int c = 0; c < 32; c += 2)
            top[(c >> 1) & 3] = max3(top[(c >> 1) & 3], __uint_as_float(a[q][c]), __uint_as_float(a[q][c + 1]));
        top_of[h] = fmaf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), f[h], lvs[h]);
      }
      const float mx = fmaxf(fmaxf(top_of[0], top_of[1]), -CUDART_INF_F);        // NaN counts as nothing here
      const bool move = mx > ref + kGrow || (ref == -CUDART_INF_F && mx > ref);
      if (__any_sync(0xffffffffu, move)) {                         // the reference moves, the sums so far follow
        const float alpha = move ? exp2_fast(ref - mx) : 1.f;
        if (move) ref = mx;
        if (j > 0) {                                               // they are complete: the commit of these scores came after
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tc::tmem_ld32(o_addr + c, o);
            tc::tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tc::tmem_st32(o_addr + c, o);
          }
        }
      }
      if (far) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (top_of[h] > -CUDART_INF_F) lvs[h] += fmaxf(ref - kFar - top_of[h], 0.f);
      }
      const float at = ref > -CUDART_INF_F ? ref : 0.f;
      float sum[2];
      // The exponentials of the two tiles take turns: at the same time they would only wait for one another and leave the
      // tensor cores idle afterwards.
      if (two) {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(turn(i, quarter), (uint32_t)(j + 1 - i) & 1u, abort_flag));
        if (!ok) break;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float shift = limit <= h * 64 ? 0.f : lvs[h] - at + kLift;
        const uint64_t f2 = pack_f32x2(f[h], f[h]), shift2 = pack_f32x2(shift, shift);
        uint64_t sum2[2] = {0ull, 0ull};
        uint32_t w[32];
        if (h == 1) {
#pragma unroll
          for (int q = 0; q < 2; ++q) tc::tmem_ld32(s_addr + 64 + q * 32, a[q]);
          tc::tmem_ld_wait();
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const uint64_t z = fma_f32x2(pack_f32x2(__uint_as_float(a[q][c]), __uint_as_float(a[q][c + 1])), f2, shift2);
            float x, y;
            unpack_f32x2(z, x, y);
            x = exp2_fast(x);
            y = exp2_fast(y);
            sum2[(c >> 1) & 1] = add_f32x2(sum2[(c >> 1) & 1], pack_f32x2(x, y));
            w[q * 16 + (c >> 1)] = pack_half(x, y);
          }
        if (h == 1 && two && lane == 0) tc::mbar_arrive(turn(i ^ 1, quarter));
        tc::tmem_st32(s_addr + h * 32, w);
        float x, y;
        unpack_f32x2(add_f32x2(sum2[0], sum2[1]), x, y);
        sum[h] = x + y;
        tc::tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(p_full(i, h));
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (limit > h * 64) {
          const float d = at - lvs[h], nml = fmaxf(ml, d);
          l = l * exp2_fast(ml - nml) + sum[h] * exp2_fast(d - nml);
          ml = nml;
        }
    }
    if (active && ok) {
      ok = __all_sync(0xffffffffu, tc::mbar_wait(done(i), 0, abort_flag));
      tc::tc_fence_after();
    }
    const bool any = active && ok && mine && l != 0.f;
    const float whole = ml + log2f(l), half = any ? exp2_fast(0.5f * (ref - whole)) : 0.f;
    const int64_t orow = (b * p.S + s_tok) * p.Hq + kvh * p.group + row % p.group;
#pragma unroll 1
    for (int c = 0; c < D; c += 32) {
      uint32_t o[32];
      if (active && ok) {
        tc::tmem_ld32(o_addr + c, o);
        tc::tmem_ld_wait();
      }
      if (row < p.rows) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float v[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) v[x] = any ? __uint_as_float(o[e + x]) * half * half : 0.f;
          if (p.splits == 1) VecIO<T, 8>::store((T*)p.out + orow * D + c + e, v);
          else VecIO<float, 8>::store(p.part + (orow * p.splits + split) * D + c + e, v);
        }
      }
    }
    if (p.splits > 1 && row < p.rows) p.lse[orow * p.splits + split] = any ? whole : -CUDART_INF_F;
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == 12) { tc::tc_fence_after(); tc::tmem_dealloc(tmem, 512); }
  if (threadIdx.x == 0 && *abort_flag) flag_status(p.status, Q3_STATUS_WAIT_TIMEOUT);
}

// out[row] = sum_i part[row, i] 2^{lse_i} / sum_i 2^{lse_i}; one warp per row, the splits' weights - divided by their sum
// first: a sum of large rows may not be finite - shared out over the lanes, 32 at a time, then every lane adds up its D / 32
// columns in the order of the splits.
template <typename T, int D>
__global__ void __launch_bounds__(128)
attention_merge_kernel(const float* __restrict__ part, const float* __restrict__ lse, T* __restrict__ out, int64_t rows, int splits) {
  constexpr int CPL = D / 32;
  cudaGridDependencySynchronize();
  const int64_t row = blockIdx.x * 4ll + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= rows) return;
  const float* ls = lse + row * splits;
  float mx = -CUDART_INF_F;
  for (int i = lane; i < splits; i += 32) mx = fmaxf(mx, ls[i]);
  mx = warp_max(mx);
  const float ref = mx > -CUDART_INF_F ? mx : 0.f;
  float tot = 0.f, acc[CPL];
  for (int i = lane; i < splits; i += 32) tot += exp2_fast(ls[i] - ref);
  tot = warp_sum(tot);
#pragma unroll
  for (int c = 0; c < CPL; ++c) acc[c] = 0.f;
  const float* src = part + row * splits * D + lane * CPL;
  for (int base = 0; base < splits; base += 32) {
    const float mine = base + lane < splits && tot != 0.f ? exp2_fast(ls[base + lane] - ref) / tot : 0.f;
    const int n = splits - base < 32 ? splits - base : 32;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const float w = __shfl_sync(0xffffffffu, mine, i);
      if constexpr (CPL == 4) {
        const float4 v = *reinterpret_cast<const float4*>(src + (int64_t)(base + i) * D);
        acc[0] = fmaf(v.x, w, acc[0]); acc[1] = fmaf(v.y, w, acc[1]); acc[2] = fmaf(v.z, w, acc[2]); acc[3] = fmaf(v.w, w, acc[3]);
      } else {
        const float2 v = *reinterpret_cast<const float2*>(src + (int64_t)(base + i) * D);
        acc[0] = fmaf(v.x, w, acc[0]); acc[1] = fmaf(v.y, w, acc[1]);
      }
    }
  }
  T* o = out + row * D + lane * CPL;
#pragma unroll
  for (int c = 0; c < CPL; ++c) o[c] = from_f32<T>(acc[c]);
}

// How a call is cut. Up to 16 rows: rows in one tile of 8 or 16, the units in `splits` pieces, for CTAs of eight warps (one per
// SM) where there are no more (sequence, head) pairs than SMs, else of four (two per SM). More rows: tiles of 256 rows, key tiles
// of 128 tokens in `splits` pieces, also where the rows are few and the cache is long (8 sequences of 32005 tokens, the last 5 of
// them new, 32 / 8 heads: 20 rows, 325 us; the cache could be read in 81; 4 new ones, 16 rows: 102 us). `longest` is the capacity
// where the lengths are on the device: 64 sequences of 1001 tokens take 33 us in a cache of 8192 tokens, 75 us in one of 32768.
// The number of pieces is the one with the shortest time in a model of it: waves of CTAs times what a CTA takes - a fixed part and
// its share of the steps - and a second launch where there are pieces to merge - up to 8 pieces of few rows are a cluster of CTAs,
// which merges them over its shared memory; all in units of one step (a block per warp, or a key tile), as measured: few rows 2.5
// + blocks per warp, and 1.5 for the merge, 0.5 within a cluster; many rows 8 + key tiles, and 2.
// Eight warps against two CTAs of four, us: 4 x 131001 tokens 160 / 174, one sequence of 32001 17.6 / 20.3, of 301 7.0 / 8.3; but
// 64 of 8001 169 / 158 and of 1001 38 / 33: uneven waves cost more when a CTA has the SM.
struct Plan {
  bool prompt;
  bool joined;
  int nt, warps, tiles, splits;
};
inline Plan plan_attention(int64_t batch_heads, int64_t rows, int64_t longest) {
  Plan pl;
  pl.prompt = rows > 16;
  pl.nt = rows <= 8 ? 1 : 2;
  pl.tiles = pl.prompt ? (int)cdiv(rows, kPromptRows) : 1;
  const int64_t base = batch_heads * pl.tiles, sms = sm_count();
  pl.warps = base <= sms ? 8 : 4;
  const int64_t steps = pl.prompt ? cdiv(longest, 128) : cdiv(cdiv(longest, kBlock), pl.warps);
  const int64_t slots = pl.prompt || pl.warps == 8 ? sms : 2 * sms;
  const float fixed = pl.prompt ? 8.f : 2.5f, merge = pl.prompt ? 2.f : 1.5f;
  float best = 0.f;
  auto consider = [&](int64_t s) {
    if (s < 1 || s > steps) return;
    s = cdiv(steps, cdiv(steps, s));                               // no more pieces than the longest of them needs
    const bool joined = !pl.prompt && s > 1 && s <= 8;
    const float cost = (float)cdiv(base * s, slots) * (fixed + (float)cdiv(steps, s)) + (joined ? 0.5f : s > 1 ? merge : 0.f);
    if (best == 0.f || cost < best) { best = cost; pl.splits = (int)s; pl.joined = joined; }
  };
  pl.splits = 1;
  pl.joined = false;
  for (int64_t s = 1; s <= 8; ++s) consider(s);
  for (int64_t waves = 1; waves <= 4; ++waves) consider(waves * slots / base);     // full waves
  return pl;
}

template <typename T, int D, int NT, int WARPS>
int launch_split(const AttendParams& p, int64_t batch_heads, cudaStream_t st) {
  auto kern = attention_split_kernel<T, D, NT, WARPS>;
  static DeviceFlags configured = {};
  const int smem = WARPS * ring_bytes(WARPS);
  if (int rc = ensure_dynamic_smem(kern, smem, &configured); rc != Q3_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(batch_heads * p.splits));
  cfg.blockDim = dim3(WARPS * 32);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.joined ? p.splits : 1;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.joined ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) { cudaGetLastError(); return Q3_ERR_CUDA - (int)e; }
  return launch_status();
}

template <typename T, int D>
int launch_prompt(const AttendParams& p, int64_t batch_heads, cudaStream_t st) {
  auto kern = attention_prompt_kernel<T, D>;
  static DeviceFlags configured = {};
  if (int rc = ensure_dynamic_smem(kern, prompt_smem<D>(), &configured); rc != Q3_OK) return rc;
  kern<<<(unsigned)(batch_heads * p.tiles * p.splits), kPromptThreads, prompt_smem<D>(), st>>>(
      p, tc::make_idesc_f16(128, 128, false, false, false), tc::make_idesc_f16(128, D, false, false, false));
  return launch_status();
}

template <typename T, int D>
int launch_merge(const AttendParams& p, int64_t rows, cudaStream_t st) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)cdiv(rows, 4));
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;   // its CTAs may be placed while the last splits finish
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, attention_merge_kernel<T, D>, (const float*)p.part, (const float*)p.lse, (T*)p.out,
                                     rows, p.splits);
  if (e != cudaSuccess) { cudaGetLastError(); return Q3_ERR_CUDA - (int)e; }
  return launch_status();
}

}  // namespace qc
}  // namespace q3

using namespace q3;

// host checks shared by the call and its workspace query, and how the call is cut; `start` < 0: lengths on the device
static int plan_checked(const q3_quantized_cache* cache, int64_t S, int64_t Hq, int64_t start, qc::Plan* plan, int64_t* bytes) {
  if (int rc = qc::check_cache(cache); rc != Q3_OK) return rc;
  if (S < 1 || S > cache->capacity || Hq < 1 || Hq % cache->heads || Hq > (int64_t)1 << 16 || start > cache->capacity)
    return Q3_ERR_SHAPE;
  const int64_t bh = cache->batch * cache->heads, rows = S * (Hq / cache->heads);
  if (rows > (int64_t)1 << 30) return Q3_ERR_SHAPE;
  *plan = qc::plan_attention(bh, rows, start < 0 || start > cache->capacity - S ? cache->capacity : start + S);
  if (bh * plan->tiles > 0x7fffffff / plan->splits) return Q3_ERR_SHAPE;
  *bytes = plan->splits == 1 || plan->joined ? 0 : cache->batch * S * Hq * plan->splits * (cache->head_dim + 1) * 4;
  return Q3_OK;
}

extern "C" int64_t q3_qcache_attention_workspace_bytes(const q3_quantized_cache* cache, int64_t S, int64_t Hq, int64_t start) {
  qc::Plan plan;
  int64_t bytes = 0;
  return plan_checked(cache, S, Hq, start, &plan, &bytes) == Q3_OK ? bytes : 0;
}

extern "C" int q3_qcache_attention(const q3_quantized_cache* cache, const void* q, void* out, void* workspace,
                                   int64_t workspace_bytes, int64_t S, int64_t Hq, int64_t start, const int64_t* starts,
                                   const int64_t* counts, double scale, int* status, q3_stream_t stream) {
  if (int rc = qc::check_cache(cache); rc != Q3_OK) return rc;
  if (!q || !out || !(scale > 0)) return Q3_ERR_ARG;
  if (!starts && (start < 0 || start > cache->capacity - (counts ? 0 : S))) return Q3_ERR_SHAPE;
  qc::Plan pl;
  int64_t need = 0;
  if (int rc = plan_checked(cache, S, Hq, starts ? -1 : start, &pl, &need); rc != Q3_OK) return rc;
  if (!aligned16(q) || !aligned16(out) || !aligned16(workspace)) return Q3_ERR_ALIGN;
  if (need > 0 && (!workspace || workspace_bytes < need)) return Q3_ERR_WORKSPACE;
  const int group = (int)(Hq / cache->heads);
  const int64_t bh = cache->batch * cache->heads, rows = S * group, out_rows = cache->batch * S * Hq;
  qc::AttendParams p;
  p.c = qc::device_view(cache);
  p.q = q; p.out = out;
  p.part = (float*)workspace;
  p.lse = p.part ? p.part + out_rows * pl.splits * cache->head_dim : nullptr;
  p.S = S; p.start = start; p.starts = starts; p.counts = counts;
  p.Hq = (int)Hq; p.group = group; p.rows = (int)rows; p.tiles = pl.tiles; p.splits = pl.splits; p.joined = pl.joined;
  p.scale_log2 = (float)(scale * 1.4426950408889634);
  p.status = status;
  cudaStream_t st = (cudaStream_t)stream;
  Q3_DISPATCH_CACHE(cache, T, D, {
    int rc;
    if (pl.prompt) rc = qc::launch_prompt<T, D>(p, bh, st);
    else if (pl.warps == 8) rc = pl.nt == 1 ? qc::launch_split<T, D, 1, 8>(p, bh, st) : qc::launch_split<T, D, 2, 8>(p, bh, st);
    else rc = pl.nt == 1 ? qc::launch_split<T, D, 1, 4>(p, bh, st) : qc::launch_split<T, D, 2, 4>(p, bh, st);
    if (rc == Q3_OK && pl.splits > 1 && !pl.joined) rc = qc::launch_merge<T, D>(p, out_rows, st);
    return rc;
  });
}
