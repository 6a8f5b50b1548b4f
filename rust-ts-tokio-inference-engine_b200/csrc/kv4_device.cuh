// Device helpers shared by the kernels that read the 4-bit KV cache.
#pragma once
#include <algorithm>
#include <cfloat>
#include <climits>

#include "kernels.h"
#include "kv4.h"
#include "tcgen05.cuh"

namespace qwen {
namespace {

constexpr int kRowsPerTile = 8;  // query rows of an MMA tile

// The attention kernels lay a call's units end to end in places counted in 32
// bits. The host refuses calls that could need kPlacesMax or more; sequences that
// overlap (cu_seqlens not ascending) can still exceed what it counted, so the sums
// stop at kPlacesMax, and a call whose sum reaches it computes nothing.
constexpr int kPlacesMax = (1 << 30) - 1;
__device__ __forceinline__ int add_places(int a, int b) { return min(a + b, kPlacesMax); }
// Tiles of `rows` query rows that a call's sequences fill at most: each the longest's,
// and together no more than the rows there are, plus a part of a tile each.
inline int64_t tiles_at_most(const Kv4AttentionArgs& a, int64_t of_longest, int rows) {
  return std::min(int64_t(a.n_seq) * of_longest, int64_t(a.tokens) * (a.cache.Hq / a.cache.Hkv) / rows + a.n_seq);
}

// Bounded waits on a barrier; a wait that runs out (about a second) sets the
// status bit and, where the CTA has roles that wait for one another, `abort`,
// which ends the other roles' waits too.
__device__ __forceinline__ bool kv4_wait(uint64_t* bar, uint32_t parity, uint32_t* status, volatile int* abort = nullptr) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
    if (mbar_try_sleep(bar, parity, 2000)) return true;
    if (abort && *abort) return false;
    if (clock64() - t0 > kWaitCycles) {
      kv4_flag(status, kErrTimeout);
      if (abort) *abort = 1;
      return false;
    }
  }
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};"
      :
      : "r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]),
        "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
        "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a b from zero accumulators (no registers to clear)
__device__ __forceinline__ void mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const uint8_t* p) {
  if constexpr (N == 4) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(p);
  else if constexpr (N == 2) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
  else w[0] = *reinterpret_cast<const uint32_t*>(p);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float(uint32_t(min(max(e, -126), 127) + 127) << 23); }

// Length of sequence s, kept within the table and, when weights are written, their rows.
__device__ __forceinline__ int kv4_length(const Kv4AttentionArgs& a, int s, bool report) {
  int64_t most = a.table_stride * kPageTokens;
  if (a.weights_out) most = min(most, a.weights_stride);
  const int len = a.kv_lens[s];
  if (len < 0 || len > most) {
    if (report) kv4_flag(a.cache.status, kErrBounds);
    return int(min(max(int64_t(len), int64_t(0)), most));
  }
  return len;
}

// A sequence's query rows (token-major: row = token * G + head of the group)
// and keys; the row range is kept inside the call's tokens.
struct Seq {
  int first, count, len, tiles;  // tiles of 8 rows; none for a sequence with more rows than the call's row_limit
};
__device__ __forceinline__ Seq load_seq(const Kv4AttentionArgs& a, int s, int G, bool report) {
  Seq q;
  q.first = min(max(a.cu_seqlens[s], 0), a.tokens);
  q.count = min(max(a.cu_seqlens[s + 1], 0), a.tokens) - q.first;
  q.len = kv4_length(a, s, report);
  if (q.count < 0 || q.count > a.max_count) {
    if (report) kv4_flag(a.cache.status, kErrBounds);
    q.count = 0;
  }
  q.tiles = q.count * G > a.row_limit ? 0 : (q.count * G + kRowsPerTile - 1) / kRowsPerTile;
  return q;
}
// Keys that the last row of tile r sees, and the pages that hold them.
__device__ __forceinline__ int tile_pages(const Seq& q, int r, int G) {
  const int token = min(q.count - 1, ((r + 1) * kRowsPerTile - 1) / G);
  return max(0, q.len - q.count + token + 1 + kPageTokens - 1) / kPageTokens;
}

// Sigmoid by the approximate reciprocal: a relative error of a few 2^-23, far below a 16-bit result's rounding.
__device__ __forceinline__ float sigmoid_fast(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

// Eight dims of one output row and its gate.
__device__ __forceinline__ void load_gate(const Kv4AttentionArgs& a, int token, int head, int dim, bool vec, float (&g)[8]) {
  const float* p = static_cast<const float*>(a.gate.data) + token * a.gate.token_stride + head * a.gate.head_stride + dim;
  if (vec) {
    const float4 lo = *reinterpret_cast<const float4*>(p), hi = *reinterpret_cast<const float4*>(p + 4);
    g[0] = lo.x, g[1] = lo.y, g[2] = lo.z, g[3] = lo.w, g[4] = hi.x, g[5] = hi.y, g[6] = hi.z, g[7] = hi.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) g[i] = p[i];
  }
}
template <class T>
__device__ __forceinline__ void write_dims(const Kv4AttentionArgs& a, int token, int head, int dim, float (&y)[8],
                                           const float (&gate)[8], bool vec) {
  if (a.gate.data) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= sigmoid_fast(gate[i]);
  }
  T* out = static_cast<T*>(a.out) + token * a.out_token_stride + head * a.out_head_stride + dim;
  alignas(16) T v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = kv4_from_float<T>(y[i]);
  if (vec) {
    *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = v[i];
  }
}

}  // namespace
}  // namespace qwen
