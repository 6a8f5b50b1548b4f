// Attention over the 4-bit paged KV cache.
//
// kv4_decode_kernel: the (sequence, KV head, tile of 8 query rows) units of a
// call are laid end to end, measured in the page pairs each has to read, and cut
// into equal ranges, one per CTA; a unit that spans CTAs leaves partial results
// that kv4_merge_kernel joins. The lengths live on the device, so every CTA
// finds its range itself from a prefix sum over the sequences.
//
// The pairs of a range are dealt to the CTA's warps, which stream them through
// private shared-memory rings, one bulk copy per (page, KV head) block; a ring
// runs on across unit borders. A warp works on 2 x 16 keys x 8 query rows:
//   S^T = K Q^T. An fp16 subnormal with the bits 0000 0000 0000 nnnn is n 2^-24
//   and one with nnnn 0000 is n 2^-20, exactly, so the masks 0x000F000F and
//   0x00F000F0 turn a word of nibbles into MMA operands with no conversion; the
//   factor 2^4 between the two is taken out of Q. Scale and bias of a group of
//   64 dims enter afterwards in 32 bits: s = scale (q . n) + bias (sum of q).
//   The stored pairs (scale, bias) are themselves a bf16 operand: against
//   (0, sum of q), the sums split into three bf16 terms, two MMAs give the
//   bias part of all 16 keys.
//   Q is fp16, each row scaled by a power of two, so fp16 and bf16 queries are
//   exact (bf16 has fewer mantissa bits and the row keeps its range).
//   O^T += V^T P^T. The nibbles of two keys are interleaved into k pairs and
//   masked the same way. The step of V is folded into the weights, P_g = p
//   scale_g, rounded to fp16 (2^-11 of a weight, the operand's own precision)
//   after a power of two per group has brought the scales that the warp has seen
//   to at most 2^6; sum p bias_g is kept in 32 bits beside it.
// The running maximum moves only when a logit exceeds it by 2^8: a vote per
// page then replaces the reduction over the keys, and the weights stay below
// 2^8 x 2^6, inside fp16.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <climits>

#include "kernels.h"
#include "kv4.h"

namespace qwen {

extern std::atomic<uint64_t> g_kernel_launches;

namespace {

constexpr int kWarps = 4;
constexpr int kStages = 2;  // page pairs of a warp's ring
constexpr int kThreads = kWarps * 32;
constexpr int kCtasPerSm = 2;
constexpr int kRowsPerTile = 8;
constexpr int kMinPairs = 8;   // fewest page pairs of a CTA's range
constexpr int kUnitPairs = 3;  // what a unit costs beside its pages, in page pairs
constexpr int kGroupsMax = 512;  // entries of the prefix table that finds a page's sequence
constexpr float kLazy = 8.f;    // log2 of how far a logit may exceed the running maximum
constexpr long long kWaitCycles = 2000000000ll;

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, uint32_t* status) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  for (;;) {
    if (mbar_try(bar, parity)) return true;
    if (clock64() - t0 > kWaitCycles) {
      kv4_flag(status, kErrTimeout);
      return false;
    }
  }
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
      "l"(src), "r"(bytes), "r"(smem_u32(bar))
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
  int first, count, len, tiles;
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
  q.tiles = (q.count * G + kRowsPerTile - 1) / kRowsPerTile;
  return q;
}
// Keys that the last row of tile r sees, and the pages that hold them.
__device__ __forceinline__ int tile_pages(const Seq& q, int r, int G) {
  const int token = min(q.count - 1, ((r + 1) * kRowsPerTile - 1) / G);
  return max(0, q.len - q.count + token + 1 + kPageTokens - 1) / kPageTokens;
}
// Length of a unit: its page pairs behind kUnitPairs places that hold none, so
// that ranges of equal length take equal time whatever the units' sizes.
__device__ __forceinline__ int unit_length(const Seq& q, int r, int G) {
  const int pages = tile_pages(q, r, G);
  return pages ? (pages + 1) / 2 + kUnitPairs : 0;
}
__device__ __forceinline__ int64_t seq_length(const Seq& q, int G) {  // of one KV head
  int64_t n = 0;
  for (int r = 0; r < q.tiles; ++r) n += unit_length(q, r, G);
  return n;
}

// Workspace: page offset of every sequence's first unit, pages per CTA, then
// per CTA two partial results (the first unit of its range and the last).
struct Workspace {
  int64_t* offsets;  // [n_seq + 1]
  int64_t* range;
  float* ml;  // [ctas][2][8][2]
  float* o;   // [ctas][2][8][D]
};
__host__ __device__ inline size_t align16(size_t n) { return (n + 15) & ~size_t(15); }
__host__ __device__ inline Workspace carve(void* base, int n_seq, int ctas) {
  Workspace w;
  uint8_t* p = static_cast<uint8_t*>(base);
  w.offsets = reinterpret_cast<int64_t*>(p);
  w.range = w.offsets + n_seq + 1;
  p += align16(size_t(n_seq + 2) * 8);
  w.ml = reinterpret_cast<float*>(p);
  p += size_t(ctas) * 2 * kRowsPerTile * 2 * 4;
  w.o = reinterpret_cast<float*>(p);
  return w;
}

// Writes 8 dims of one output row, gated.
__device__ __forceinline__ void load_gate(const Kv4AttentionArgs& a, int token, int head, int dim, float (&g)[8]) {
  const float* p = static_cast<const float*>(a.gate.data) + token * a.gate.token_stride + head * a.gate.head_stride + dim;
#pragma unroll
  for (int i = 0; i < 8; ++i) g[i] = p[i];
}
template <class T>
__device__ __forceinline__ void write_dims(const Kv4AttentionArgs& a, int token, int head, int dim, float (&y)[8],
                                           const float (&gate)[8], bool vec) {
  if (a.gate.data) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= sigmoidf_(gate[i]);
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

template <int D>
struct Smem {
  alignas(128) uint8_t ring[kWarps][kStages][2][Kv4Layout<D>::kBlock];
  alignas(16) float o[2][kRowsPerTile][D];
  alignas(16) uint32_t q[Kv4Layout<D>::kLaneWords][32][4];  // B fragments of the tile's rows
  uint32_t q_sum[3][kRowsPerTile][4];  // sums over the groups as bf16 terms, above a zero
  float q_back[kRowsPerTile];
  int q_seen[kRowsPerTile];
  float ml[kWarps][kRowsPerTile][2];
  int64_t scan[kWarps];
  int64_t offsets[kGroupsMax + 1];  // first place of each group of sequences
  alignas(16) uint64_t blocks[kWarps][64][2];  // blocks of a warp's next places, two windows of 32; 0: none
  int start;                        // the group that holds the range's first place
  uint64_t full[kWarps][kStages];
};

// The query rows of a tile as B fragments (lane = 4 row + t, register j of word
// i: dims 2 j, 2 j + 1 of the word's eight), 16 threads per row. A row is
// scaled by a power of two so that its largest value lies in [2^13, 2^14):
// fp16 and bf16 queries stay exact; the pairs that meet nibbles carrying 2^4
// are lowered by as much. Beside them: the factor that brings (q . n) 2^-24
// back to a logit in base 2, the row's sums over the groups in base 2, and how
// many keys it sees. A row with a value that is not finite gets NaN sums, so
// its logits are all NaN.
template <int D, class T>
__device__ __forceinline__ void load_tile(const Kv4AttentionArgs& a, const Seq& seq, int head0, int r, int G, bool vec,
                                          int tid, uint32_t (*frag)[32][4], uint32_t (*sums)[kRowsPerTile][4], float* back, int* seen) {
  constexpr int kPer = D / 128 > 0 ? D / 128 : 1;  // words of a thread
  const int rr = tid / 16, j = tid % 16, row = r * kRowsPerTile + rr, token = row / G;
  const bool real = token < seq.count;
  const T* src = static_cast<const T*>(a.q.data) + (seq.first + token) * a.q.token_stride + (head0 + row % G) * a.q.head_stride;
  float x[kPer][8], most = 0.f, sum[kPer];
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int w = j + 16 * k;
    alignas(16) T raw[8] = {};
    if (real && w < D / 8) {
      if (vec) {
        *reinterpret_cast<uint4*>(raw) = *reinterpret_cast<const uint4*>(src + 8 * w);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) raw[e] = src[8 * w + e];
      }
    }
    sum[k] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[k][e] = kv4_to_float(raw[e]);
      sum[k] += x[k][e];
      // the largest magnitude; a NaN's bits are above every number's
      most = __uint_as_float(max(__float_as_uint(most), __float_as_uint(x[k][e]) & 0x7FFFFFFFu));
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], o);
  }
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) most = __uint_as_float(max(__float_as_uint(most), __shfl_xor_sync(0xffffffffu, __float_as_uint(most), o)));
  const bool fine = __float_as_uint(most) < 0x7F800000u;
  const int e = most > 0.f && fine ? int(__float_as_uint(most) >> 23) - 126 : 0;  // |row| < 2^e
  const float up = pow2i((14 - e) / 2), up2 = fine ? pow2i(14 - e - (14 - e) / 2) : 0.f;
  const float factor = a.scale * 1.4426950408889634f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int w = j + 16 * k;
    if (w < D / 8) {
      uint32_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float lift = (i & 1 ? 0.0625f : 1.f) * up2;
        v[i] = fine ? pack_f16(x[k][2 * i] * up * lift, x[k][2 * i + 1] * up * lift) : 0u;
      }
      *reinterpret_cast<uint4*>(frag[2 * (w / 8) + w % 8 / 4][4 * rr + w % 4]) = make_uint4(v[0], v[1], v[2], v[3]);
      if (w % 8 == 0) {
        const float total = fine ? sum[k] * factor : NAN;
        float rest = total;
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const uint32_t top = uint32_t(float_to_bf16_bits(rest)) << 16;
          sums[i][rr][w / 8] = top;
          rest -= __uint_as_float(top);
        }
      }
    }
  }
  if (j >= D / 64 && j < 4) {  // groups this head_dim does not have
#pragma unroll
    for (int i = 0; i < 3; ++i) sums[i][rr][j] = 0u;
  }
  if (j == 0) {
    back[rr] = factor * pow2i((e + 10) / 2) * pow2i(e + 10 - (e + 10) / 2);
    seen[rr] = real ? seq.len - seq.count + token + 1 : INT_MAX;  // rows past the last are not written
  }
}

// Position in the laid-out units.
struct Cursor {
  int s, g, r;
  int64_t at;  // page offset of the unit
};

template <int D, class T>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) kv4_decode_kernel(Kv4AttentionArgs a, bool q_vec, bool out_vec) {
  pdl_trigger();
  pdl_wait();
  using L = Kv4Layout<D>;
  constexpr int NG = L::kGroups, LW = L::kLaneWords;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  const int Hkv = a.cache.Hkv, G = a.cache.Hq / Hkv;
  const Workspace ws = carve(a.workspace, a.n_seq, gridDim.x);
  if (tid < kWarps * kStages) mbar_init(&sm.full[0][0] + tid, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");

  // page offsets of the sequences, in groups of `per` when there are many
  const int per = (a.n_seq + kGroupsMax - 1) / kGroupsMax, groups = (a.n_seq + per - 1) / per;
  int64_t total = 0;
  for (int g0 = 0; g0 < groups; g0 += kThreads) {
    const int gi = g0 + tid;
    int64_t n = 0;
    for (int s = gi * per; s < min(a.n_seq, (gi + 1) * per); ++s)
      n += seq_length(load_seq(a, s, G, blockIdx.x == 0), G) * Hkv;
    int64_t x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) sm.scan[warp] = x;
    __syncthreads();
    int64_t before = total;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sm.scan[w];
      total += sm.scan[w];
    }
    if (gi < groups) sm.offsets[gi] = before + x - n;
    __syncthreads();
  }
  if (tid == 0) sm.offsets[groups] = total;
  __syncthreads();
  const int64_t range = max(int64_t(kMinPairs), (total + gridDim.x - 1) / gridDim.x);
  const int64_t begin = blockIdx.x * range, end = min(total, begin + range);
  if (blockIdx.x == 0) {  // for the merge
    for (int gi = tid; gi < groups; gi += kThreads) {
      int64_t off = sm.offsets[gi];
      for (int s = gi * per; s < min(a.n_seq, (gi + 1) * per); ++s) {
        ws.offsets[s] = off;
        off += seq_length(load_seq(a, s, G, false), G) * Hkv;
      }
    }
    if (tid == 0) {
      ws.offsets[a.n_seq] = total;
      *ws.range = range;
    }
  }
  if (begin >= end) return;

  // the unit that holds place p, in or behind group gi
  auto locate = [&](int64_t p, int gi, Cursor& c, Seq& q) {
    c.s = gi * per;
    c.at = sm.offsets[gi];
    int64_t one;
    for (;;) {
      q = load_seq(a, c.s, G, false);
      one = seq_length(q, G);
      if (c.at + one * Hkv > p) break;
      c.at += one * Hkv;
      ++c.s;
    }
    c.g = 0;
    while (c.at + one <= p) {
      c.at += one;
      ++c.g;
    }
    c.r = 0;
    while (c.at + unit_length(q, c.r, G) <= p) c.at += unit_length(q, c.r++, G);
  };
  auto advance = [&](Cursor& c, Seq& q, int& length) {  // to the next unit that has pages
    do {
      c.at += length;
      if (++c.r >= q.tiles) {
        c.r = 0;
        if (++c.g >= Hkv) {
          c.g = 0;
          do q = load_seq(a, ++c.s, G, false);
          while (q.tiles == 0);
        }
      }
      length = unit_length(q, c.r, G);
    } while (length == 0);
  };
  for (int gi = tid; gi < groups; gi += kThreads)
    if (sm.offsets[gi] <= begin && begin < sm.offsets[gi + 1]) sm.start = gi;
  __syncthreads();
  Cursor u;
  Seq seq;
  locate(begin, sm.start, u, seq);
  int length = unit_length(seq, u.r, G);

  // the warp's places are begin + warp + kWarps i; window w holds i = 32 w .. 32 w + 31
  const int n_mine = int((end - begin - warp + kWarps - 1) / kWarps);
  auto look_up = [&](int i) {
    if (i >= n_mine) return;
    const int64_t p = begin + warp + int64_t(kWarps) * i;
    Cursor c = u;
    Seq q = seq;
    if (p >= u.at + length) {
      int lo = sm.start, hi = groups;  // the last group that starts at or before p
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (sm.offsets[mid] <= p) lo = mid;
        else hi = mid;
      }
      locate(p, lo, c, q);
    }
    const int64_t at = (p - c.at - kUnitPairs) * 2;
    const int pages = tile_pages(q, c.r, G);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint64_t block = 0;
      if (at >= 0 && at + h < pages) {
        const int64_t page = a.table[c.s * a.table_stride + at + h];
        if (page >= 0 && uint64_t(page) < a.cache.pages) block = reinterpret_cast<uint64_t>(a.cache.block(uint64_t(page), c.g));
        else kv4_flag(a.cache.status, kErrBounds);
      }
      sm.blocks[warp][i & 63][h] = block;
    }
  };
  auto issue = [&](int i, int stage) {  // lane 0
    if (i >= n_mine) return;
    const ulonglong2 from = *reinterpret_cast<const ulonglong2*>(sm.blocks[warp][i & 63]);
    uint64_t* bar = &sm.full[warp][stage];
    if (!(from.x | from.y)) {
      mbar_arrive(bar);
      return;
    }
    mbar_expect_tx(bar, (from.x ? L::kBlock : 0) + (from.y ? L::kBlock : 0));
    if (from.x) bulk_load(sm.ring[warp][stage][0], reinterpret_cast<const void*>(from.x), L::kBlock, bar);
    if (from.y) bulk_load(sm.ring[warp][stage][1], reinterpret_cast<const void*>(from.y), L::kBlock, bar);
  };
  look_up(lane);
  __syncwarp();
  if (lane == 0)
    for (int i = 0; i < kStages; ++i) issue(i, i);

  bool alive = true;  // false after a wait ran out
  int place = warp;   // the warp's next place, from `begin`
  while (true) {  // units of the range
    const int64_t u_begin = max(u.at, begin), u_end = min(u.at + length, end);
    const bool whole = u.at >= begin && u.at + length <= end;
    const int slot = u_begin == begin ? 0 : 1;
    if (u_end <= u.at + kUnitPairs) {  // none of its pages lies in the range
      for (int e = tid; e < kRowsPerTile; e += kThreads) {
        float* ml = ws.ml + ((size_t(blockIdx.x) * 2 + slot) * kRowsPerTile + e) * 2;
        ml[0] = -FLT_MAX;
        ml[1] = 0.f;
      }
      break;  // the range ends here
    }
    load_tile<D, T>(a, seq, u.g * G, u.r, G, q_vec, tid, sm.q, sm.q_sum, sm.q_back, sm.q_seen);
    __syncthreads();
    {
      uint32_t qf[LW][4];
      float f1[2];
      int seen[2];
      const uint32_t qs0 = sm.q_sum[0][gr][tq], qs1 = sm.q_sum[1][gr][tq], qs2 = sm.q_sum[2][gr][tq];
#pragma unroll
      for (int i = 0; i < LW; ++i) *reinterpret_cast<uint4*>(qf[i]) = *reinterpret_cast<const uint4*>(sm.q[i][lane]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        f1[c] = sm.q_back[2 * tq + c];
        seen[c] = sm.q_seen[2 * tq + c];
      }
      const int least = __reduce_min_sync(0xffffffffu, min(seen[0], seen[1]));

      float o[NG][4][4], extra[2][NG], m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {0.f, 0.f};
      float vinv[NG];  // the power of two on V's steps
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        extra[0][g] = extra[1][g] = 0.f;
        vinv[g] = pow2i(126);
#pragma unroll
        for (int i = 0; i < 4; ++i) o[g][i][0] = o[g][i][1] = o[g][i][2] = o[g][i][3] = 0.f;
      }

      const int first = int(u.at - begin) + kUnitPairs, rel_end = int(u_end - begin);
      for (; place < rel_end; place += kWarps) {
        const int done = place / kWarps, stage = done % kStages;
        if (done % 32 == 0) {
          look_up(done + 32 + lane);
          __syncwarp();
        }
        const ulonglong2 from = *reinterpret_cast<const ulonglong2*>(sm.blocks[warp][done & 63]);
        if (!mbar_wait(&sm.full[warp][stage], done / kStages & 1, a.cache.status)) {
          alive = false;
          place = INT_MAX / 2;  // leaves every loop
          break;
        }
        if (!(from.x | from.y)) {
          __syncwarp();
          if (lane == 0) issue(done + kStages, stage);
          continue;
        }
        float s[4][2];  // [key][row]: keys gr and gr + 8 of each page, rows 2 tq and 2 tq + 1
        alignas(16) uint32_t vm[4][NG];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* blk = sm.ring[warp][stage][h];
          float acc[NG][4], part[4];
          alignas(16) uint32_t w0[LW], w1[LW];
#pragma unroll
          for (int i = 0; i < LW; i += L::kChunk) {
            const uint8_t* p0 = blk + ((i / L::kChunk * kPageTokens + gr) * 4 + tq) * L::kChunk * 4;
            const uint8_t* p1 = p0 + 8 * 4 * L::kChunk * 4;
            if constexpr (L::kChunk == 4) {
              *reinterpret_cast<uint4*>(&w0[i]) = *reinterpret_cast<const uint4*>(p0);
              *reinterpret_cast<uint4*>(&w1[i]) = *reinterpret_cast<const uint4*>(p1);
            } else {
              *reinterpret_cast<uint2*>(&w0[i]) = *reinterpret_cast<const uint2*>(p0);
              *reinterpret_cast<uint2*>(&w1[i]) = *reinterpret_cast<const uint2*>(p1);
            }
          }
          const uint32_t m0 = *reinterpret_cast<const uint32_t*>(blk + L::k_meta(gr, tq % NG));
          const uint32_t m1 = *reinterpret_cast<const uint32_t*>(blk + L::k_meta(gr + 8, tq % NG));
#pragma unroll
          for (int j = 0; j < 4; ++j)  // word j / 2 of every group, its low or high bytes
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const int i = 2 * g + j / 2;
              const uint32_t x = j & 1 ? w0[i] >> 8 : w0[i], y = j & 1 ? w1[i] >> 8 : w1[i];
              if (j == 0) mma_f16_first(acc[g], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, qf[i][0], qf[i][1]);
              else mma_f16(acc[g], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, qf[i][2 * (j & 1)], qf[i][2 * (j & 1) + 1]);
            }
          mma_bf16_first(part, m0, m1, m0, m1, qs0, qs1);
          mma_bf16(part, m0, m1, m0, m1, qs2, 0u);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            alignas(16) uint32_t km[NG];
            load_words<NG>(km, blk + L::k_meta(gr + 8 * k, 0));
            load_words<NG>(vm[2 * h + k], blk + L::v_meta(gr + 8 * k, 0));
            float x0 = kv4_scale(km[0]) * acc[0][2 * k], x1 = kv4_scale(km[0]) * acc[0][2 * k + 1];
#pragma unroll
            for (int g = 1; g < NG; ++g) {
              x0 = fmaf(kv4_scale(km[g]), acc[g][2 * k], x0);
              x1 = fmaf(kv4_scale(km[g]), acc[g][2 * k + 1], x1);
            }
            s[2 * h + k][0] = fmaf(x0, f1[0], part[2 * k]);
            s[2 * h + k][1] = fmaf(x1, f1[1], part[2 * k + 1]);
          }
        }
        // keys behind a row's limit and pages that are not there: no weight, and no step or bias that could be NaN
        const int key0 = (place - first) * 2 * kPageTokens;
        const bool edge = key0 + 2 * kPageTokens > least || !from.x || !from.y;
        if (edge) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int key = key0 + gr + 8 * k;
            const bool there = k < 2 ? from.x != 0 : from.y != 0;
            if (!there || key >= seen[0]) s[k][0] = -INFINITY;
            if (!there || key >= seen[1]) s[k][1] = -INFINITY;
            if (!there || key >= seq.len) {
#pragma unroll
              for (int g = 0; g < NG; ++g) vm[k][g] = 0u;
            }
          }
        }
        const float h0 = fmaxf(fmaxf(s[0][0], s[1][0]), fmaxf(s[2][0], s[3][0]));
        const float h1 = fmaxf(fmaxf(s[0][1], s[1][1]), fmaxf(s[2][1], s[3][1]));
        if (__any_sync(0xffffffffu, h0 > m[0] + kLazy || h1 > m[1] + kLazy)) {
          float top[2] = {h0, h1};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 4));
            top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 8));
            top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 16));
            top[c] = fmaxf(top[c], m[c]);
            const float f = exp2_fast(m[c] - top[c]);
            m[c] = top[c];
            l[c] *= f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              extra[c][g] *= f;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                o[g][i][c] *= f;
                o[g][i][2 + c] *= f;
              }
            }
          }
        }
        // V's steps to at most 2^6
        float big = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g)
          big = fmaxf(big, vinv[g] * fmaxf(fmaxf(kv4_scale(vm[0][g]), kv4_scale(vm[1][g])), fmaxf(kv4_scale(vm[2][g]), kv4_scale(vm[3][g]))));
        if (__any_sync(0xffffffffu, big > 64.f)) {
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float top = warp_max(fmaxf(fmaxf(kv4_scale(vm[0][g]), kv4_scale(vm[1][g])), fmaxf(kv4_scale(vm[2][g]), kv4_scale(vm[3][g]))));
            const float fresh = fminf(vinv[g], pow2i(min(126, 132 - int(__float_as_uint(top) >> 23))));
            const float f = pow2i(int(__float_as_uint(fresh) >> 23) - int(__float_as_uint(vinv[g]) >> 23));
            vinv[g] = fresh;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              o[g][i][0] *= f;
              o[g][i][1] *= f;
              o[g][i][2] *= f;
              o[g][i][3] *= f;
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            s[k][c] = exp2_fast(s[k][c] - m[c]);
            l[c] += s[k][c];
          }
        if (edge) {  // a bias that is NaN counts only for the rows that see its key
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const float bias = kv4_bias(vm[k][g]);
              extra[0][g] = fmaf(s[k][0], key0 + gr + 8 * k < seen[0] ? bias : 0.f, extra[0][g]);
              extra[1][g] = fmaf(s[k][1], key0 + gr + 8 * k < seen[1] ? bias : 0.f, extra[1][g]);
            }
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              const float bias = kv4_bias(vm[k][g]);
              extra[0][g] = fmaf(s[k][0], bias, extra[0][g]);
              extra[1][g] = fmaf(s[k][1], bias, extra[1][g]);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t pb[NG][2];
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const float step = kv4_scale(vm[2 * h + k][g]) * vinv[g];
              pb[g][k] = transpose8x8(pack_f16(s[2 * h + k][0] * step, s[2 * h + k][1] * step));
            }
          // nibbles of keys 2 tq, 2 tq + 1 (even places first) and 2 tq + 8, 2 tq + 9
          alignas(16) uint32_t w[4][NG];
          const uint8_t* pv = sm.ring[warp][stage][h] + L::kV + (gr / L::kRows * kPageTokens + tq) * 32 + gr % L::kRows * (D / 16);
#pragma unroll
          for (int k = 0; k < 4; ++k) load_words<NG>(w[k], pv + ((k & 1) * 8 + (k >> 1) * 4) * 32);
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int g = 0; g < NG; ++g) {
              uint32_t x = __byte_perm(w[0][g], w[1][g], b ? 0x7632 : 0x5410);
              uint32_t y = __byte_perm(w[2][g], w[3][g], b ? 0x7632 : 0x5410);
              mma_f16(o[g][2 * b], x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u, pb[g][0], pb[g][1]);
              x >>= 8;
              y >>= 8;
              mma_f16(o[g][2 * b + 1], x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u, pb[g][0], pb[g][1]);
            }
        }
        __syncwarp();
        if (lane == 0) issue(done + kStages, stage);
      }

      // join the warps: row maxima and sums, then the rows one warp at a time
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          l[c] += __shfl_xor_sync(0xffffffffu, l[c], x);
#pragma unroll
          for (int g = 0; g < NG; ++g) extra[c][g] += __shfl_xor_sync(0xffffffffu, extra[c][g], x);
        }
        if (gr == 0) {
          sm.ml[warp][2 * tq + c][0] = m[c];
          sm.ml[warp][2 * tq + c][1] = l[c];
        }
      }
      __syncthreads();
      float f[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float M = -FLT_MAX;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.ml[w][2 * tq + c][0]);
        f[c] = exp2_fast(m[c] - M);
      }
      // gates of the rows this thread will write
      constexpr int kItems = kRowsPerTile * (D / 8) / kThreads > 0 ? kRowsPerTile * (D / 8) / kThreads : 1;
      float gate[kItems][8];
      if (whole && a.gate.data) {
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
          const int e = tid + k * kThreads, row = u.r * kRowsPerTile + e / (D / 8), token = row / G;
          if (e < kRowsPerTile * (D / 8) && token < seq.count)
            load_gate(a, seq.first + token, u.g * G + row % G, e % (D / 8) * 8, gate[k]);
        }
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {  // warps 0, 1 store, then 2, 3 add
        if (warp / 2 == half) {
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float back = pow2i(24 + 127 - int(__float_as_uint(vinv[g]) >> 23));  // 2^24 over the power on V's steps
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float* row = &sm.o[warp % 2][2 * tq + c][64 * g + 8 * gr];
              float y[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                y[2 * i] = fmaf(o[g][i][c], back, extra[c][g]) * f[c];
                y[2 * i + 1] = fmaf(o[g][i][2 + c], back * 0.0625f, extra[c][g]) * f[c];
              }
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                float4 v = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
                float4* at = reinterpret_cast<float4*>(row) + i;
                if (half) {
                  const float4 old = *at;
                  v = make_float4(old.x + v.x, old.y + v.y, old.z + v.z, old.w + v.w);
                }
                *at = v;
              }
            }
          }
        }
        __syncthreads();
      }
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        const int e = tid + k * kThreads;
        if (e >= kRowsPerTile * (D / 8)) break;
        const int rr = e / (D / 8), dim = e % (D / 8) * 8;
        float M = -FLT_MAX, sum = 0.f, y[8];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.ml[w][rr][0]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += sm.ml[w][rr][1] * exp2_fast(sm.ml[w][rr][0] - M);
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          const float4 p = *reinterpret_cast<const float4*>(&sm.o[0][rr][dim + i]);
          const float4 q = *reinterpret_cast<const float4*>(&sm.o[1][rr][dim + i]);
          y[i] = p.x + q.x;
          y[i + 1] = p.y + q.y;
          y[i + 2] = p.z + q.z;
          y[i + 3] = p.w + q.w;
        }
        if (whole) {
          const int row = u.r * kRowsPerTile + rr, token = row / G;
          if (token >= seq.count) continue;
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] *= inv;
          write_dims<T>(a, seq.first + token, u.g * G + row % G, dim, y, gate[k], out_vec);
          if (dim == 0 && a.lse)
            a.lse[size_t(seq.first + token) * a.cache.Hq + u.g * G + row % G] =
                sum == 0.f ? -INFINITY : (M + log2f(sum)) * 0.6931471805599453f;
        } else {
          float* dst = ws.o + ((size_t(blockIdx.x) * 2 + slot) * kRowsPerTile + rr) * D + dim;
#pragma unroll
          for (int i = 0; i < 2; ++i) reinterpret_cast<float4*>(dst)[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
          if (dim == 0) {
            float* ml = ws.ml + ((size_t(blockIdx.x) * 2 + slot) * kRowsPerTile + rr) * 2;
            ml[0] = M;
            ml[1] = sum;
          }
        }
      }
    }
    if (u_end == end) break;
    __syncthreads();
    advance(u, seq, length);
  }
  if (!alive && lane == 0) {
    // a wait ran out: let copies in flight land before the CTA leaves
    for (int i = 0; i < 2 * kStages; ++i) mbar_wait(&sm.full[warp][i % kStages], i / kStages, a.cache.status);
  }
}

// Joins the partial results of a unit whose pages span several CTAs, and
// writes the rows of a unit that has no page. One CTA per unit; a warp per row
// weighs the parts, then the threads sum them.
constexpr int kMergeParts = 64;  // weighed at a time
template <int D, class T>
__global__ void __launch_bounds__(256) kv4_merge_kernel(Kv4AttentionArgs a, int ctas, int tiles, bool out_vec) {
  pdl_trigger();
  pdl_wait();
  __shared__ float weight[kRowsPerTile][kMergeParts], row_m[kRowsPerTile], row_l[kRowsPerTile];
  const int Hkv = a.cache.Hkv, G = a.cache.Hq / Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.x % tiles, g = blockIdx.x / tiles % Hkv, s = blockIdx.x / tiles / Hkv;
  const Workspace ws = carve(a.workspace, a.n_seq, ctas);
  const int64_t first = ws.offsets[s], next = ws.offsets[s + 1], range = *ws.range;
  const Seq seq = load_seq(a, s, G, false);
  if (r >= seq.tiles) return;
  int64_t at = first + g * ((next - first) / Hkv);
  for (int i = 0; i < r; ++i) at += unit_length(seq, i, G);
  const int length = unit_length(seq, r, G);
  const int64_t c0 = at / range, c1 = length ? (at + length - 1) / range : c0 - 1;
  if (length && c0 == c1) return;  // whole in one CTA
  // a CTA's first unit is in its slot 0, another that ends behind it in slot 1
  const auto part = [&](int64_t c) { return size_t(c * 2 + (at > c * range ? 1 : 0)) * kRowsPerTile; };
  constexpr int kItems = kRowsPerTile * (D / 8) / 256 > 0 ? kRowsPerTile * (D / 8) / 256 : 1;
  const int rr = threadIdx.x / (D / 8), dim = threadIdx.x % (D / 8) * 8;
  static_assert(kItems == 1 && kRowsPerTile == 8, "a thread writes 8 dims of one row");
  const int row = r * kRowsPerTile + rr, token = row / G;
  const bool mine = rr < kRowsPerTile && token < seq.count;
  float gate[8], y[8] = {};
  if (mine && a.gate.data) load_gate(a, seq.first + token, g * G + row % G, dim, gate);
  float M = -FLT_MAX, sum = 0.f;
  for (int64_t c = c0; c <= c1; c += kMergeParts) {
    const int n = int(min(c1 - c + 1, int64_t(kMergeParts)));
    float m[kMergeParts / 32], l[kMergeParts / 32], top = M;
#pragma unroll
    for (int k = 0; k < kMergeParts / 32; ++k) {
      const int i = lane + 32 * k;
      m[k] = -FLT_MAX;
      l[k] = 0.f;
      if (i < n) {
        const float2 ml = *reinterpret_cast<const float2*>(ws.ml + (part(c + i) + warp) * 2);
        m[k] = ml.x;
        l[k] = ml.y;
      }
      top = fmaxf(top, m[k]);
    }
    top = warp_max(top);
    const float old = exp2_fast(M - top);
    float add = 0.f;
#pragma unroll
    for (int k = 0; k < kMergeParts / 32; ++k) {
      const float w = exp2_fast(m[k] - top);
      add += l[k] * w;
      weight[warp][lane + 32 * k] = l[k] == 0.f ? 0.f : w;  // a part that saw no key may hold anything
    }
    sum = sum * old + warp_sum(add);
    M = top;
    if (lane == 0) row_m[warp] = old;
    __syncthreads();
    if (mine) {
      const float f = row_m[rr];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] *= f;
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float w = weight[rr][i];
        const float* p = ws.o + (part(c + i) + rr) * D + dim;
        const float4 lo = *reinterpret_cast<const float4*>(p), hi = *reinterpret_cast<const float4*>(p + 4);
        if (w != 0.f) {
          y[0] = fmaf(lo.x, w, y[0]);
          y[1] = fmaf(lo.y, w, y[1]);
          y[2] = fmaf(lo.z, w, y[2]);
          y[3] = fmaf(lo.w, w, y[3]);
          y[4] = fmaf(hi.x, w, y[4]);
          y[5] = fmaf(hi.y, w, y[5]);
          y[6] = fmaf(hi.z, w, y[6]);
          y[7] = fmaf(hi.w, w, y[7]);
        }
      }
    }
    __syncthreads();
  }
  if (lane == 0) {
    row_m[warp] = M;
    row_l[warp] = sum;
  }
  __syncthreads();
  if (!mine) return;
  M = row_m[rr];
  sum = row_l[rr];
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] *= inv;
  write_dims<T>(a, seq.first + token, g * G + row % G, dim, y, gate, out_vec);
  if (dim == 0 && a.lse)
    a.lse[size_t(seq.first + token) * a.cache.Hq + g * G + row % G] =
        sum == 0.f ? -INFINITY : (M + log2f(sum)) * 0.6931471805599453f;
}

// Lane's dims lane E .. lane E + E - 1 of K of one cached token.
template <int D>
__device__ __forceinline__ void load_key(const uint8_t* block, int tok, int lane, float (&x)[D / 32]) {
  using L = Kv4Layout<D>;
  constexpr int E = D / 32;
  const int w = lane * E / 8;
  const uint32_t word = *reinterpret_cast<const uint32_t*>(block + L::k_word(tok, w));
  const uint32_t pair = *reinterpret_cast<const uint32_t*>(block + L::k_meta(tok, w / 8));
#pragma unroll
  for (int e = 0; e < E; ++e)
    x[e] = fmaf(kv4_scale(pair), float((word >> (4 * kv4_k_nibble(lane * E % 8 + e))) & 15u), kv4_bias(pair));
}

// One CTA per (sequence, KV head, page): what each key received from the
// sequence's query tokens and the head's group, added to what it had.
template <int D, class T>
__global__ void __launch_bounds__(128) kv4_weights_kernel(Kv4AttentionArgs a, const float* __restrict__ lse) {
  pdl_trigger();
  pdl_wait(lse);
  constexpr int E = D / 32;
  const int s = blockIdx.y / a.cache.Hkv, g = blockIdx.y % a.cache.Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.cache.Hq / a.cache.Hkv;
  const Seq q = load_seq(a, s, G, false);
  for (int p = blockIdx.x * kPageTokens + warp; p < min(q.len, (int(blockIdx.x) + 1) * kPageTokens); p += 4) {
    const size_t at = (size_t(s) * a.cache.Hkv + g) * a.weights_stride + p;
    float sum = a.weights_in && p < q.len - q.count ? a.weights_in[at] : 0.f;
    const int64_t page = a.table[s * a.table_stride + p / kPageTokens];
    if (page >= 0 && uint64_t(page) < a.cache.pages) {
      float k[E];
      load_key<D>(a.cache.block(uint64_t(page), g), p % kPageTokens, lane, k);
      for (int j = max(0, p - (q.len - q.count)); j < q.count; ++j)
        for (int h = g * G; h < (g + 1) * G; ++h) {
          const T* x = static_cast<const T*>(a.q.data) + (q.first + j) * a.q.token_stride + h * a.q.head_stride;
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) dot = fmaf(kv4_to_float(x[lane * E + e]), k[e], dot);
          sum += __expf(warp_sum(dot) * a.scale - lse[size_t(q.first + j) * a.cache.Hq + h]);
        }
    }
    if (lane == 0) a.weights_out[at] = sum;
  }
}

void count_launch() { g_kernel_launches.fetch_add(1, std::memory_order_relaxed); }

template <int D, class T>
void attend(const Kv4AttentionArgs& a, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, [] {
    QWEN_CUDA(cudaFuncSetAttribute(kv4_decode_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(Smem<D>))));
  });
  Kv4AttentionArgs b = a;
  const int G = a.cache.Hq / a.cache.Hkv, ctas = a.sm_count * kCtasPerSm;
  const int tiles = (a.max_count * G + kRowsPerTile - 1) / kRowsPerTile;
  const bool q_vec = reinterpret_cast<uintptr_t>(a.q.data) % 16 == 0 && a.q.token_stride % 8 == 0 && a.q.head_stride % 8 == 0;
  const bool vec = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_token_stride % 8 == 0 && a.out_head_stride % 8 == 0;
  if (a.weights_out && !a.lse)
    b.lse = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) +
                                     kv4_workspace_bytes(a.cache.Hq, a.cache.Hkv, D, a.n_seq, 0, a.sm_count));
  launch_pdl(kv4_decode_kernel<D, T>, ctas, kThreads, sizeof(Smem<D>), s, b, q_vec, vec);
  count_launch();
  launch_pdl(kv4_merge_kernel<D, T>, dim3(unsigned(a.n_seq * a.cache.Hkv * tiles)), 256, 0, s, b, ctas, tiles, vec);
  count_launch();
  if (a.weights_out) {
    launch_pdl(kv4_weights_kernel<D, T>, dim3(unsigned(a.table_stride), a.n_seq * a.cache.Hkv), 128, 0, s, b,
               static_cast<const float*>(b.lse));
    count_launch();
  }
}

}  // namespace

size_t kv4_workspace_bytes(int Hq, int Hkv, int D, size_t n_seq, size_t tokens, int sm_count) {
  (void)Hkv;
  return align16((n_seq + 2) * 8) + size_t(sm_count) * kCtasPerSm * 2 * kRowsPerTile * (D + 2) * 4 +
         align16(tokens * size_t(Hq) * 4);
}

void launch_kv4_attention(const Kv4AttentionArgs& a, cudaStream_t s) {
  if (a.tokens <= 0 || a.n_seq <= 0) return;
  const bool half = a.type == kKv4F16;
  if (a.cache.D == 64) half ? attend<64, __half>(a, s) : attend<64, __nv_bfloat16>(a, s);
  else if (a.cache.D == 128) half ? attend<128, __half>(a, s) : attend<128, __nv_bfloat16>(a, s);
  else half ? attend<256, __half>(a, s) : attend<256, __nv_bfloat16>(a, s);
}

}  // namespace qwen
