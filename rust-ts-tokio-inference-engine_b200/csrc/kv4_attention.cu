// Attention over the 4-bit paged KV cache.
//
// kv4_decode_kernel: the (sequence, KV head, tile of 8 query rows) units of a
// call are laid end to end, measured in the pages each has to read, and cut
// into equal ranges, one per CTA; a unit that spans CTAs leaves partial results
// that kv4_merge_kernel joins. The lengths live on the device, so every CTA
// finds its range itself from a prefix sum over the sequences.
//
// The pages of a range are dealt to the CTA's warps through private
// shared-memory rings; in one more warp each lane owns a ring slot and keeps it
// filled, one bulk copy per (page, KV head) block, across unit borders. A warp
// works on 16 keys x 8 query rows:
//   S^T = K Q^T. An fp16 subnormal with the bits 0000 0000 0000 nnnn is n 2^-24
//   and one with nnnn 0000 is n 2^-20, exactly, so the masks 0x000F000F and
//   0x00F000F0 turn a word of nibbles into MMA operands with no conversion; the
//   factor 2^4 between the two is taken out of Q. Scale and bias of a group of
//   64 dims enter afterwards in 32 bits: s = scale (q . n) + bias (sum of q).
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

constexpr int kWarps = 4;   // that compute; one more fetches
constexpr int kStages = 4;  // pages of a warp's ring
constexpr int kThreads = (kWarps + 1) * 32;
constexpr int kCtasPerSm = 2;
constexpr int kRowsPerTile = 8;
constexpr int kMinPages = 8;  // fewest pages of a CTA's range
static_assert(kWarps * kStages <= 32, "one fetching lane per ring slot");
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
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {  // does not wait
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
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
__device__ __forceinline__ int64_t seq_pages(const Seq& q, int G) {  // of one KV head
  int64_t n = 0;
  for (int r = 0; r < q.tiles; ++r) n += tile_pages(q, r, G);
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

// Writes 8 dims of one output row: y / l, gated.
template <class T>
__device__ __forceinline__ void write_dims(const Kv4AttentionArgs& a, int token, int head, int dim, float (&y)[8], bool vec) {
  if (a.gate.data) {
    const float* g = static_cast<const float*>(a.gate.data) + token * a.gate.token_stride + head * a.gate.head_stride + dim;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= sigmoidf_(g[i]);
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
  alignas(128) uint8_t ring[kWarps][kStages][Kv4Layout<D>::kBlock];
  alignas(16) float o[kRowsPerTile][D];
  float ml[kWarps][kRowsPerTile][2];
  int64_t scan[kWarps + 1];
  int64_t start_offset;
  int start_seq;
  int absent[kWarps][kStages];  // the slot's page is outside the pool
  uint64_t full[kWarps][kStages], empty[kWarps][kStages];
};

__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWarps * 32) : "memory"); }

// Position in the laid-out units.
struct Cursor {
  int s, g, r;
  int64_t at;  // page offset of the unit
};

template <int D, class T>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) kv4_decode_kernel(Kv4AttentionArgs a, bool out_vec) {
  pdl_trigger();
  pdl_wait();
  using L = Kv4Layout<D>;
  constexpr int NG = L::kGroups, LW = L::kLaneWords;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  const int Hkv = a.cache.Hkv, G = a.cache.Hq / Hkv;
  const Workspace ws = carve(a.workspace, a.n_seq, gridDim.x);
  if (tid < kWarps * kStages) {
    mbar_init(&sm.full[0][0] + tid, 1);
    mbar_init(&sm.empty[0][0] + tid, 1);
  }
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");

  // total pages, then the sequence in which this CTA's range starts
  int64_t total = 0;
  {
    int64_t mine = 0;
    for (int s = tid; s < a.n_seq; s += blockDim.x)
      mine += seq_pages(load_seq(a, s, G, blockIdx.x == 0), G) * Hkv;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    if (lane == 0) sm.scan[warp] = mine;
    __syncthreads();
#pragma unroll
    for (int w = 0; w <= kWarps; ++w) total += sm.scan[w];
    __syncthreads();
  }
  const int64_t range = max(int64_t(kMinPages), (total + gridDim.x - 1) / gridDim.x);
  const int64_t begin = blockIdx.x * range, end = min(total, begin + range);
  if (blockIdx.x == 0 && tid == 0) *ws.range = range;
  if (begin < end || blockIdx.x == 0) {
    int64_t base = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += blockDim.x) {
      const int s = s0 + tid;
      const int64_t n = s < a.n_seq ? seq_pages(load_seq(a, s, G, false), G) * Hkv : 0;
      int64_t x = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
      }
      if (lane == 31) sm.scan[warp] = x;
      __syncthreads();
      int64_t before = base, sum = 0;
#pragma unroll
      for (int w = 0; w <= kWarps; ++w) {
        if (w < warp) before += sm.scan[w];
        sum += sm.scan[w];
      }
      const int64_t off = before + x - n;
      if (blockIdx.x == 0) {
        if (s < a.n_seq) ws.offsets[s] = off;
        if (s == a.n_seq - 1) ws.offsets[a.n_seq] = off + n;
      }
      if (n && begin >= off && begin < off + n) {
        sm.start_seq = s;
        sm.start_offset = off;
      }
      base += sum;
      __syncthreads();
    }
  }
  if (begin >= end) return;

  // cursor at the unit that holds `begin`
  auto advance = [&](Cursor& c, Seq& q, int& pages) {  // to the next unit with pages
    do {
      c.at += pages;
      if (++c.r >= q.tiles) {
        c.r = 0;
        if (++c.g >= Hkv) {
          c.g = 0;
          do q = load_seq(a, ++c.s, G, false);
          while (q.tiles == 0);
        }
      }
      pages = tile_pages(q, c.r, G);
    } while (pages == 0);
  };
  Cursor u{sm.start_seq, 0, 0, sm.start_offset};
  Seq seq = load_seq(a, u.s, G, false);
  int pages = tile_pages(seq, 0, G);
  while (pages == 0 || u.at + pages <= begin) advance(u, seq, pages);

  if (warp == kWarps) {
    // lane = (warp, slot): its pages are begin + warp + kWarps (slot + kStages n)
    if (lane >= kWarps * kStages) return;
    const int w = lane / kStages, slot = lane % kStages;
    int64_t p = begin + w + int64_t(kWarps) * slot;
    int64_t block = -1;
    auto look_up = [&] {
      while (u.at + pages <= p) advance(u, seq, pages);
      const int64_t page = a.table[u.s * a.table_stride + (p - u.at)];
      const bool ok = page >= 0 && uint64_t(page) < a.cache.pages;
      if (!ok) kv4_flag(a.cache.status, kErrBounds);
      block = ok ? page * Hkv + u.g : -1;
    };
    if (p < end) look_up();
    uint32_t n = 0;  // pages this lane has fetched
    long long t0 = clock64();
    while (p < end) {
      if (n == 0 || mbar_test(&sm.empty[w][slot], (n - 1) & 1u)) {
        sm.absent[w][slot] = block < 0;
        if (block < 0) {
          mbar_arrive(&sm.full[w][slot]);
        } else {
          mbar_expect_tx(&sm.full[w][slot], L::kBlock);
          bulk_load(sm.ring[w][slot], a.cache.pool + uint64_t(block) * L::kBlock, L::kBlock, &sm.full[w][slot]);
        }
        ++n;
        p += kWarps * kStages;
        if (p < end) look_up();
        t0 = clock64();
      } else if (clock64() - t0 > 2 * kWaitCycles) {
        kv4_flag(a.cache.status, kErrTimeout);
        break;
      } else {
        __nanosleep(40);
      }
    }
    // every copy has landed before the CTA may leave
    if (n) mbar_wait(&sm.full[w][slot], (n - 1) & 1u, a.cache.status);
    return;
  }

  bool alive = true;  // false after a wait ran out
  int done = 0;       // pages this warp has finished
  {
    while (true) {  // units of the range
      const int64_t u_begin = max(u.at, begin), u_end = min(u.at + pages, end);
      // query rows of the tile: B fragments (row gr), sums and factors (rows 2 tq, 2 tq + 1)
      static_assert(sizeof(T) == 2, "query type");
      uint32_t qf[LW][4];
      float f1[2], qs[2][NG];
      int seen[2];
      {
        const int row = u.r * kRowsPerTile + gr, token = row / G;
        const bool real = token < seq.count;
        const T* src = static_cast<const T*>(a.q.data) + (seq.first + token) * a.q.token_stride +
                       (u.g * G + row % G) * a.q.head_stride;
        float x[LW][8], most = 0.f, sum[NG];
        bool fine = true;
#pragma unroll
        for (int g = 0; g < NG; ++g) sum[g] = 0.f;
#pragma unroll
        for (int i = 0; i < LW; ++i) {
          const int dim = 64 * (i / 2) + 32 * (i % 2) + 8 * tq;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            x[i][e] = real ? kv4_to_float(src[dim + e]) : 0.f;
            fine = fine && isfinite(x[i][e]);
            most = fmaxf(most, fabsf(x[i][e]));
            sum[i / 2] += x[i][e];
          }
        }
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        fine = __shfl_xor_sync(0xffffffffu, int(fine), 1) && fine;
        fine = __shfl_xor_sync(0xffffffffu, int(fine), 2) && fine;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
          sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
          if (!fine) sum[g] = NAN;  // the row's logits are then all NaN
        }
        // |row| < 2^e: the row times 2^(14 - e) stays below 2^14
        const int e = most > 0.f && fine ? int(__float_as_uint(most) >> 23) - 126 : 0;
        const float up = pow2i((14 - e) / 2), up2 = pow2i(14 - e - (14 - e) / 2);
#pragma unroll
        for (int i = 0; i < LW; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float lift = j & 1 ? 0.0625f : 1.f;  // against the nibbles that carry 2^4
            qf[i][j] = fine ? pack_f16(x[i][2 * j] * up * up2 * lift, x[i][2 * j + 1] * up * up2 * lift) : 0u;
          }
        const float factor = a.scale * 1.4426950408889634f;
        // (q . n) 2^-24 2^(14 - e) -> logit in base 2
        const float back = factor * pow2i((e + 10) / 2) * pow2i(e + 10 - (e + 10) / 2);
        const int lim = real ? seq.len - seq.count + token + 1 : INT_MAX;  // rows past the last are not written
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int from = (2 * tq + c) * 4;
          f1[c] = __shfl_sync(0xffffffffu, back, from);
          seen[c] = __shfl_sync(0xffffffffu, lim, from);
#pragma unroll
          for (int g = 0; g < NG; ++g) qs[c][g] = __shfl_sync(0xffffffffu, sum[g], from) * factor;
        }
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

      for (; begin + warp + int64_t(done) * kWarps < u_end; ++done) {
        const int stage = done % kStages;
        if (!alive) continue;
        if (!mbar_wait(&sm.full[warp][stage], done / kStages & 1, a.cache.status)) {
          alive = false;
          continue;
        }
        if (sm.absent[warp][stage]) {
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.empty[warp][stage]);
          continue;
        }
        const uint8_t* blk = sm.ring[warp][stage];
        // S^T: keys gr and gr + 8, rows 2 tq and 2 tq + 1
        float acc[NG][4];
#pragma unroll
        for (int g = 0; g < NG; ++g) acc[g][0] = acc[g][1] = acc[g][2] = acc[g][3] = 0.f;
        {
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
#pragma unroll
          for (int i = 0; i < LW; ++i) {
            mma_f16(acc[i / 2], w0[i] & 0x000F000Fu, w1[i] & 0x000F000Fu, w0[i] & 0x00F000F0u, w1[i] & 0x00F000F0u, qf[i][0], qf[i][1]);
            const uint32_t h0 = w0[i] >> 8, h1 = w1[i] >> 8;
            mma_f16(acc[i / 2], h0 & 0x000F000Fu, h1 & 0x000F000Fu, h0 & 0x00F000F0u, h1 & 0x00F000F0u, qf[i][2], qf[i][3]);
          }
        }
        alignas(16) uint32_t vm[2][NG];
        float s[2][2];  // [key][row]
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t* kp = reinterpret_cast<const uint32_t*>(blk + L::k_meta(gr + 8 * k, 0));
          const uint32_t* vp = reinterpret_cast<const uint32_t*>(blk + L::v_meta(gr + 8 * k, 0));
          alignas(16) uint32_t km[NG];
          if constexpr (NG == 4) {
            *reinterpret_cast<uint4*>(km) = *reinterpret_cast<const uint4*>(kp);
            *reinterpret_cast<uint4*>(vm[k]) = *reinterpret_cast<const uint4*>(vp);
          } else if constexpr (NG == 2) {
            *reinterpret_cast<uint2*>(km) = *reinterpret_cast<const uint2*>(kp);
            *reinterpret_cast<uint2*>(vm[k]) = *reinterpret_cast<const uint2*>(vp);
          } else {
            km[0] = kp[0];
            vm[k][0] = vp[0];
          }
          float x0 = 0.f, x1 = 0.f, b0 = 0.f, b1 = 0.f;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            x0 = fmaf(kv4_scale(km[g]), acc[g][2 * k], x0);
            x1 = fmaf(kv4_scale(km[g]), acc[g][2 * k + 1], x1);
            b0 = fmaf(kv4_bias(km[g]), qs[0][g], b0);
            b1 = fmaf(kv4_bias(km[g]), qs[1][g], b1);
          }
          s[k][0] = fmaf(x0, f1[0], b0);
          s[k][1] = fmaf(x1, f1[1], b1);
        }
        // keys behind a row's limit: no weight, and no step or bias that could be NaN
        const int key0 = int(begin + warp + int64_t(done) * kWarps - u.at) * kPageTokens;
        const bool edge = key0 + kPageTokens > least;
        if (edge) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int key = key0 + gr + 8 * k;
            if (key >= seen[0]) s[k][0] = -INFINITY;
            if (key >= seen[1]) s[k][1] = -INFINITY;
            if (key >= seq.len) {
#pragma unroll
              for (int g = 0; g < NG; ++g) vm[k][g] = 0u;
            }
          }
        }
        const float h0 = fmaxf(s[0][0], s[1][0]), h1 = fmaxf(s[0][1], s[1][1]);
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
        float p[2][2];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            p[k][c] = exp2_fast(s[k][c] - m[c]);
            l[c] += p[k][c];
          }
        // V's steps to at most 2^6
        float big = 0.f;
#pragma unroll
        for (int g = 0; g < NG; ++g) big = fmaxf(big, fmaxf(kv4_scale(vm[0][g]), kv4_scale(vm[1][g])) * vinv[g]);
        if (__any_sync(0xffffffffu, big > 64.f)) {
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            const float top = warp_max(fmaxf(kv4_scale(vm[0][g]), kv4_scale(vm[1][g])));
            const float fresh = fminf(vinv[g], pow2i(min(126, 132 - int(__float_as_uint(top) >> 23))));
            const float f = fresh / vinv[g];
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
        uint32_t pb[NG][2];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float step = kv4_scale(vm[k][g]) * vinv[g], bias = kv4_bias(vm[k][g]);
            pb[g][k] = transpose8x8(pack_f16(p[k][0] * step, p[k][1] * step));
            if (edge) {  // a bias that is NaN counts only for the rows that see its key
              if (key0 + gr + 8 * k < seen[0]) extra[0][g] = fmaf(p[k][0], bias, extra[0][g]);
              if (key0 + gr + 8 * k < seen[1]) extra[1][g] = fmaf(p[k][1], bias, extra[1][g]);
            } else {
              extra[0][g] = fmaf(p[k][0], bias, extra[0][g]);
              extra[1][g] = fmaf(p[k][1], bias, extra[1][g]);
            }
          }
        {
          // nibbles of keys 2 tq, 2 tq + 1 (even places first) and 2 tq + 8, 2 tq + 9
          alignas(16) uint32_t w[4][NG];
          const uint8_t* pv = blk + L::kV + (gr / L::kRows * kPageTokens + tq) * 32 + gr % L::kRows * (D / 16);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint8_t* q = pv + ((k & 1) * 8 + (k >> 1) * 4) * 32;
            if constexpr (NG == 4) *reinterpret_cast<uint4*>(w[k]) = *reinterpret_cast<const uint4*>(q);
            else if constexpr (NG == 2) *reinterpret_cast<uint2*>(w[k]) = *reinterpret_cast<const uint2*>(q);
            else w[k][0] = *reinterpret_cast<const uint32_t*>(q);
          }
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t x = __byte_perm(w[0][g], w[1][g], h ? 0x7632 : 0x5410);
              uint32_t y = __byte_perm(w[2][g], w[3][g], h ? 0x7632 : 0x5410);
              mma_f16(o[g][2 * h], x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u, pb[g][0], pb[g][1]);
              x >>= 8;
              y >>= 8;
              mma_f16(o[g][2 * h + 1], x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u, pb[g][0], pb[g][1]);
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.empty[warp][stage]);
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
      consumers_sync();
      float f[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float M = -FLT_MAX;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.ml[w][2 * tq + c][0]);
        f[c] = exp2_fast(m[c] - M);
      }
      for (int w = 0; w < kWarps; ++w) {
        if (w == warp) {
#pragma unroll
          for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float* row = &sm.o[2 * tq + c][64 * g + 8 * gr];
              const float back = 16777216.f / vinv[g];  // 2^24 over the power on V's steps
              float y[8];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                y[2 * i] = fmaf(o[g][i][c], back, extra[c][g]) * f[c];
                y[2 * i + 1] = fmaf(o[g][i][2 + c], back * 0.0625f, extra[c][g]) * f[c];
              }
              if (w > 0) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] += row[i];
              }
#pragma unroll
              for (int i = 0; i < 2; ++i) reinterpret_cast<float4*>(row)[i] = make_float4(y[4 * i], y[4 * i + 1], y[4 * i + 2], y[4 * i + 3]);
            }
        }
        consumers_sync();
      }
      const bool whole = u.at >= begin && u.at + pages <= end;
      const int slot = u_begin == begin ? 0 : 1;
      for (int e = tid; e < kRowsPerTile * (D / 8); e += kWarps * 32) {
        const int rr = e / (D / 8), dim = e % (D / 8) * 8;
        float M = -FLT_MAX, sum = 0.f, y[8];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.ml[w][rr][0]);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum += sm.ml[w][rr][1] * exp2_fast(sm.ml[w][rr][0] - M);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = sm.o[rr][dim + i];
        if (whole) {
          const int row = u.r * kRowsPerTile + rr, token = row / G;
          if (token >= seq.count) continue;
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] *= inv;
          write_dims<T>(a, seq.first + token, u.g * G + row % G, dim, y, out_vec);
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
      consumers_sync();
      if (u_end == end) break;
      advance(u, seq, pages);
    }
  }
}

// Joins the partial results of a unit whose pages span several CTAs, and
// writes the rows of a unit that has no page. One CTA per unit.
template <int D, class T>
__global__ void __launch_bounds__(256) kv4_merge_kernel(Kv4AttentionArgs a, int ctas, int tiles, bool out_vec) {
  pdl_trigger();
  pdl_wait();
  const int Hkv = a.cache.Hkv, G = a.cache.Hq / Hkv;
  const int r = blockIdx.x % tiles, g = blockIdx.x / tiles % Hkv, s = blockIdx.x / tiles / Hkv;
  const Seq seq = load_seq(a, s, G, false);
  if (r >= seq.tiles) return;
  const Workspace ws = carve(a.workspace, a.n_seq, ctas);
  int64_t at = ws.offsets[s] + g * ((ws.offsets[s + 1] - ws.offsets[s]) / Hkv);
  for (int i = 0; i < r; ++i) at += tile_pages(seq, i, G);
  const int pages = tile_pages(seq, r, G);
  const int64_t range = *ws.range;
  const int64_t c0 = at / range, c1 = pages ? (at + pages - 1) / range : c0;
  if (pages && c0 == c1) return;  // whole in one CTA
  for (int e = threadIdx.x; e < kRowsPerTile * (D / 8); e += blockDim.x) {
    const int rr = e / (D / 8), dim = e % (D / 8) * 8, row = r * kRowsPerTile + rr, token = row / G;
    if (token >= seq.count) continue;
    float M = -FLT_MAX, sum = 0.f, y[8] = {};
    if (pages) {
      for (int64_t c = c0; c <= c1; ++c) {
        const size_t slot = (size_t(c) * 2 + (max(at, c * range) == c * range ? 0 : 1)) * kRowsPerTile + rr;
        const float2 ml = *reinterpret_cast<const float2*>(ws.ml + slot * 2);
        const float4 lo = *reinterpret_cast<const float4*>(ws.o + slot * D + dim);
        const float4 hi = *reinterpret_cast<const float4*>(ws.o + slot * D + dim + 4);
        const float top = fmaxf(M, ml.x), f0 = exp2_fast(M - top), f1 = exp2_fast(ml.x - top);
        M = top;
        sum = sum * f0 + ml.y * f1;
        y[0] = y[0] * f0 + lo.x * f1;
        y[1] = y[1] * f0 + lo.y * f1;
        y[2] = y[2] * f0 + lo.z * f1;
        y[3] = y[3] * f0 + lo.w * f1;
        y[4] = y[4] * f0 + hi.x * f1;
        y[5] = y[5] * f0 + hi.y * f1;
        y[6] = y[6] * f0 + hi.z * f1;
        y[7] = y[7] * f0 + hi.w * f1;
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] *= inv;
    write_dims<T>(a, seq.first + token, g * G + row % G, dim, y, out_vec);
    if (dim == 0 && a.lse)
      a.lse[size_t(seq.first + token) * a.cache.Hq + g * G + row % G] =
          sum == 0.f ? -INFINITY : (M + log2f(sum)) * 0.6931471805599453f;
  }
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
  const bool vec = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_token_stride % 8 == 0 && a.out_head_stride % 8 == 0;
  if (a.weights_out && !a.lse)
    b.lse = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) +
                                     kv4_workspace_bytes(a.cache.Hq, a.cache.Hkv, D, a.n_seq, 0, a.sm_count));
  launch_pdl(kv4_decode_kernel<D, T>, ctas, kThreads, sizeof(Smem<D>), s, b, vec);
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
