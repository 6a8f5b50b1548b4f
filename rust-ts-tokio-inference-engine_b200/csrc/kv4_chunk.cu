// Attention over the 4-bit paged KV cache for sequences that feed many rows
// (prefill chunks, speculative verification): tcgen05 tiles of 128 query rows.
//
// The (sequence, KV head, tile of 128 rows) units are laid end to end, measured
// in the blocks of 64 keys each has to read, and cut into equal ranges, one per
// CTA (one CTA per SM); a unit cut in two leaves partial results that
// kv4_chunk_merge_kernel joins. Per block:
//   S[128 x 64] = Q K^T   Q in TMEM (128 columns), K in shared memory
//   O[128 x D] += P V     P in TMEM, V^T in shared memory, O in TMEM (D columns)
// so each MMA reads only its B operand from shared memory. Warp roles:
//   0-7   softmax: two threads per row, each with half of a block's keys; they tell
//         each other their maximum, so both hold the row's; sums in registers
//   8-11  dequantisation of K, 12-15 of V: nibbles -> fp16 operands in the 128B-swizzled layout
//   16    MMA issue    17, 18  bulk copies of the pages' K and V parts
// 2048 tokens of 16 + 2 heads of 256 behind 14336 keys: 750 us a call with its
// merge (0.69 PFLOP/s; 838 with one softmax thread per row), this kernel alone 731
// under the profiler. What is left is the chain of a block in the dequantisation
// warps (steps, meeting, values) and, in the last CTA, the table of the units'
// parts, which one thread per sequence writes before its range (20 us for 256 units
// when that loop had one select more).
// The nibbles of the page layout come out as the operands' element pairs: two
// dims of a K row, two keys of a V^T row. Masked, a pair is an fp16 subnormal
// pair n 2^-24 (or n 2^-20), so one fused multiply-add with the step times 2^24
// makes it a value, rounded once. For that step to fit, the operands carry a
// power of two, one for K and one per group of 64 dims of V, kept from block to
// block and raised when a block needs it (O's columns are then rescaled): the
// largest magnitude so far lies in [2^-10, 2^-6), so a value is off by 2^-11 of
// itself or, if it is much smaller than the largest, by 2^-15 of that. The
// softmax weights are rounded to fp16 as well; sums and maxima are 32-bit.
// Calls that ask for the log-sum-exp or the keys' weights, which are 32-bit
// results, do not come here: kv4_decode_kernel multiplies the exact nibbles.
#include <algorithm>
#include <atomic>

#include "kv4_device.cuh"

namespace qwen {

extern std::atomic<uint64_t> g_kernel_launches;

namespace {

constexpr int kRows = 128, kKeys = 64, kBlockPages = kKeys / kPageTokens;
constexpr int kSoftWarps = 8, kDeqWarps = 4, kMmaWarp = 16, kLoadK = 17, kLoadV = 18;
constexpr int kThreads = 20 * 32;  // the last warp only completes its warpgroup
constexpr int kSoftRegs = 104, kOtherRegs = 88;  // of 640 x 96 registers at launch: 256 x 104 + 384 x 88
constexpr int kRaw = 3;         // raw page stages, K and V each
constexpr int kSets = 2;        // sets of steps and biases, K and V each
constexpr int kUnitBlocks = 4;  // what a unit costs beside its blocks, in blocks
constexpr int kMinBlocks = 8;   // shortest range
constexpr int kGroupsMax = 512;
constexpr float kLazy = 8.f;    // log2 of how far a logit may exceed the running maximum
// TMEM columns
constexpr uint32_t kTmO = 0, kTmQ = 256, kTmS = 384, kTmP = 448;

__device__ __forceinline__ int chunk_tiles(const Seq& q, int G, int limit) {
  return q.count * G > limit ? (q.count * G + kRows - 1) / kRows : 0;
}
__device__ __forceinline__ int chunk_pages(const Seq& q, int r, int G) {
  const int token = min(q.count - 1, ((r + 1) * kRows - 1) / G);
  return max(0, q.len - q.count + token + 1 + kPageTokens - 1) / kPageTokens;
}
__device__ __forceinline__ int unit_blocks(const Seq& q, int r, int G) {
  return (chunk_pages(q, r, G) + kBlockPages - 1) / kBlockPages;
}
__device__ __forceinline__ int unit_length(const Seq& q, int r, int G) {
  const int n = unit_blocks(q, r, G);
  return n ? n + kUnitBlocks : 0;
}

struct Workspace {
  int2* units;  // as in the decode kernel, for tiles of 128 rows
  float2* ml;   // [ctas][2][128]
  float* o;     // [ctas][2][128][D]
};
__host__ __device__ inline size_t align16(size_t n) { return (n + 15) & ~size_t(15); }
__host__ __device__ inline size_t unit_entries(size_t tokens, size_t n_seq, int G, int Hkv) {
  return (tokens * G / kRows + n_seq + 1) * Hkv;
}
__device__ __forceinline__ size_t unit_index(const Seq& q, int s, int r, int g, int G, int Hkv) {
  return (size_t(q.first) * G / kRows + s + r) * Hkv + g;
}
__host__ __device__ inline Workspace carve(void* base, size_t units, int ctas) {
  Workspace w;
  uint8_t* p = static_cast<uint8_t*>(base);
  w.units = reinterpret_cast<int2*>(p);
  p += align16(units * 8);
  w.ml = reinterpret_cast<float2*>(p);
  p += size_t(ctas) * 2 * kRows * 8;
  w.o = reinterpret_cast<float*>(p);
  return w;
}

template <int D>
struct Smem {
  static constexpr int kHalf = 8 * D;  // nibbles of K or V of a page and head
  alignas(1024) uint8_t k[2][kKeys * D * 2];  // [stage][chunk of 64 dims][key][128 B]
  alignas(1024) uint8_t v[2][kKeys * D * 2];  // [stage][dim][64 keys]
  alignas(16) uint8_t kraw[kRaw][kBlockPages][kHalf + D];  // nibbles, then pairs
  alignas(16) uint8_t vraw[kRaw][kBlockPages][kHalf + D];
  alignas(16) uint32_t kst[kSets][kKeys][D / 64][4];      // K: step 2^24, step 2^20, bias (each twice, fp16x2)
  alignas(16) uint32_t vst[kSets][D / 64][kKeys / 2][4];  // V: the same for the two keys of a pair
  // by block: K's power of two, V's of every group and the one before, the keys
  // (even, odd of each pair) whose group is NaN
  alignas(8) float2 kinfo[8];               // K's power times 2^-10, and the bits of the pages that are not there
  alignas(4) uint8_t vflags[8][4];          // by group: 1 the power has moved, 2 it holds a NaN
  int ve[8][D / 64], ve_was[8][D / 64];
  uint32_t vnan[8][D / 64][2];
  int absent_v[8];
  int absent[8];                            // pages of a block that are outside the pool, by block
  uint64_t kraw_full[kRaw], kraw_empty[kRaw], vraw_full[kRaw], vraw_empty[kRaw];
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full, s_empty, p_full[2], p_empty[2], q_full, o_empty;
  uint32_t tmem;
  int abort;
  int scan[kThreads / 32];
  float top[2][2][kRows], sum[2][kRows];    // what the two threads of a row tell each other
  int offsets[kGroupsMax + 1];
};

struct Cursor {
  int s, g, r;
  int at;
};

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// The pairs in the low nibbles of x and in the next ones as step * n + bias.
__device__ __forceinline__ uint32_t value_low(uint32_t x, uint32_t step24, uint32_t bias) { return hfma2(x & 0x000F000Fu, step24, bias); }
__device__ __forceinline__ uint32_t value_high(uint32_t x, uint32_t step20, uint32_t bias) { return hfma2(x & 0x00F000F0u, step20, bias); }
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 z, x, y, z;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 z, x, y;\n\t"
      "mov.b64 {%0, %1}, z;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
// Largest magnitude that a pair (scale, bias) stands for.
__device__ __forceinline__ float pair_most(uint32_t pair) {
  return fmaxf(fabsf(kv4_bias(pair)), fabsf(fmaf(15.f, kv4_scale(pair), kv4_bias(pair))));
}
// The power of two that operands are divided by. Divided, magnitudes have to stay
// below 2^-6 (a step is then at most 2^-5 / 15, and 2^24 times that inside fp16);
// a new power puts the largest below 2^-9.
constexpr int kNone = -1000;
struct Power {
  int e = kNone;
  float limit = 0.f;  // magnitudes from here on need a larger power
  float down = 1.f, down2 = 1.f;  // 2^-e, as two factors for the range's ends
  // raises the power if the warp's largest magnitude asks for it (an infinity's does not count)
  __device__ __forceinline__ void raise(float most, bool first) {
    if (first) *this = Power();
    if (__any_sync(0xffffffffu, most > limit && most < INFINITY)) {
      // not below -125, so that 2^(e - 10) is a normal number
      const int top = max(int(__reduce_max_sync(0xffffffffu, most < INFINITY ? __float_as_uint(most) : 0u) >> 23) - 126, -125);
      e = top + 9;
      limit = e > 133 ? FLT_MAX : pow2i(e - 6);
      down = pow2i(-e / 2);
      down2 = pow2i(-e - (-e / 2));
    }
  }
};
__device__ __forceinline__ void sts128(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(smem_u32(p)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int D, class T>
__global__ void __launch_bounds__(kThreads, 1) kv4_chunk_kernel(Kv4AttentionArgs a, void* workspace, bool q_vec, bool gate_vec, bool out_vec) {
  pdl_wait();
  using L = Kv4Layout<D>;
  constexpr int NG = L::kGroups, LW = L::kLaneWords;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int Hkv = a.cache.Hkv, G = a.cache.Hq / Hkv, ctas = gridDim.x;
  const Workspace ws = carve(workspace, unit_entries(a.tokens, a.n_seq, G, Hkv), ctas);

  if (tid == 0) {
    for (int i = 0; i < kRaw; ++i) {
      mbar_init(&sm.kraw_full[i], 1);
      mbar_init(&sm.vraw_full[i], 1);
      mbar_init(&sm.kraw_empty[i], kDeqWarps);
      mbar_init(&sm.vraw_empty[i], kDeqWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sm.k_full[i], kDeqWarps);
      mbar_init(&sm.k_empty[i], 1);
      mbar_init(&sm.v_full[i], kDeqWarps);
      mbar_init(&sm.v_empty[i], 1);
      mbar_init(&sm.p_full[i], kSoftWarps);
      mbar_init(&sm.p_empty[i], 1);
    }
    mbar_init(&sm.s_full, 1);
    mbar_init(&sm.s_empty, kSoftWarps);
    mbar_init(&sm.q_full, kSoftWarps);
    mbar_init(&sm.o_empty, kSoftWarps);
    sm.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }

  // places of the sequences (in groups when there are many), the range, the units' parts for the merge
  const int per = (a.n_seq + kGroupsMax - 1) / kGroupsMax, groups = (a.n_seq + per - 1) / per;
  const int limit = a.row_limit;
  auto seq_at = [&](int s) {
    Seq q = load_seq(a, s, G, false);
    q.tiles = chunk_tiles(q, G, limit);
    return q;
  };
  auto seq_length = [&](const Seq& q) {
    int n = 0;
    for (int r = 0; r < q.tiles; ++r) n += unit_length(q, r, G);
    return n;
  };
  int total = 0;
  for (int g0 = 0; g0 < groups; g0 += kThreads) {
    const int gi = g0 + tid;
    int n = 0;
    for (int s = gi * per; s < min(a.n_seq, (gi + 1) * per); ++s) n = add_places(n, seq_length(seq_at(s)) * Hkv);
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = add_places(x, y);
    }
    if (lane == 31) sm.scan[warp] = x;
    __syncthreads();
    int before = total;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before = add_places(before, sm.scan[w]);
      total = add_places(total, sm.scan[w]);
    }
    if (gi < groups) sm.offsets[gi] = before + x - n;
    __syncthreads();
  }
  const bool over = total == kPlacesMax;
  if (over) {
    if (blockIdx.x == 0 && tid == 0) kv4_flag(a.cache.status, kErrBounds);
    total = 0;
  }
  if (tid == 0) sm.offsets[groups] = total;
  __syncthreads();
  const int range = max(kMinBlocks, (total + ctas - 1) / ctas);
  const int begin = min(int64_t(blockIdx.x) * range, int64_t(total)), end = min(int64_t(begin) + range, int64_t(total));
  if (int(blockIdx.x) == ctas - 1) {
    for (int gi = tid; gi < groups; gi += kThreads) {
      int at = sm.offsets[gi];
      for (int s = gi * per; s < min(a.n_seq, (gi + 1) * per); ++s) {
        const Seq q = seq_at(s);
        for (int i = 0; i < Hkv * q.tiles; ++i) {
          const int n = unit_length(q, i % q.tiles, G), w0 = at / range;
          ws.units[unit_index(q, s, i % q.tiles, i / q.tiles, G, Hkv)] =
              make_int2(w0 * 2 + (at > w0 * range ? 1 : 0), n && !over ? (at + n - 1) / range - w0 + 1 : 0);
          at += n;
        }
      }
    }
  }
  if (begin >= end) return;

  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sm.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_trigger();  // not before the TMEM is taken: a dependent kernel's CTA could hold it and wait for this one
  const uint32_t tmem = sm.tmem;
  volatile int* abort = &sm.abort;
  // False when the wait ran out, here or in another warp (the status word has it).
  // Warps that meet others at a barrier go on all the same, on whatever the shared
  // memory holds and with no further waiting, so that none is left there.
  auto wait = [&](uint64_t* bar, uint32_t parity) { return kv4_wait(bar, parity, a.cache.status, abort); };

  if (warp < kSoftWarps) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));

  // every role walks the same units: f(cursor, sequence, first block, blocks, whole, slot) returns false to give up
  auto for_units = [&](auto f) {
    int lo = 0, hi = groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (sm.offsets[mid] <= begin) lo = mid;
      else hi = mid;
    }
    Cursor u{lo * per, 0, 0, sm.offsets[lo]};
    Seq q;
    int one;
    for (;;) {
      q = seq_at(u.s);
      one = seq_length(q);
      if (u.at + one * Hkv > begin) break;
      u.at += one * Hkv;
      ++u.s;
    }
    u.g = (begin - u.at) / one;
    u.at += u.g * one;
    while (u.at + unit_length(q, u.r, G) <= begin) u.at += unit_length(q, u.r++, G);
    for (;;) {
      const int length = unit_length(q, u.r, G);
      if (length) {
        const int j0 = max(0, begin - u.at - kUnitBlocks), j1 = min(u.at + length, end) - u.at - kUnitBlocks;
        const bool whole = u.at >= begin && u.at + length <= end;
        if (!f(u, q, j0, max(0, j1 - j0), whole, u.at > begin ? 1 : 0)) return;
        if (u.at + length >= end) return;
      }
      u.at += length;
      if (++u.r >= q.tiles) {
        u.r = 0;
        if (++u.g >= Hkv) {
          u.g = 0;
          do q = seq_at(++u.s);
          while (q.tiles == 0);
        }
      }
    }
  };

  if (warp == kLoadK || warp == kLoadV) {
    const bool key = warp == kLoadK;
    uint64_t* full = key ? sm.kraw_full : sm.vraw_full;
    uint64_t* empty = key ? sm.kraw_empty : sm.vraw_empty;
    constexpr int kHalf = Smem<D>::kHalf;
    uint32_t n = 0;  // blocks fetched
    for_units([&](const Cursor& u, const Seq& q, int j0, int blocks, bool, int) {
      const int pages = chunk_pages(q, u.r, G);
      auto look_up = [&](int j) {  // lane < 4: the block of page 4 j + lane
        const int at = j * kBlockPages + lane;
        if (lane >= kBlockPages || at >= pages) return uint64_t(0);
        const int64_t page = a.table[u.s * a.table_stride + at];
        if (page < 0 || uint64_t(page) >= a.cache.pages) {
          kv4_flag(a.cache.status, kErrBounds);
          return uint64_t(0);
        }
        return reinterpret_cast<uint64_t>(a.cache.block(uint64_t(page), u.g));
      };
      uint64_t next = look_up(j0);
      for (int j = j0; j < j0 + blocks; ++j, ++n) {
        const uint64_t from = next;
        if (j + 1 < j0 + blocks) next = look_up(j + 1);
        const int st = n % kRaw;
        if (n >= kRaw && !wait(&empty[st], (n / kRaw - 1) & 1)) return false;
        const uint32_t there = __ballot_sync(0xffffffffu, from != 0);
        if (lane == 0) {
          (key ? sm.absent : sm.absent_v)[n & 7] = ~there & ((1 << kBlockPages) - 1);
          if (there) mbar_expect_tx(&full[st], __popc(there) * (kHalf + D));
          else mbar_arrive(&full[st]);
        }
        __syncwarp();
        if (from) {
          const uint8_t* src = reinterpret_cast<const uint8_t*>(from);
          uint8_t* dst = key ? sm.kraw[st][lane] : sm.vraw[st][lane];
          bulk_load(dst, src + (key ? 0 : L::kV), kHalf, &full[st]);
          bulk_load(dst + kHalf, src + (key ? L::kKMeta : L::kVMeta), D, &full[st]);
        }
        __syncwarp();
      }
      return true;
    });
    // copies in flight land before the CTA leaves (a wait above may have run out)
    for (uint32_t i = n > kRaw ? n - kRaw : 0; i < n; ++i) kv4_wait(&full[i % kRaw], i / kRaw & 1, a.cache.status);
  } else if (warp == kMmaWarp) {
    const uint32_t idesc_s = idesc_f16(kKeys), idesc_o = idesc_f16(D);
    const uint64_t kdesc = smem_desc_sw128(smem_u32(sm.k[0])), vdesc = smem_desc_sw128(smem_u32(sm.v[0]));
    uint32_t n = 0, units = 0;  // blocks and units done
    auto pv = [&](uint32_t i, bool first) {
      if (!wait(&sm.v_full[i & 1], i / 2 & 1) || !wait(&sm.p_full[i & 1], i / 2 & 1)) return false;
      if (first && units > 0 && !wait(&sm.o_empty, (units - 1) & 1)) return false;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k)
          mma_ts(tmem + kTmO, tmem + kTmP + (i & 1) * 32 + k * 8, vdesc + uint64_t((i & 1) * sizeof(sm.v[0]) / 16 + k * 2), idesc_o, !first || k > 0);
        mma_commit(&sm.v_empty[i & 1]);
        mma_commit(&sm.p_empty[i & 1]);
      }
      __syncwarp();
      return true;
    };
    for_units([&](const Cursor&, const Seq&, int, int blocks, bool, int) {
      if (!blocks) return true;
      if (!wait(&sm.q_full, units & 1)) return false;
      for (int j = 0; j < blocks; ++j, ++n) {
        if (!wait(&sm.k_full[n & 1], n / 2 & 1)) return false;
        if (n > 0 && !wait(&sm.s_empty, (n - 1) & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ts(tmem + kTmS, tmem + kTmQ + k * 8, kdesc + uint64_t(((n & 1) * sizeof(sm.k[0]) + (k / 4) * kKeys * 128) / 16 + k % 4 * 2),
                   idesc_s, k > 0);
          mma_commit(&sm.k_empty[n & 1]);
          mma_commit(&sm.s_full);
        }
        __syncwarp();
        if (j > 0 && !pv(n - 1, j == 1)) return false;
      }
      if (!pv(n - 1, blocks == 1)) return false;
      ++units;
      return true;
    });
  } else if (warp >= kSoftWarps && warp < kSoftWarps + kDeqWarps) {
    const int dt = tid - kSoftWarps * 32, dw = dt >> 5;
    uint32_t n = 0;
    Power power;  // the same in all warps, for the groups' products add up
    // Steps and biases of block n as fp16 operands, one set ahead of its values: a
    // warp per group, a lane for keys lane and lane + 32.
    auto scales = [&](const Seq& q, int j, bool first) {
      wait(&sm.kraw_full[n % kRaw], n / kRaw & 1);
      __syncwarp();
      if (dw < NG) {
        float most = 0.f;
        uint32_t own[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int key = lane + 32 * i, page = key / kPageTokens;
          alignas(16) uint32_t pair[NG];
          load_words<NG>(pair, sm.kraw[n % kRaw][page] + Smem<D>::kHalf + key % kPageTokens * NG * 4);
          const bool there = !(sm.absent[n & 7] >> page & 1) && j * kKeys + key < q.len;  // others are masked later
          own[i] = 0u;
#pragma unroll
          for (int g = 0; g < NG; ++g) {
            if (there) most = fmaxf(most, pair_most(pair[g]));
            if (g == dw && there) own[i] = pair[g];
          }
        }
        power.raise(most, first);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float s = kv4_scale(own[i]) * power.down * power.down2 * 1048576.f, b = kv4_bias(own[i]) * power.down * power.down2;
          *reinterpret_cast<uint4*>(sm.kst[n % kSets][lane + 32 * i][dw]) = make_uint4(pack_f16(s * 16.f, s * 16.f), pack_f16(s, s), pack_f16(b, b), 0u);
        }
        if (dt == 0) sm.kinfo[n & 7] = make_float2(power.e == kNone ? 0.f : pow2i(power.e - 10), __int_as_float(sm.absent[n & 7]));
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kDeqWarps * 32) : "memory");
    };
    auto values = [&] {
      const int st = n % kRaw;
      if (n >= 2) wait(&sm.k_empty[n & 1], (n / 2 - 1) & 1);
      __syncwarp();
      const int t = dt % 4;
      alignas(16) uint32_t w[2][LW];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = dt / 4 + 32 * h;
#pragma unroll
        for (int i = 0; i < LW; i += L::kChunk) {
          const uint8_t* p = sm.kraw[st][key / kPageTokens] + ((i / L::kChunk * kPageTokens + key % kPageTokens) * 4 + t) * L::kChunk * 4;
          if constexpr (L::kChunk == 4) *reinterpret_cast<uint4*>(&w[h][i]) = *reinterpret_cast<const uint4*>(p);
          else *reinterpret_cast<uint2*>(&w[h][i]) = *reinterpret_cast<const uint2*>(p);
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int key = dt / 4 + 32 * h;
        uint8_t* dst = sm.k[n & 1] + key * 128;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const uint4 c = *reinterpret_cast<const uint4*>(sm.kst[n % kSets][key][g]);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int half = i ^ (key & 1);  // odd keys the other half first: no two keys of a store share banks
            const uint32_t x = half ? w[h][2 * g + 1] : w[h][2 * g], y = x >> 8;
            sts128(dst + g * kKeys * 128 + ((4 * half + t) ^ (key & 7)) * 16, value_low(x, c.x, c.z), value_high(x, c.y, c.z),
                   value_low(y, c.x, c.z), value_high(y, c.y, c.z));
          }
        }
      }
      proxy_fence();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.kraw_empty[st]);
        mbar_arrive(&sm.k_full[n & 1]);
      }
      ++n;
    };
    for_units([&](const Cursor&, const Seq& q, int j0, int blocks, bool, int) {
      if (blocks) scales(q, j0, true);
      for (int j = 0; j < blocks; ++j) {
        values();
        if (j + 1 < blocks) scales(q, j0 + j + 1, false);
      }
      return true;
    });
  } else if (warp >= kSoftWarps + kDeqWarps && warp < kMmaWarp) {
    const int dt = tid - (kSoftWarps + kDeqWarps) * 32, dw = dt >> 5;
    uint32_t n = 0;
    Power power;  // of this warp's group
    auto scales = [&](const Seq& q, int j, bool first) {  // a warp per group, a lane per pair of keys
      wait(&sm.vraw_full[n % kRaw], n / kRaw & 1);
      __syncwarp();
      if (dw < NG) {
        const int tok = lane * 2 % kPageTokens, page = lane * 2 / kPageTokens;
        const uint8_t* raw = sm.vraw[n % kRaw][page] + Smem<D>::kHalf + tok * NG * 4 + dw * 4;
        uint32_t a0 = *reinterpret_cast<const uint32_t*>(raw), a1 = *reinterpret_cast<const uint32_t*>(raw + NG * 4);
        const bool there = !(sm.absent_v[n & 7] >> page & 1);
        if (!there || j * kKeys + lane * 2 >= q.len) a0 = 0u;
        if (!there || j * kKeys + lane * 2 + 1 >= q.len) a1 = 0u;
        // a NaN stands as zero in the operand; the rows that see it are made NaN
        const uint32_t na = __ballot_sync(0xffffffffu, isnan(kv4_bias(a0))), nb = __ballot_sync(0xffffffffu, isnan(kv4_bias(a1)));
        if (na >> lane & 1) a0 = 0u;
        if (nb >> lane & 1) a1 = 0u;
        const int was = first ? kNone : power.e;
        power.raise(fmaxf(pair_most(a0), pair_most(a1)), first);
        const float s0 = kv4_scale(a0) * power.down * power.down2 * 1048576.f, s1 = kv4_scale(a1) * power.down * power.down2 * 1048576.f;
        *reinterpret_cast<uint4*>(sm.vst[n % kSets][dw][lane]) =
            make_uint4(pack_f16(s0 * 16.f, s1 * 16.f), pack_f16(s0, s1),
                       pack_f16(kv4_bias(a0) * power.down * power.down2, kv4_bias(a1) * power.down * power.down2), 0u);
        if (lane == 0) {
          sm.ve[n & 7][dw] = power.e;
          sm.ve_was[n & 7][dw] = was;
          sm.vnan[n & 7][dw][0] = na;
          sm.vnan[n & 7][dw][1] = nb;
          sm.vflags[n & 7][dw] = (was != kNone && was != power.e ? 1 : 0) | (na | nb ? 2 : 0);
        }
      } else if (lane == 0) {
        sm.vflags[n & 7][dw] = 0;
      }
      asm volatile("bar.sync 2, %0;" ::"n"(kDeqWarps * 32) : "memory");
    };
    auto values = [&] {
      const int st = n % kRaw;
      if (n >= 2) wait(&sm.v_empty[n & 1], (n / 2 - 1) & 1);
      __syncwarp();
#pragma unroll 1
      for (int part = dw; part < 2 * NG; part += kDeqWarps) {
        // Lane = (word of four, octet of keys). A lane takes its octet's four key
        // pairs in an order turned by the octet, so that the loads of a warp touch
        // every bank once; the columns of V^T keep that order (the weights follow).
        const int ko = lane & 7, slot = (lane >> 3) + 4 * ((part & 1) ^ (ko >> 2)), seg = part >> 1;
        const int group = slot % NG, gr = seg * L::kRows + slot / NG;
        const uint8_t* raw = sm.vraw[st][ko >> 1] + seg * kPageTokens * 32 + slot * 4;
        uint8_t* dst = sm.v[n & 1] + (64 * group + 8 * gr) * 128;
        uint32_t r[8][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int pr = (i + ko) & 3, place = 4 * (ko & 1) + pr;
          const uint32_t x = *reinterpret_cast<const uint32_t*>(raw + place * 32), y = *reinterpret_cast<const uint32_t*>(raw + (place + 8) * 32);
          const uint4 c = *reinterpret_cast<const uint4*>(sm.vst[n % kSets][group][ko * 4 + pr]);
          const uint32_t lo = __byte_perm(x, y, 0x5410), hi = __byte_perm(x, y, 0x7632), lo8 = lo >> 8, hi8 = hi >> 8;
          r[0][i] = value_low(lo, c.x, c.z);
          r[1][i] = value_high(lo, c.y, c.z);
          r[2][i] = value_low(lo8, c.x, c.z);
          r[3][i] = value_high(lo8, c.y, c.z);
          r[4][i] = value_low(hi, c.x, c.z);
          r[5][i] = value_high(hi, c.y, c.z);
          r[6][i] = value_low(hi8, c.x, c.z);
          r[7][i] = value_high(hi8, c.y, c.z);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) sts128(dst + i * 128 + ((ko ^ i) & 7) * 16, r[i][0], r[i][1], r[i][2], r[i][3]);
      }
      proxy_fence();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&sm.vraw_empty[st]);
        mbar_arrive(&sm.v_full[n & 1]);
      }
      ++n;
    };
    for_units([&](const Cursor&, const Seq& q, int j0, int blocks, bool, int) {
      if (blocks) scales(q, j0, true);
      for (int j = 0; j < blocks; ++j) {
        values();
        if (j + 1 < blocks) scales(q, j0 + j + 1, false);
      }
      return true;
    });
  } else if (warp < kSoftWarps) {
    // two threads per row, each with half of a block's keys and of O's dims
    const int quadrant = warp & 3, half = warp >> 2, row = quadrant * 32 + lane;
    const uint32_t lanes = tmem + (uint32_t(quadrant * 32) << 16);
    uint32_t n = 0;
    auto both = [&] { asm volatile("bar.sync %0, 64;" ::"r"(3 + quadrant) : "memory"); };
    constexpr int kMine = kKeys / 2;
    for_units([&](const Cursor& u, const Seq& q, int j0, int blocks, bool whole, int slot) {
      const int at = u.r * kRows + row, token = at / G, head = u.g * G + at % G;
      const bool real = token < q.count;
      float m = -FLT_MAX, l = 0.f;
      if (blocks) {
        // the row as fp16, scaled by a power of two so that its largest value lies in [2^13, 2^14)
        const T* src = static_cast<const T*>(a.q.data) + (q.first + token) * a.q.token_stride + head * a.q.head_stride;
        auto load8 = [&](int d, T* x) {
          if (!real) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = kv4_from_float<T>(0.f);
          } else if (q_vec) {
            *reinterpret_cast<uint4*>(x) = *reinterpret_cast<const uint4*>(src + d);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = src[d + e];
          }
        };
        uint32_t most = 0u;
#pragma unroll 2
        for (int d = 0; d < D; d += 8) {
          alignas(16) T x[8];
          load8(d, x);
#pragma unroll
          for (int e = 0; e < 8; ++e) most = max(most, __float_as_uint(kv4_to_float(x[e])) & 0x7FFFFFFFu);
        }
        const bool fine = most < 0x7F800000u;
        // at least -110: f1 below is then a normal number, and fp16 has room for the smaller row
        const int e = most && fine ? max(int(most >> 23) - 126, -110) : 0;
        const float up = pow2i((14 - e) / 2), up2 = fine ? pow2i(14 - e - (14 - e) / 2) : 0.f;
#pragma unroll 1
        for (int d = 64 * half; d < D; d += 128) {
          uint32_t v[32];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            alignas(16) T x[8];
            load8(d + 8 * k, x);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              v[4 * k + i] = fine ? pack_f16(kv4_to_float(x[2 * i]) * up * up2, kv4_to_float(x[2 * i + 1]) * up * up2) : 0u;
          }
          tmem_st32(lanes + kTmQ + d / 2, v);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.q_full);
        const float factor = a.scale * 1.4426950408889634f;
        const float f1 = factor * pow2i((e - 4) / 2) * pow2i(e - 4 - (e - 4) / 2);  // 2^(e - 14), and the 2^10 that K's power lacks
        const int seen = real ? q.len - q.count + token + 1 : INT_MAX;
        const int least = __reduce_min_sync(0xffffffffu, seen);
        uint32_t poison = 0u;  // groups of which the row sees a NaN
        for (int j = j0; j < j0 + blocks; ++j, ++n) {
          wait(&sm.s_full, n & 1);
          tc_fence_after();
          float2 x[kMine / 2];
          {
            uint32_t s[kMine];
            __syncwarp();
            tmem_ld32(lanes + kTmS + kMine * half, s);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < kMine / 2; ++i) x[i] = make_float2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1]));
          }
          tc_fence_before();
          const float2 info = sm.kinfo[n & 7];
          const int absent = __float_as_int(info.y);
          float fk = fmaxf(f1 * info.x, FLT_MIN);  // above zero: a masked -infinity stays one
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.s_empty);
          const int key0 = j * kKeys + kMine * half;
          if (key0 + kMine > least || absent) {
            const int gone = absent >> (kMine / kPageTokens * half);
#pragma unroll
            for (int i = 0; i < kMine / 2; ++i) {
              if (key0 + 2 * i >= seen || (gone >> (2 * i / kPageTokens) & 1)) x[i].x = -INFINITY;
              if (key0 + 2 * i + 1 >= seen || (gone >> (2 * i / kPageTokens) & 1)) x[i].y = -INFINITY;
            }
          }
          float tops[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) tops[i] = fmaxf(x[i].x, x[i].y);
#pragma unroll
          for (int i = 4; i < kMine / 2; ++i) tops[i % 4] = fmaxf(fmaxf(tops[i % 4], x[i].x), x[i].y);
          float most = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
          sm.top[n & 1][half][row] = most;
          both();
          most = fmaxf(most, sm.top[n & 1][half ^ 1][row]);
          const float top = most * fk;
          const bool grow = top > m + kLazy;
          float shrink = 1.f;
          if (grow) {
            shrink = exp2_fast(m - top);
            m = top;
            l *= shrink;
          }
          // The fused difference below is off by the maximum's own rounding, the same
          // for the whole row. Beyond 2^24 that could be large: round the products first.
          if (__any_sync(0xffffffffu, fabsf(m) > 16777216.f && m > -FLT_MAX)) {
#pragma unroll
            for (int i = 0; i < kMine / 2; ++i) x[i] = make_float2(x[i].x * fk, x[i].y * fk);
            fk = 1.f;
          }
          // weights, packed octet by octet in V^T's order of the key pairs
          float2 sum = make_float2(0.f, 0.f);
          uint32_t p[kMine / 2];
#pragma unroll
          for (int o = 0; o < kMine / 8; ++o) {
#pragma unroll
            for (int i = 4 * o; i < 4 * o + 4; ++i) {
              x[i] = fma2(x[i], make_float2(fk, fk), make_float2(-m, -m));
              x[i].x = exp2_fast(x[i].x);
              x[i].y = exp2_fast(x[i].y);
              sum = add2(sum, x[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 v = x[4 * o + ((i + o) & 3)];
              p[4 * o + i] = pack_f16(v.x, v.y);
            }
          }
          l += sum.x + sum.y;
          // With V of this block in place the MMAs on the block before the last are done, so P's buffer is free too
          wait(&sm.v_full[n & 1], n / 2 & 1);
          __syncwarp();
          tmem_st16(lanes + kTmP + (n & 1) * 32 + kMine / 2 * half, p);
          const uint32_t flags = *reinterpret_cast<const uint32_t*>(sm.vflags[n & 7]);
          const bool moved = flags & 0x01010101u;
          if (flags & 0x02020202u) {
#pragma unroll 1
            for (int g = 0; g < NG; ++g)
#pragma unroll 1
              for (int i = 0; i < kKeys; ++i)
                if ((sm.vnan[n & 7][g][i & 1] >> (i / 2) & 1) && j * kKeys + i < seen) poison |= 1u << g;
          }
          if (j > j0 && (moved || __any_sync(0xffffffffu, grow))) {
            // O so far to the new maximum and powers, when the MMAs on it are done
            wait(&sm.p_empty[(n - 1) & 1], ((n - 1) / 2) & 1);
            __syncwarp();
            tc_fence_after();
#pragma unroll 1
            for (int c = D / 2 * half; c < D / 2 * (half + 1); c += 32) {
              const int was = sm.ve_was[n & 7][c / 64];
              const float f = shrink * (was == kNone ? 1.f : pow2i(was - sm.ve[n & 7][c / 64]));
              uint32_t v[32];
              tmem_ld32(lanes + kTmO + c, v);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
              tmem_st32(lanes + kTmO + c, v);
            }
          }
          tmem_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sm.p_full[n & 1]);
        }
        // the rows
        wait(&sm.p_empty[(n - 1) & 1], ((n - 1) / 2) & 1);
        sm.sum[half][row] = l;
        both();
        l += sm.sum[half ^ 1][row];
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const size_t part = (size_t(blockIdx.x) * 2 + slot) * kRows + row;
#pragma unroll 1
        for (int c = D / 2 * half; c < D / 2 * (half + 1); c += 16) {
          uint32_t v[16];
          tmem_ld16(lanes + kTmO + c, v);
          tmem_wait_ld();
          const int e2 = sm.ve[(n - 1) & 7][c / 64];
          float f = pow2i(e2 == kNone ? 0 : e2 / 2) * (whole ? inv : 1.f);
          const float f2 = pow2i(e2 == kNone ? 0 : e2 - e2 / 2);
          // a query that is not finite went in as zeros: NaN where the row has seen a key, and zero where it has none
          if ((poison >> (c / 64) & 1) || (!fine && l != 0.f)) f = NAN;
          if (real) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float y[8], gate[8];
              if (whole && a.gate.data) load_gate(a, q.first + token, head, c + 8 * h, gate_vec, gate);
#pragma unroll
              for (int i = 0; i < 8; ++i) y[i] = __uint_as_float(v[8 * h + i]) * f * f2;
              if (whole) {
                write_dims<T>(a, q.first + token, head, c + 8 * h, y, gate, out_vec);
              } else {
                float4* dst = reinterpret_cast<float4*>(ws.o + part * D + c + 8 * h);
                dst[0] = make_float4(y[0], y[1], y[2], y[3]);
                dst[1] = make_float4(y[4], y[5], y[6], y[7]);
              }
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sm.o_empty);
      }
      if (!whole && real && half == 0) {
        const size_t part = (size_t(blockIdx.x) * 2 + slot) * kRows + row;
        ws.ml[part] = make_float2(m, l);
        if (!blocks)
          for (int c = 0; c < D; c += 4) *reinterpret_cast<float4*>(ws.o + part * D + c) = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      return true;
    });
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

// Joins the parts of a unit that spans CTAs and writes the rows of one that sees
// no key. A warp per row, eight rows per CTA: 28 us for 256 units of 128 rows, about
// 150 of which lie in two CTAs (58 MB read; issue slots 37 %, waits for memory
// first). The grid has the longest sequence's tiles for every sequence: beside 120
// decoding sequences the same chunk's grid has 496 thousand CTAs, 4096 of them with
// rows, and the call takes 1.38 ms instead of 0.8.
template <int D, class T>
__global__ void __launch_bounds__(256) kv4_chunk_merge_kernel(Kv4AttentionArgs a, void* workspace, int ctas, int tiles) {
  pdl_trigger();
  pdl_wait();
  constexpr int E = D / 32;
  const int Hkv = a.cache.Hkv, G = a.cache.Hq / Hkv, lane = threadIdx.x & 31;
  const int r = blockIdx.x % tiles, g = blockIdx.x / tiles % Hkv, s = blockIdx.x / tiles / Hkv;
  Seq q = load_seq(a, s, G, false);
  q.tiles = chunk_tiles(q, G, a.row_limit);
  const int row = int(blockIdx.y) * 8 + int(threadIdx.x >> 5), at = r * kRows + row, token = at / G, head = g * G + at % G;
  if (r >= q.tiles || token >= q.count) return;
  const Workspace ws = carve(workspace, unit_entries(a.tokens, a.n_seq, G, Hkv), ctas);
  const int2 unit = ws.units[unit_index(q, s, r, g, G, Hkv)];
  if (unit.y == 1) return;
  float M = -FLT_MAX, sum = 0.f, y[E] = {};
  for (int i = 0; i < unit.y; ++i) {
    const size_t part = size_t(i ? (unit.x / 2 + i) * 2 : unit.x) * kRows + row;
    const float2 ml = ws.ml[part];
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = ws.o[part * D + 32 * e + lane];
    const float top = fmaxf(M, ml.x), f0 = exp2_fast(M - top), f1 = exp2_fast(ml.x - top);
    M = top;
    sum = sum * f0 + ml.y * f1;
#pragma unroll
    for (int e = 0; e < E; ++e) y[e] = y[e] * f0 + v[e] * f1;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int dim = 32 * e + lane;
    float v = y[e] * inv;
    if (a.gate.data)
      v *= sigmoid_fast(static_cast<const float*>(a.gate.data)[(q.first + token) * a.gate.token_stride + head * a.gate.head_stride + dim]);
    static_cast<T*>(a.out)[(q.first + token) * a.out_token_stride + head * a.out_head_stride + dim] = kv4_from_float<T>(v);
  }
}

// Tiles of the longest sequence.
int most_tiles(const Kv4AttentionArgs& a) { return int((int64_t(a.max_count) * (a.cache.Hq / a.cache.Hkv) + kRows - 1) / kRows); }

template <int D, class T>
void chunk(const Kv4AttentionArgs& a, void* workspace, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, [] {
    QWEN_CUDA(cudaFuncSetAttribute(kv4_chunk_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(Smem<D>))));
  });
  const int G = a.cache.Hq / a.cache.Hkv, tiles = most_tiles(a);
  const bool q_vec = reinterpret_cast<uintptr_t>(a.q.data) % 16 == 0 && a.q.token_stride % 8 == 0 && a.q.head_stride % 8 == 0;
  const bool gate_vec = reinterpret_cast<uintptr_t>(a.gate.data) % 16 == 0 && a.gate.token_stride % 4 == 0 && a.gate.head_stride % 4 == 0;
  const bool vec = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_token_stride % 8 == 0 && a.out_head_stride % 8 == 0;
  launch_pdl(kv4_chunk_kernel<D, T>, a.sm_count, kThreads, sizeof(Smem<D>), s, a, workspace, q_vec, gate_vec, vec);
  launch_pdl(kv4_chunk_merge_kernel<D, T>, dim3(unsigned(a.n_seq * a.cache.Hkv * tiles), unsigned((std::min(kRows, a.max_count * G) + 7) / 8)), 256,
             0, s, a, workspace, a.sm_count, tiles);
  g_kernel_launches.fetch_add(2, std::memory_order_relaxed);
}

}  // namespace

size_t kv4_chunk_workspace_bytes(int Hq, int Hkv, int D, size_t n_seq, size_t tokens, int sm_count) {
  return align16(unit_entries(tokens, n_seq, Hq / Hkv, Hkv) * 8) + size_t(sm_count) * 2 * kRows * (D + 2) * 4;
}

void check_kv4_chunk(const Kv4AttentionArgs& a) {
  if (tiles_at_most(a, most_tiles(a), kRows) * a.cache.Hkv >= kPlacesMax / (a.table_stride / kBlockPages + 1 + kUnitBlocks) ||
      int64_t(a.n_seq) * a.cache.Hkv * most_tiles(a) > INT32_MAX)
    throw std::invalid_argument("kv4 attention: kv_heads x query tiles x pages beyond 2^31; split the call");
}

void launch_kv4_chunk(const Kv4AttentionArgs& a, void* workspace, cudaStream_t s) {
  const bool half = a.type == kKv4F16;
  if (a.cache.D == 64) half ? chunk<64, __half>(a, workspace, s) : chunk<64, __nv_bfloat16>(a, workspace, s);
  else if (a.cache.D == 128) half ? chunk<128, __half>(a, workspace, s) : chunk<128, __nv_bfloat16>(a, workspace, s);
  else half ? chunk<256, __half>(a, workspace, s) : chunk<256, __nv_bfloat16>(a, workspace, s);
}

}  // namespace qwen
