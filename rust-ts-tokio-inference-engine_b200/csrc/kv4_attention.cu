// Attention over the 4-bit paged KV cache.
//
// kv4_decode_kernel: the (sequence, KV head, tile of 8 query rows) units of a
// call are laid end to end, measured in the page pairs each has to read, and cut
// into equal ranges, one per warp of the grid; a unit that spans warps leaves
// partial results that kv4_merge_kernel joins. The lengths live on the device,
// so every CTA finds the ranges itself from a prefix sum over the sequences;
// after it the warps never wait for one another.
// 64 sequences of 128 to 32768 keys, 2 KV heads of 256 (219 MB): 66 us with
// the merge behind it, against 33 at the copy's rate. Two things fill the rest: an
// SM has work for 105 of the profiled launch's 135 thousand cycles, for equal
// ranges do not end together, and some 14 thousand of them start the ranges. 128
// sequences of 4 tokens: 100 us, bound by the instructions of the four tiles.
//
// A warp streams its pages through a private shared-memory ring, one bulk copy
// per (page, KV head) block, across unit borders, and works on 2 x 16 keys x 8
// query rows at a time:
//   S^T = K Q^T. An fp16 subnormal with the bits 0000 0000 0000 nnnn is n 2^-24
//   and one with nnnn 0000 is n 2^-20, exactly, so the masks 0x000F000F and
//   0x00F000F0 turn a word of nibbles into MMA operands with no conversion; the
//   factor 2^4 between the two is taken out of Q. Scale and bias of a group of
//   64 dims enter afterwards in 32 bits: s = scale (q . n) + bias (sum of q).
//   The stored pairs (scale, bias) are themselves a bf16 operand: against
//   (0, sum of q), the sums split into three bf16 terms, two MMAs give the
//   bias part of all 16 keys.
//   Q is fp16, each row scaled by a power of two, so fp16 and bf16 queries are
//   exact (bf16 has fewer mantissa bits and the row keeps its range). Brought back,
//   a row of 2^116 / scale and above overflows and comes out NaN; below 2^-110 the
//   three terms of its sums lose bits.
//   O^T += V^T P^T. The nibbles of two keys are interleaved into k pairs and
//   masked the same way. The step of V is folded into the weights, P_g = p
//   scale_g, rounded to fp16 (2^-11 of a weight, the operand's own precision)
//   after a power of two per group has brought the scales that the warp has seen
//   to at most 2^6; sum p bias_g is kept in 32 bits beside it. Since n is not
//   centred, that rounding moves a row by 2^-11 of twice its size, which bf16
//   rows do not show but fp16 rows do (4.6e-4 relative to 64 bits for 33
//   sequences of head_dim 128, of which fp16's own rounding is 2.1e-4): for fp16
//   what the rounding left out is multiplied too.
// The running maximum moves only when a logit exceeds it by 2^8: a vote per
// page then replaces the reduction over the keys, and the weights stay below
// 2^8 x 2^6, inside fp16.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv4_device.cuh"

namespace qwen {

extern std::atomic<uint64_t> g_kernel_launches;

namespace {

constexpr int kWarps = 4;
constexpr int kStages = 2;  // page pairs of a warp's ring
constexpr int kThreads = kWarps * 32;
constexpr int kCtasPerSm = 2;
constexpr int kMinPairs = 7;     // shortest range
constexpr int kUnitPairs = 3;    // what a unit costs beside its pages, in page pairs
constexpr int kGroupsMax = 512;  // entries of the prefix table that finds a place's sequence
constexpr float kLazy = 8.f;     // log2 of how far a logit may exceed the running maximum

// Length of a unit: its page pairs behind kUnitPairs places that hold none, so
// that ranges of equal length take equal time whatever the units' sizes.
__device__ __forceinline__ int unit_length(const Seq& q, int r, int G) {
  const int pages = tile_pages(q, r, G);
  return pages ? (pages + 1) / 2 + kUnitPairs : 0;
}
__device__ __forceinline__ int seq_length(const Seq& q, int G) {  // of one KV head
  int n = 0;
  for (int r = 0; r < q.tiles; ++r) n += unit_length(q, r, G);
  return n;
}

// Workspace: where the parts of every unit are, then per warp of the grid two
// partial results: the unit that its range starts in, and another that the range
// ends in.
struct Workspace {
  int2* units;  // [tiles][Hkv], see unit_index: the unit's first part, number of warps that worked on it
  float2* ml;   // [warps][2][8]: row maximum and sum
  float* o;     // [warps][2][8][D]
};
__host__ __device__ inline size_t align16(size_t n) { return (n + 15) & ~size_t(15); }
// Entry of (sequence, tile r, KV head g) without a prefix sum: a sequence has at
// most as many tiles as its rows alone would fill, and one more.
__device__ __forceinline__ size_t unit_index(const Seq& q, int s, int r, int g, int G, int Hkv) {
  return (size_t(q.first) * G / kRowsPerTile + s + r) * Hkv + g;
}
__host__ __device__ inline size_t unit_entries(size_t tokens, size_t n_seq, int G, int Hkv) {
  return (tokens * G / kRowsPerTile + n_seq + 1) * Hkv;
}
__host__ __device__ inline Workspace carve(void* base, size_t units, int workers) {
  Workspace w;
  uint8_t* p = static_cast<uint8_t*>(base);
  w.units = reinterpret_cast<int2*>(p);
  p += align16(units * 8);
  w.ml = reinterpret_cast<float2*>(p);
  p += size_t(workers) * 2 * kRowsPerTile * 8;
  w.o = reinterpret_cast<float*>(p);
  return w;
}

template <int D>
struct Smem {
  alignas(128) uint8_t ring[kWarps][kStages][2][Kv4Layout<D>::kBlock];
  alignas(16) uint64_t blocks[kWarps][64][2];  // blocks of a warp's next places, two windows of 32; 0: none
  uint64_t full[kWarps][kStages];
  int scan[kWarps];
  int offsets[kGroupsMax + 1];  // first place of each group of sequences
  int first[kGroupsMax], count[kGroupsMax], len[kGroupsMax];  // of each sequence, when groups are single ones
};

// Position in the laid-out units.
struct Cursor {
  int s, g, r;
  int at;  // the unit's first place
};

template <int D, class T>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) kv4_decode_kernel(Kv4AttentionArgs a, bool q_vec, bool gate_vec, bool out_vec) {
  pdl_trigger();
  pdl_wait();
  using L = Kv4Layout<D>;
  constexpr bool kFine = std::is_same_v<T, __half>;
  constexpr int NG = L::kGroups, LW = L::kLaneWords;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  Smem<D>& sm = *reinterpret_cast<Smem<D>*>(smem_raw);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  const int Hkv = a.cache.Hkv, G = a.cache.Hq / Hkv;
  const int workers = int(gridDim.x) * kWarps, worker = warp * int(gridDim.x) + int(blockIdx.x);
  const Workspace ws = carve(a.workspace, unit_entries(a.tokens, a.n_seq, G, Hkv), workers);
  if (tid < kWarps * kStages) mbar_init(&sm.full[0][0] + tid, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");

  // places of the sequences, in groups of `per` when there are many
  const int per = (a.n_seq + kGroupsMax - 1) / kGroupsMax, groups = (a.n_seq + per - 1) / per;
  int total = 0;
  for (int g0 = 0; g0 < groups; g0 += kThreads) {
    const int gi = g0 + tid;
    int n = 0;
    for (int s = gi * per; s < min(a.n_seq, (gi + 1) * per); ++s) {
      const Seq q = load_seq(a, s, G, blockIdx.x == 0);
      n = add_places(n, seq_length(q, G) * Hkv);
      sm.first[gi] = q.first;
      sm.count[gi] = q.count;
      sm.len[gi] = q.len;
    }
    int x = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = add_places(x, y);
    }
    if (lane == 31) sm.scan[warp] = x;
    __syncthreads();
    int before = total;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
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
  const int range = max(kMinPairs, (total + workers - 1) / workers);
  const int begin = min(int64_t(worker) * range, int64_t(total)), end = min(int64_t(begin) + range, int64_t(total));
  auto seq_at = [&](int s) {
    if (per > 1) return load_seq(a, s, G, false);
    Seq q{sm.first[s], sm.count[s], sm.len[s], 0};
    q.tiles = q.count * G > a.row_limit ? 0 : (q.count * G + kRowsPerTile - 1) / kRowsPerTile;
    return q;
  };
  if (blockIdx.x == gridDim.x - 1) {  // for the merge
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

  // the unit that holds place p, not before group `lo`
  auto locate = [&](int p, int lo, Cursor& c, Seq& q) {
    int hi = groups;  // the last group that starts at or before p
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (sm.offsets[mid] <= p) lo = mid;
      else hi = mid;
    }
    c.s = lo * per;
    c.at = sm.offsets[lo];
    int one;
    for (;;) {
      q = seq_at(c.s);
      one = seq_length(q, G);
      if (c.at + one * Hkv > p) break;
      c.at += one * Hkv;
      ++c.s;
    }
    c.g = (p - c.at) / one;
    c.at += c.g * one;
    c.r = 0;
    while (c.at + unit_length(q, c.r, G) <= p) c.at += unit_length(q, c.r++, G);
  };
  Cursor u;
  Seq seq;
  locate(begin, 0, u, seq);
  int length = unit_length(seq, u.r, G);

  // the warp's places are begin + i; window w holds i = 32 w .. 32 w + 31
  const int n_mine = end - begin;
  auto look_up = [&](int i) {
    if (i >= n_mine) return;
    const int p = begin + i;
    Cursor c = u;
    Seq q = seq;
    if (p >= u.at + length) locate(p, u.s / per, c, q);
    const int at = (p - c.at - kUnitPairs) * 2, pages = tile_pages(q, c.r, G);
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
  // The pages in flight fill the memory system's queues, so a load that a unit
  // starts or ends with would wait behind them: its lines are asked for ahead.
  auto prefetch_rows = [&](const Kv4Rows& r, int bytes, int s_first, int tokens, int tile, int head0) {
    const int lines = D * bytes / 128;  // of a row
    for (int i = lane; i < kRowsPerTile * lines; i += 32) {
      const int row = tile * kRowsPerTile + i / lines, token = row / G;
      if (token < tokens)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const uint8_t*>(r.data) +
                                                      ((s_first + token) * r.token_stride + (head0 + row % G) * r.head_stride) * bytes + i % lines * 128));
    }
  };

  prefetch_rows(a.q, 2, seq.first, seq.count, u.r, u.g * G);
  look_up(lane);
  __syncwarp();
  if (lane == 0)
    for (int i = 0; i < kStages; ++i) issue(i, i);

  int done = 0;  // places this warp has finished
  while (true) {  // units of the range
    const int u_end = min(u.at + length, end);
    const bool whole = u.at >= begin && u.at + length <= end;
    if (whole && a.gate.data) prefetch_rows(a.gate, 4, seq.first, seq.count, u.r, u.g * G);
    if (u_end < end) {
      if (u.r + 1 < seq.tiles) prefetch_rows(a.q, 2, seq.first, seq.count, u.r + 1, u.g * G);
      else if (u.g + 1 < Hkv) prefetch_rows(a.q, 2, seq.first, seq.count, 0, (u.g + 1) * G);
      else if (u.s + 1 < a.n_seq) {
        const Seq q = seq_at(u.s + 1);
        prefetch_rows(a.q, 2, q.first, q.count, 0, 0);
      }
    }
    // The query rows as B fragments: lane = 4 row + t, register j of word i holds
    // dims 2 j, 2 j + 1 of the word's eight. A row is scaled by a power of two so
    // that its largest value lies in [2^13, 2^14); the pairs that meet nibbles
    // carrying 2^4 are lowered by as much. A row with a value that is not finite
    // gets NaN sums, so its logits are all NaN.
    uint32_t qf[LW][4], qs[3];
    float f1[2];
    int seen[2];
    {
      const int row = u.r * kRowsPerTile + gr, token = row / G;
      const bool real = token < seq.count;
      const T* src = static_cast<const T*>(a.q.data) + (seq.first + token) * a.q.token_stride + (u.g * G + row % G) * a.q.head_stride;
      alignas(16) T x[LW][8];
#pragma unroll
      for (int i = 0; i < LW; ++i) {
        const T* p = src + 64 * (i / 2) + 32 * (i % 2) + 8 * tq;
        if (!real) {
          *reinterpret_cast<uint4*>(x[i]) = make_uint4(0u, 0u, 0u, 0u);
        } else if (q_vec) {
          *reinterpret_cast<uint4*>(x[i]) = *reinterpret_cast<const uint4*>(p);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[i][e] = p[e];
        }
      }
      uint32_t most = 0u;  // bits of the largest magnitude; a NaN's are above every number's
      float sum[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        sum[g] = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = kv4_to_float(x[2 * g + e / 8][e % 8]);
          sum[g] += v;
          most = max(most, __float_as_uint(v) & 0x7FFFFFFFu);
        }
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 1);
        sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], 2);
      }
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
      const bool fine = most < 0x7F800000u;
      const int e = most && fine ? int(most >> 23) - 126 : 0;  // |row| < 2^e
      const float up = pow2i((14 - e) / 2), up2 = fine ? pow2i(14 - e - (14 - e) / 2) : 0.f, low = up2 * 0.0625f;
#pragma unroll
      for (int i = 0; i < LW; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          qf[i][j] = fine ? pack_f16(kv4_to_float(x[i][2 * j]) * up * (j & 1 ? low : up2),
                                     kv4_to_float(x[i][2 * j + 1]) * up * (j & 1 ? low : up2)) : 0u;
      const float factor = a.scale * 1.4426950408889634f;
      // this lane's group sum in three bf16 terms, each above a zero (against the scale)
      float rest = 0.f;
#pragma unroll
      for (int g = 0; g < NG; ++g)
        if (tq == g) rest = fine ? sum[g] * factor : NAN;
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        qs[i] = uint32_t(float_to_bf16_bits(rest)) << 16;
        rest -= __uint_as_float(qs[i]);
      }
      const float back = factor * pow2i((e + 10) / 2) * pow2i(e + 10 - (e + 10) / 2);  // (q . n) 2^-24 to a logit in base 2
      const int limit = real ? seq.len - seq.count + token + 1 : INT_MAX;  // rows past the last are not written
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        f1[c] = __shfl_sync(0xffffffffu, back, (2 * tq + c) * 4);
        seen[c] = __shfl_sync(0xffffffffu, limit, (2 * tq + c) * 4);
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
    const int first = u.at - begin + kUnitPairs, rel_end = u_end - begin;
    for (; done < rel_end; ++done) {
      const int stage = done % kStages;
      if (done % 32 == 0) {
        look_up(done + 32 + lane);
        __syncwarp();
      }
      const ulonglong2 from = *reinterpret_cast<const ulonglong2*>(sm.blocks[warp][done & 63]);
      if (!kv4_wait(&sm.full[warp][stage], done / kStages & 1, a.cache.status)) {
        // a wait ran out: let the copies in flight land before leaving
        if (lane == 0)
          for (int i = 0; i < 2 * kStages; ++i) kv4_wait(&sm.full[warp][i % kStages], i / kStages, a.cache.status);
        return;
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
        mma_bf16_first(part, m0, m1, m0, m1, qs[0], qs[1]);
        mma_bf16(part, m0, m1, m0, m1, qs[2], 0u);
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
      const int key0 = (done - first) * 2 * kPageTokens;
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
        uint32_t pb[NG][2], rest[kFine ? NG : 1][2];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float step = kv4_scale(vm[2 * h + k][g]) * vinv[g];
            const float p0 = s[2 * h + k][0] * step, p1 = s[2 * h + k][1] * step;
            const uint32_t p = pack_f16(p0, p1);
            pb[g][k] = transpose8x8(p);
            if (kFine) {
              const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&p));
              rest[g][k] = transpose8x8(pack_f16(p0 - r.x, p1 - r.y));
            }
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
            if (kFine) mma_f16(o[g][2 * b], x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u, rest[g][0], rest[g][1]);
            x >>= 8;
            y >>= 8;
            mma_f16(o[g][2 * b + 1], x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u, pb[g][0], pb[g][1]);
            if (kFine) mma_f16(o[g][2 * b + 1], x & 0x000F000Fu, x & 0x00F000F0u, y & 0x000F000Fu, y & 0x00F000F0u, rest[g][0], rest[g][1]);
          }
      }
      __syncwarp();
      if (lane == 0) issue(done + kStages, stage);
    }

    // the unit's rows, or this warp's part of them; all gates are asked for at once
    float gate[2][NG][8];
    if (whole && a.gate.data) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = u.r * kRowsPerTile + 2 * tq + c, token = row / G;
        if (token < seq.count) {
#pragma unroll
          for (int g = 0; g < NG; ++g) load_gate(a, seq.first + token, u.g * G + row % G, 64 * g + 8 * gr, gate_vec, gate[c][g]);
        }
      }
    }
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) {
        l[c] += __shfl_xor_sync(0xffffffffu, l[c], x);
#pragma unroll
        for (int g = 0; g < NG; ++g) extra[c][g] += __shfl_xor_sync(0xffffffffu, extra[c][g], x);
      }
    const size_t part = (size_t(worker) * 2 + (u.at > begin ? 1 : 0)) * kRowsPerTile;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int rr = 2 * tq + c, row = u.r * kRowsPerTile + rr, token = row / G, head = u.g * G + row % G;
      const float inv = l[c] == 0.f ? 0.f : 1.f / l[c];
      if (whole && token >= seq.count) continue;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const float back = pow2i(24 + 127 - int(__float_as_uint(vinv[g]) >> 23));  // 2^24 over the power on V's steps
        const int dim = 64 * g + 8 * gr;
        float y[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          y[2 * i] = fmaf(o[g][i][c], back, extra[c][g]);
          y[2 * i + 1] = fmaf(o[g][i][2 + c], back * 0.0625f, extra[c][g]);
        }
        if (whole) {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] *= inv;
          write_dims<T>(a, seq.first + token, head, dim, y, gate[c][g], out_vec);
        } else {
          float4* dst = reinterpret_cast<float4*>(ws.o + (part + rr) * D + dim);
          dst[0] = make_float4(y[0], y[1], y[2], y[3]);
          dst[1] = make_float4(y[4], y[5], y[6], y[7]);
        }
      }
      if (gr == 0) {
        if (!whole) ws.ml[part + rr] = make_float2(m[c], l[c]);
        else if (a.lse) a.lse[size_t(seq.first + token) * a.cache.Hq + head] = l[c] == 0.f ? -INFINITY : (m[c] + log2f(l[c])) * 0.6931471805599453f;
      }
    }
    if (u_end == end) return;
    do {  // the next unit that has pages
      u.at += length;
      if (++u.r >= seq.tiles) {
        u.r = 0;
        if (++u.g >= Hkv) {
          u.g = 0;
          do seq = seq_at(++u.s);
          while (seq.tiles == 0);
        }
      }
      length = unit_length(seq, u.r, G);
    } while (length == 0);
  }
}

// Joins the partial results of a unit whose pages span several warps, and writes
// the rows of a unit that has no page. One CTA per (unit, row): its threads
// weigh the parts while they fetch them, D / 4 threads to a part. 7 us for 128 units
// of 8 rows (64 sequences), 16 for 1024: the latency of unit, statistics, parts
// (issue slots 39 %, waits for memory first). The grid has the longest sequence's
// tiles for every sequence, so many short ones beside a long chunk pay for CTAs that
// find no row.
constexpr int kMergeThreads = 128, kMergeFetch = 8;
template <int D, class T>
__global__ void __launch_bounds__(kMergeThreads) kv4_merge_kernel(Kv4AttentionArgs a, int workers, int tiles) {
  pdl_trigger();
  pdl_wait();
  constexpr int kLanes = D / 4, kSets = kMergeThreads / kLanes;  // parts read at a time
  __shared__ float weight[kMergeThreads], red[2][kMergeThreads / 32];
  __shared__ alignas(16) float sums[kSets][D];
  const int Hkv = a.cache.Hkv, G = a.cache.Hq / Hkv, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r = blockIdx.x % tiles, g = blockIdx.x / tiles % Hkv, s = blockIdx.x / tiles / Hkv, rr = blockIdx.y;
  const Workspace ws = carve(a.workspace, unit_entries(a.tokens, a.n_seq, G, Hkv), workers);
  const Seq seq = load_seq(a, s, G, false);
  const int row = r * kRowsPerTile + rr, token = row / G, head = g * G + row % G;
  if (r >= seq.tiles || token >= seq.count) return;  // a tile without rows has no entry either
  const int2 unit = ws.units[unit_index(seq, s, r, g, G, Hkv)];
  const int n = unit.y;
  if (n == 1) return;  // whole in one warp
  // part 0 is at unit.x; the others lie in part 0 of the following warps
  const auto part = [&](int i) { return size_t(i ? (unit.x / 2 + i) * 2 : unit.x) * kRowsPerTile + rr; };
  const int set = tid / kLanes, dim = tid % kLanes * 4;
  float4 gate;
  if (set == 0 && a.gate.data) {
    const float* p = static_cast<const float*>(a.gate.data) + (seq.first + token) * a.gate.token_stride + head * a.gate.head_stride + dim;
    gate = make_float4(p[0], p[1], p[2], p[3]);
  }
  float M = -FLT_MAX, sum = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += kMergeThreads) {
    const int m = min(n - i0, kMergeThreads);
    const float2 ml = tid < m ? ws.ml[part(i0 + tid)] : make_float2(-FLT_MAX, 0.f);
    float4 v[kMergeFetch];
#pragma unroll
    for (int k = 0; k < kMergeFetch; ++k)
      if (set + k * kSets < m) v[k] = *reinterpret_cast<const float4*>(ws.o + part(i0 + set + k * kSets) * D + dim);
    float top = warp_max(ml.x);
    if (lane == 0) red[0][warp] = top;
    __syncthreads();
    top = M;
#pragma unroll
    for (int i = 0; i < kMergeThreads / 32; ++i) top = fmaxf(top, red[0][i]);
    const float f = exp2_fast(ml.x - top), old = exp2_fast(M - top), add = warp_sum(ml.y * f);
    weight[tid] = f;
    if (lane == 0) red[1][warp] = add;
    __syncthreads();
    M = top;
    sum *= old;
#pragma unroll
    for (int i = 0; i < kMergeThreads / 32; ++i) sum += red[1][i];
    y = make_float4(y.x * old, y.y * old, y.z * old, y.w * old);
    for (int i = set; i < m; i += kSets * kMergeFetch) {
#pragma unroll
      for (int k = 0; k < kMergeFetch; ++k) {
        if (i + k * kSets < m) {
          const float w = weight[i + k * kSets];
          y = make_float4(fmaf(v[k].x, w, y.x), fmaf(v[k].y, w, y.y), fmaf(v[k].z, w, y.z), fmaf(v[k].w, w, y.w));
        }
      }
#pragma unroll
      for (int k = 0; k < kMergeFetch; ++k) {
        const int next = i + (k + kMergeFetch) * kSets;
        if (next < m) v[k] = *reinterpret_cast<const float4*>(ws.o + part(i0 + next) * D + dim);
      }
    }
    __syncthreads();
  }
  *reinterpret_cast<float4*>(&sums[set][dim]) = y;
  __syncthreads();
  if (set) return;
#pragma unroll
  for (int i = 1; i < kSets; ++i) {
    const float4 v = *reinterpret_cast<const float4*>(&sums[i][dim]);
    y = make_float4(y.x + v.x, y.y + v.y, y.z + v.z, y.w + v.w);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  y = make_float4(y.x * inv, y.y * inv, y.z * inv, y.w * inv);
  if (a.gate.data) y = make_float4(y.x * sigmoid_fast(gate.x), y.y * sigmoid_fast(gate.y), y.z * sigmoid_fast(gate.z), y.w * sigmoid_fast(gate.w));
  T* out = static_cast<T*>(a.out) + (seq.first + token) * a.out_token_stride + head * a.out_head_stride + dim;
  out[0] = kv4_from_float<T>(y.x);
  out[1] = kv4_from_float<T>(y.y);
  out[2] = kv4_from_float<T>(y.z);
  out[3] = kv4_from_float<T>(y.w);
  if (tid == 0 && a.lse)
    a.lse[size_t(seq.first + token) * a.cache.Hq + head] = sum == 0.f ? -INFINITY : (M + log2f(sum)) * 0.6931471805599453f;
}

// What every cached key received from the call's query rows, added to what it
// had: sum over the rows of exp(logit - lse), with the logits multiplied again from
// the exact nibbles, as in the decode kernel. The K half of the pages is read once
// more, 144 bytes a key at head_dim 256; logits kept in 32 bits would be written and
// read instead, 8 bytes a key and row, which is less up to 17 rows. One CTA per
// (sequence, KV head, 64 pages), eight pages per warp; a key's sum belongs to one
// warp, rows in order, so there are no atomics. 32 sequences of 256 to 16384 keys, 2
// KV heads of 256: 19 us (2 TB/s of nibbles and weights; issue slots 34 %, waits for
// memory first: latency, not bytes). 2048 tokens behind 14336 keys: 8.6 ms, the
// instructions of 2048 tiles.
constexpr int kWtWarps = 8, kWtPages = 8, kWtTiles = 4;  // pages of a warp; tiles of query rows held at a time

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

template <int D>
struct WtSmem {
  alignas(16) uint32_t q[kWtTiles][Kv4Layout<D>::kLaneWords][32][4];
  uint32_t sum[kWtTiles][3][kRowsPerTile][4];
  float back[kWtTiles][kRowsPerTile], lse[kWtTiles][kRowsPerTile];
  int seen[kWtTiles][kRowsPerTile];
  float acc[kWtWarps][kWtPages][kPageTokens];
};

template <int D, class T>
__global__ void __launch_bounds__(kWtWarps * 32) kv4_weights_kernel(Kv4AttentionArgs a, int chunks, bool q_vec) {
  pdl_trigger();
  pdl_wait();
  using L = Kv4Layout<D>;
  constexpr int NG = L::kGroups, LW = L::kLaneWords;
  __shared__ WtSmem<D> sm;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tq = lane & 3;
  const int Hkv = a.cache.Hkv, G = a.cache.Hq / Hkv;
  const int chunk = blockIdx.x % chunks, g = blockIdx.x / chunks % Hkv, s = blockIdx.x / chunks / Hkv;
  const Seq seq = load_seq(a, s, G, false);
  const int page0 = chunk * kWtWarps * kWtPages, pages = (seq.len + kPageTokens - 1) / kPageTokens;
  if (page0 >= pages) return;
  const int mine = min(kWtPages, max(0, (pages - page0 - warp + kWtWarps - 1) / kWtWarps));
  for (int i = lane; i < kWtPages * kPageTokens; i += 32) (&sm.acc[warp][0][0])[i] = 0.f;
  const int tiles = (seq.count * G + kRowsPerTile - 1) / kRowsPerTile;
  for (int r0 = 0; r0 < tiles; r0 += kWtTiles) {
    const int n_tiles = min(kWtTiles, tiles - r0);
    __syncthreads();
    for (int i = tid / 128; i < n_tiles; i += kWtWarps * 32 / 128) {
      const int r = r0 + i, t16 = tid % 128;
      load_tile<D, T>(a, seq, g * G, r, G, q_vec, t16, sm.q[i], sm.sum[i], sm.back[i], sm.seen[i]);
      if (t16 % 16 == 0) {
        const int row = r * kRowsPerTile + t16 / 16, token = row / G;
        const bool real = token < seq.count;
        // a row without a sum (all its keys are absent, or the call was too large) gives no weight: exp(x - infinity)
        const float lse = real ? a.lse[size_t(seq.first + token) * a.cache.Hq + g * G + row % G] * 1.4426950408889634f : 0.f;
        sm.lse[i][t16 / 16] = lse == -INFINITY ? INFINITY : lse;
        if (!real) sm.seen[i][t16 / 16] = 0;
      }
    }
    __syncthreads();
    for (int k = 0; k < mine; ++k) {
      const int page = page0 + warp + k * kWtWarps;
      const int64_t id = a.table[s * a.table_stride + page];
      if (id < 0 || uint64_t(id) >= a.cache.pages) continue;
      const uint8_t* blk = a.cache.block(uint64_t(id), g);
      alignas(16) uint32_t w0[LW], w1[LW], km[2][NG];
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
      load_words<NG>(km[0], blk + L::k_meta(gr, 0));
      load_words<NG>(km[1], blk + L::k_meta(gr + 8, 0));
      uint32_t m0 = km[0][0], m1 = km[1][0];  // the pair of group tq % NG
#pragma unroll
      for (int i = 1; i < NG; ++i)
        if (tq % NG == i) m0 = km[0][i], m1 = km[1][i];
      float sum[2] = {0.f, 0.f};
      for (int i = 0; i < n_tiles; ++i) {
        const int seen0 = sm.seen[i][2 * tq], seen1 = sm.seen[i][2 * tq + 1];
        float acc[NG][4], part[4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint4 q[NG];
#pragma unroll
          for (int e = 0; e < NG; ++e) q[e] = *reinterpret_cast<const uint4*>(sm.q[i][2 * e + j][lane]);
#pragma unroll
          for (int e = 0; e < NG; ++e) {
            const uint32_t x = w0[2 * e + j], y = w1[2 * e + j];
            if (j == 0) mma_f16_first(acc[e], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, q[e].x, q[e].y);
            else mma_f16(acc[e], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, q[e].x, q[e].y);
          }
#pragma unroll
          for (int e = 0; e < NG; ++e) {
            const uint32_t x = w0[2 * e + j] >> 8, y = w1[2 * e + j] >> 8;
            mma_f16(acc[e], x & 0x000F000Fu, y & 0x000F000Fu, x & 0x00F000F0u, y & 0x00F000F0u, q[e].z, q[e].w);
          }
        }
        mma_bf16_first(part, m0, m1, m0, m1, sm.sum[i][0][gr][tq], sm.sum[i][1][gr][tq]);
        mma_bf16(part, m0, m1, m0, m1, sm.sum[i][2][gr][tq], 0u);
        const float f0 = sm.back[i][2 * tq], f1 = sm.back[i][2 * tq + 1], l0 = sm.lse[i][2 * tq], l1 = sm.lse[i][2 * tq + 1];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x0 = kv4_scale(km[c][0]) * acc[0][2 * c], x1 = kv4_scale(km[c][0]) * acc[0][2 * c + 1];
#pragma unroll
          for (int e = 1; e < NG; ++e) {
            x0 = fmaf(kv4_scale(km[c][e]), acc[e][2 * c], x0);
            x1 = fmaf(kv4_scale(km[c][e]), acc[e][2 * c + 1], x1);
          }
          const int key = page * kPageTokens + gr + 8 * c;
          const float p0 = exp2_fast(fmaf(x0, f0, part[2 * c]) - l0), p1 = exp2_fast(fmaf(x1, f1, part[2 * c + 1]) - l1);
          sum[c] += (key < seen0 ? p0 : 0.f) + (key < seen1 ? p1 : 0.f);
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], 1);
        sum[c] += __shfl_xor_sync(0xffffffffu, sum[c], 2);
        if (tq == 0) sm.acc[warp][k][gr + 8 * c] += sum[c];
      }
    }
  }
  __syncwarp();
  const int from = a.weights_in_rows ? a.weights_in_rows[s] : s, to = a.weights_out_rows ? a.weights_out_rows[s] : s;
  const float* in = a.weights_in && from >= 0 ? a.weights_in + (size_t(from) * Hkv + g) * a.weights_stride : nullptr;
  float* out = a.weights_out + (size_t(to) * Hkv + g) * a.weights_stride;
  for (int i = lane; i < mine * kPageTokens; i += 32) {
    const int key = (page0 + warp + i / kPageTokens * kWtWarps) * kPageTokens + i % kPageTokens;
    if (key >= seq.len) continue;
    const float old = in && key < seq.len - seq.count ? in[key] : 0.f;
    out[key] = old + sm.acc[warp][i / kPageTokens][i % kPageTokens];
  }
}

size_t decode_workspace(int Hq, int Hkv, int D, size_t n_seq, size_t tokens, int sm_count) {
  return align16(unit_entries(tokens, n_seq, Hq / Hkv, Hkv) * 8) +
         size_t(sm_count) * kCtasPerSm * kWarps * 2 * kRowsPerTile * (D + 2) * 4;
}

// Rows of a sequence up to which it runs here when neither lse nor weights are
// asked for: four tiles, for each of which this kernel reads the pages again. From
// five on the 128-row tiles of kv4_chunk_kernel are faster: 64 sequences of 4096
// keys take 129 us here with 32 rows and 134 there, 158 and 137 with 40 (2 KV heads
// of 256), 155 and 184, 191 and 186 (4 of 128). Only bf16 rows go there: its fp16
// operands (keys, values, weights) leave 3.5e-4 of error, nothing beside bf16's own
// rounding (1.7e-3) and twice fp16's (2.1e-4). That precision has its price: 2048
// fp16 tokens behind 14336 keys take 6.3 ms here, bf16 ones 0.75 ms there (256
// behind 3840: 262 and 73 us).
constexpr int kChunkRows = 32;

bool uses_chunks(const Kv4AttentionArgs& a) {
  return (a.type == kKv4BF16 || a.coarse) && !a.lse && !a.weights_out && int64_t(a.max_count) * (a.cache.Hq / a.cache.Hkv) > kChunkRows;
}
// Tiles of the longest sequence that runs here.
int most_tiles(const Kv4AttentionArgs& a) {
  const int64_t rows = int64_t(a.max_count) * (a.cache.Hq / a.cache.Hkv);
  return int((std::min(rows, uses_chunks(a) ? int64_t(kChunkRows) : rows) + kRowsPerTile - 1) / kRowsPerTile);
}
// CTAs per (sequence, KV head) of the weights kernel.
int64_t weight_chunks(const Kv4AttentionArgs& a) { return (a.table_stride + kWtWarps * kWtPages - 1) / (kWtWarps * kWtPages); }

template <int D, class T>
void attend(const Kv4AttentionArgs& a, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  once_per_device(configured, [] {
    QWEN_CUDA(cudaFuncSetAttribute(kv4_decode_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(Smem<D>))));
  });
  Kv4AttentionArgs b = a;
  const int G = a.cache.Hq / a.cache.Hkv, ctas = a.sm_count * kCtasPerSm;
  const bool chunks = uses_chunks(a);
  b.row_limit = chunks ? kChunkRows : INT_MAX;
  const int tiles = most_tiles(a);
  const bool q_vec = reinterpret_cast<uintptr_t>(a.q.data) % 16 == 0 && a.q.token_stride % 8 == 0 && a.q.head_stride % 8 == 0;
  const bool gate_vec = reinterpret_cast<uintptr_t>(a.gate.data) % 16 == 0 && a.gate.token_stride % 4 == 0 && a.gate.head_stride % 4 == 0;
  const bool vec = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_token_stride % 8 == 0 && a.out_head_stride % 8 == 0;
  if (a.weights_out && !a.lse)
    b.lse = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + a.workspace_bytes / 16 * 16 -
                                     align16(size_t(a.tokens) * a.cache.Hq * 4));  // the workspace's end
  launch_pdl(kv4_decode_kernel<D, T>, ctas, kThreads, sizeof(Smem<D>), s, b, q_vec, gate_vec, vec);
  launch_pdl(kv4_merge_kernel<D, T>, dim3(unsigned(a.n_seq * a.cache.Hkv * tiles), std::min(int64_t(kRowsPerTile), int64_t(a.max_count) * G)),
             kMergeThreads, 0, s, b, ctas * kWarps, tiles);
  g_kernel_launches.fetch_add(2, std::memory_order_relaxed);
  if (chunks) launch_kv4_chunk(b, static_cast<uint8_t*>(a.workspace) + decode_workspace(a.cache.Hq, a.cache.Hkv, D, a.n_seq, a.tokens, a.sm_count), s);
  if (a.weights_out) {
    const int64_t pieces = weight_chunks(a);
    launch_pdl(kv4_weights_kernel<D, T>, unsigned(pieces * a.n_seq * a.cache.Hkv), kWtWarps * 32, 0, s, b, int(pieces), q_vec);
    g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
  }
}

}  // namespace

size_t kv4_workspace_bytes(int Hq, int Hkv, int D, size_t n_seq, size_t tokens, int sm_count) {
  return decode_workspace(Hq, Hkv, D, n_seq, tokens, sm_count) + kv4_chunk_workspace_bytes(Hq, Hkv, D, n_seq, tokens, sm_count) +
         align16(tokens * size_t(Hq) * 4);
}

void check_kv4_attention(const Kv4AttentionArgs& a) {
  // places of all units (the last pair of an odd table counts whole), and the merge's grid
  if (tiles_at_most(a, most_tiles(a), kRowsPerTile) * a.cache.Hkv >= kPlacesMax / (a.table_stride / 2 + 1 + kUnitPairs) ||
      int64_t(a.n_seq) * a.cache.Hkv * most_tiles(a) > INT32_MAX)
    throw std::invalid_argument("kv4 attention: kv_heads x query tiles x pages beyond 2^31; split the call");
  if (uses_chunks(a)) check_kv4_chunk(a);
  if (a.weights_out && weight_chunks(a) * a.n_seq * a.cache.Hkv > INT32_MAX)
    throw std::invalid_argument("kv4 attention: n_seq x kv_heads x pages beyond 2^31; split the call");
}

void launch_kv4_attention(const Kv4AttentionArgs& a, cudaStream_t s) {
  if (a.tokens <= 0 || a.n_seq <= 0) return;
  check_kv4_attention(a);
  const bool half = a.type == kKv4F16;
  if (a.cache.D == 64) half ? attend<64, __half>(a, s) : attend<64, __nv_bfloat16>(a, s);
  else if (a.cache.D == 128) half ? attend<128, __half>(a, s) : attend<128, __nv_bfloat16>(a, s);
  else half ? attend<256, __half>(a, s) : attend<256, __nv_bfloat16>(a, s);
}

}  // namespace qwen
