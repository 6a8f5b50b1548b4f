// 4-bit paged KV cache: append (q / k RMSNorm, partial RoPE, quantisation and
// the write into the pages in one pass), read back, and eviction by accumulated
// attention weight. The attention over the pages is in kv4_attention.cu.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "kernels.h"
#include "kv4.h"

namespace qwen {

extern std::atomic<uint64_t> g_kernel_launches;

namespace {

// E contiguous elements at p as floats; vec: p is aligned to E elements (16 bytes at most).
template <class T, int E>
__device__ __forceinline__ void load_row(const T* p, bool vec, float (&out)[E]) {
  constexpr int kBytes = E * int(sizeof(T));
  if (vec) {
    T t[E];
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        reinterpret_cast<uint4*>(t)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(t) = *reinterpret_cast<const uint2*>(p);
    } else {
      *reinterpret_cast<uint32_t*>(t) = *reinterpret_cast<const uint32_t*>(p);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = kv4_to_float(t[e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = kv4_to_float(p[e]);
  }
}

// Sum of the split-K partials of a row piece, in split order (fp32 rows only).
template <class T, int E>
__device__ __forceinline__ void load_parts(const T* p, int splits, size_t stride, bool vec, float (&out)[E]) {
  load_row<T, E>(p, vec, out);
  for (int sp = 1; sp < splits; ++sp) {
    float part[E];
    load_row<T, E>(p + sp * stride, vec, part);
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] += part[e];
  }
}

template <class T, int E>
__device__ __forceinline__ void store_row(T* p, const float (&v)[E]) {
  alignas(16) T t[E];
#pragma unroll
  for (int e = 0; e < E; ++e) t[e] = kv4_from_float<T>(v[e]);
  constexpr int kBytes = E * int(sizeof(T));
  if constexpr (kBytes >= 16) {
#pragma unroll
    for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(t)[i];
  } else if constexpr (kBytes == 8) {
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(t);
  } else {
    *reinterpret_cast<uint32_t*>(p) = *reinterpret_cast<const uint32_t*>(t);
  }
}

__device__ __forceinline__ double warp_sum_d(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ float lower(float a, float b) { return fminf(a, b); }
__device__ __forceinline__ float higher(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ double lower(double a, double b) { return a < b ? a : b; }
__device__ __forceinline__ double higher(double a, double b) { return a > b ? a : b; }

// Quantises a warp's row (lane l holds dims l E .. l E + E - 1; V: 32 or 64 bits)
// and writes nibbles and pairs of token `tok` of `block`. A group with a value
// that is not finite, or whose minimum rounds to an infinity in bf16, gets a NaN
// bias: every value of it then reads back as NaN.
// A nibble is rint((x - bias) / step), by its exact value: found in 32 bits when
// that is safely away from the border between two nibbles, and by the division in
// 64 bits when not (bf16 inputs lie exactly on the border often enough to show).
template <int D, bool kKey, class V>
__device__ __forceinline__ void quantise_store(const V (&x)[D / 32], uint8_t* block, int tok, int lane) {
  using L = Kv4Layout<D>;
  constexpr int E = D / 32, kLanes = 64 / E;  // lanes of a group
  bool fine = true;
  V lo = x[0], hi = x[0];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    fine = fine && isfinite(x[e]);
    lo = lower(lo, x[e]);
    hi = higher(hi, x[e]);
  }
  const uint32_t group_lanes = (kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u) << (lane & ~(kLanes - 1)));
  fine = (__ballot_sync(0xffffffffu, fine) & group_lanes) == group_lanes;
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    lo = lower(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = higher(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  __nv_bfloat16 scale = __float2bfloat16_rn(float((double(hi) - double(lo)) / 15.0)), bias = __float2bfloat16_rn(float(lo));
  fine = fine && (__bfloat16_as_ushort(bias) & 0x7F80) != 0x7F80;  // a minimum that bf16 has no number for
  if (!fine) {
    scale = __ushort_as_bfloat16(0);
    bias = __ushort_as_bfloat16(0x7FC0);
  }
  const float s = __bfloat162float(scale), b = __bfloat162float(bias);
  uint32_t word = 0;
  const int e0 = lane * E % 8;  // the lane's first dim inside its word
  if (fine && s > 0.f) {
    const float inv = 1.f / s;
    // (x - b) / s in 32 bits: x, the difference, the reciprocal and the product are
    // each off by 2^-24 of themselves, and the terms are at most |x| + |b| and 16
    const float margin = 0x1p-22f * (fmaxf(fabsf(float(lo)), fabsf(float(hi))) + fabsf(b)) * inv + 0x1p-18f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float q = (float(x[e]) - b) * inv;
      float n = rintf(q);
      if (!(fabsf(fabsf(q - n) - 0.5f) > margin)) n = float(rint((double(x[e]) - double(b)) / double(s)));
      const int place = kKey ? kv4_k_nibble(e0 + e) : e0 + e;
      word |= uint32_t(int(fminf(fmaxf(n, 0.f), 15.f))) << (4 * place);
    }
  }
#pragma unroll
  for (int o = 8 / E / 2; o > 0; o >>= 1) word |= __shfl_xor_sync(0xffffffffu, word, o);
  if (lane % (8 / E) == 0) {
    const int w = lane * E / 8;
    *reinterpret_cast<uint32_t*>(block + (kKey ? L::k_word(tok, w) : L::v_word(tok, w))) = word;
  }
  if (lane % kLanes == 0) {
    const uint32_t pair = uint32_t(__bfloat16_as_ushort(scale)) | uint32_t(__bfloat16_as_ushort(bias)) << 16;
    const int group = lane / kLanes;
    *reinterpret_cast<uint32_t*>(block + (kKey ? L::k_meta(tok, group) : L::v_meta(tok, group))) = pair;
  }
}

// Partner of a lane's elements in the rotation: dim j < half turns with dim
// j + half. Lane l holds dims l E .. l E + E - 1, so when E divides half the
// partners lie in one other lane, at the same places.
template <int E, class V>
__device__ __forceinline__ void rotation_partner(const V (&x)[E], V (&o)[E], int lane, int half) {
  if (half % E == 0) {
    const int other = lane * E < half ? lane + half / E : lane * E < 2 * half ? lane - half / E : lane;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = __shfl_sync(0xffffffffu, x[e], other);
  } else {
    // kept rolled and in local memory: no geometry in use comes here, and unrolled it would cost the others registers
    V from[E], to[E];
#pragma unroll
    for (int e = 0; e < E; ++e) from[e] = x[e];
#pragma unroll 1
    for (int e = 0; e < E; ++e) {
      const int dim = lane * E + e, other = dim < half ? dim + half : dim < 2 * half ? dim - half : dim;
#pragma unroll 1
      for (int f = 0; f < E; ++f) {
        const V got = __shfl_sync(0xffffffffu, from[f], other / E);
        if (other % E == f) to[e] = got;
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = to[e];
  }
}

// theta^(-2 j / rope), made on the host: a power in 64 bits costs a thread some
// hundred dependent instructions, as long as the rest of a decode step's append.
struct Frequencies {
  double f[128];
};

// A CTA takes `batch` tokens: first all their rotations (sines and cosines in 64
// bits, one per thread), then rows, a warp per value or key row and per kQ query
// rows of a token; lane l owns D/32 contiguous dims of a row. Queries are
// normalised and rotated in 32 bits (the angle, its sine and cosine in 64). Keys go
// through 64 bits up to the nibble: a key that lands next to the border between two
// nibbles is then decided by its value, not by the order of a sum, so the same
// tokens give the same cache whatever the batch around them.
// 2168 fp32 tokens of 16 + 2 + 2 rows of 256: 28 us (74 MB, 2.6 TB/s; all keys in
// 64 bits with a division each took 106). Neither bytes nor one pipe bounds it: issue
// slots 48 %, warps 40 %, waits for shuffles and 64-bit results first (3.9 cycles an
// instruction), for memory next (2.7). 64 bf16 tokens: 6.5 us (11), the latency of
// one sine and one row.
constexpr int kMaxBatch = 8;
// kFused: fp32 rows as split-K partials, and a gate beside every query row
// (the session's projection).
template <int D, class T, class Q, int kQ, bool kFused>
__global__ void __launch_bounds__(kQ == 1 ? 640 : 256, kQ == 1 ? 1 : 4) kv4_append_kernel(Kv4AppendArgs a, const __grid_constant__ Frequencies freq, int batch, bool vec) {
  pdl_trigger();
  pdl_wait();
  constexpr int E = D / 32;
  extern __shared__ __align__(16) double2 rot[];  // [batch][half]: cosine, sine; the same in 32 bits behind them
  const int t0 = blockIdx.x * batch, n_tok = min(batch, a.tokens - t0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const int half = a.rope / 2, Hq = a.cache.Hq, Hkv = a.cache.Hkv;
  for (int i = threadIdx.x; i < n_tok * half; i += blockDim.x) {
    double sn, cs;
    sincos(double(a.positions[t0 + i / half]) * freq.f[i % half], &sn, &cs);
    rot[i] = make_double2(cs, sn);
    reinterpret_cast<float2*>(rot + batch * half)[i] = make_float2(float(cs), float(sn));
  }
  const int n_kv = a.k.data ? 2 * Hkv : 0, n_q = a.q.data ? (Hq + kQ - 1) / kQ : 0;
  const int kv_tasks = n_tok * n_kv, tasks = kv_tasks + n_tok * n_q;
  if (half > 0) __syncthreads();
  for (int i = warp; i < tasks; i += nw) {
    if (i < kv_tasks) {
      const int t = t0 + i / n_kv, v = i % n_kv, g = v >= Hkv ? v - Hkv : v;
      const bool key = v < Hkv;
      const int64_t slot = a.slots[t];
      if (slot < 0) continue;
      if (uint64_t(slot) / kPageTokens >= a.cache.pages) {
        if (lane == 0) kv4_flag(a.cache.status, kErrBounds);
        continue;
      }
      const int tok = int(uint64_t(slot) % kPageTokens);
      const Kv4Rows& r = key ? a.k : a.v;
      float val[E];
      load_parts<T, E>(static_cast<const T*>(r.data) + t * r.token_stride + g * r.head_stride + lane * E, kFused ? a.splits : 1,
                       a.split_stride, vec, val);
      uint8_t* block = a.cache.block(uint64_t(slot) / kPageTokens, g);
      if (!key) {
        quantise_store<D, false>(val, block, tok, lane);
        continue;
      }
      double x[E];
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = val[e];
      if (a.k_norm) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) ss += x[e] * x[e];
        const double inv = 1.0 / sqrt(warp_sum_d(ss) / D + double(a.eps));
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = x[e] * inv * double(a.k_norm[lane * E + e]);
      }
      if (half > 0) {
        const double2* cs = rot + (t - t0) * half;
        double o[E];
        rotation_partner<E>(x, o, lane, half);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int dim = lane * E + e;
          if (dim < 2 * half) {
            const double2 r = cs[dim < half ? dim : dim - half];
            x[e] = x[e] * r.x + (dim < half ? -o[e] : o[e]) * r.y;
          }
        }
      }
      quantise_store<D, true>(x, block, tok, lane);
      continue;
    }
    const int t = t0 + (i - kv_tasks) / n_q, h0 = (i - kv_tasks) % n_q * kQ;
    const T* src = static_cast<const T*>(a.q.data) + t * a.q.token_stride + h0 * a.q.head_stride + lane * E;
    float val[kQ][E];
#pragma unroll
    for (int k = 0; k < kQ; ++k)
      if (h0 + k < Hq) load_parts<T, E>(src + k * a.q.head_stride, kFused ? a.splits : 1, a.split_stride, vec, val[k]);
    float gate[kQ][E];
    if (kFused) {
#pragma unroll
      for (int k = 0; k < kQ; ++k)
        if (h0 + k < Hq)
          load_parts<float, E>(a.gate + t * a.q.token_stride + (h0 + k) * a.q.head_stride + lane * E, a.splits, a.split_stride, vec, gate[k]);
    }
#pragma unroll
    for (int k = 0; k < kQ; ++k) {
      if (h0 + k >= Hq) break;
      if (a.q_norm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss += val[k][e] * val[k][e];
        const float inv = rsqrtf(warp_sum(ss) / D + a.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) val[k][e] = val[k][e] * inv * a.q_norm[lane * E + e];
      }
      if (half > 0) {
        const float2* cs = reinterpret_cast<const float2*>(rot + batch * half) + (t - t0) * half;
        float o[E];
        rotation_partner<E>(val[k], o, lane, half);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int dim = lane * E + e;
          if (dim < 2 * half) {
            const float2 r = cs[dim < half ? dim : dim - half];
            val[k][e] = fmaf(val[k][e], r.x, (dim < half ? -o[e] : o[e]) * r.y);
          }
        }
      }
      const size_t row = (size_t(t) * Hq + h0 + k) * D + lane * E;
      store_row<Q, E>(static_cast<Q*>(a.q_out) + row, val[k]);
      if (kFused) store_row<float, E>(a.gate_out + row, gate[k]);
    }
  }
}

// One thread per 16 bytes of K and of V values of a cached token, so that a warp's
// stores are contiguous. 121925 tokens of 2 x 256 in fp32 (570 MB): 121 us,
// 4.7 TB/s (142 us with four items per thread); fp16 or bf16 (320 MB): 72 us. Issue
// slots 62 %, ALU 58 %: the wait for slot, then nibbles, and the unpacking around it.
template <int D, class T, class Index>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4View c, Index tokens, const int64_t* __restrict__ slots,
                                                       T* k, T* v) {
  pdl_trigger();
  pdl_wait(slots);
  using L = Kv4Layout<D>;
  constexpr int kDims = 16 / int(sizeof(T)), W = D / kDims;
  const Index i = Index(blockIdx.x) * 256 + threadIdx.x;
  if (i >= tokens * Index(c.Hkv) * W) return;
  const int dim = int(i % W) * kDims, w = dim / 8, h = int(i / W % Index(c.Hkv));
  const Index t = i / W / Index(c.Hkv);
  const int64_t slot = slots[t];
  float kv[kDims] = {}, vv[kDims] = {};
  if (slot >= 0) {
    if (uint64_t(slot) / kPageTokens >= c.pages) {
      kv4_flag(c.status, kErrBounds);
    } else {
      const uint8_t* block = c.block(uint64_t(slot) / kPageTokens, h);
      const int tok = int(slot % kPageTokens);
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(block + L::k_word(tok, w));
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(block + L::v_word(tok, w));
      const uint32_t km = *reinterpret_cast<const uint32_t*>(block + L::k_meta(tok, w / 8));
      const uint32_t vm = *reinterpret_cast<const uint32_t*>(block + L::v_meta(tok, w / 8));
#pragma unroll
      for (int e = 0; e < kDims; ++e) {
        // scale * n is exact (8 + 4 bits): one rounding, of the sum
        kv[e] = fmaf(kv4_scale(km), float((kw >> (4 * kv4_k_nibble(dim % 8 + e))) & 15u), kv4_bias(km));
        vv[e] = fmaf(kv4_scale(vm), float((vw >> (4 * (dim % 8 + e))) & 15u), kv4_bias(vm));
      }
    }
  }
  const size_t at = (size_t(t) * c.Hkv + h) * D + dim;
  store_row<T, kDims>(k + at, kv);
  store_row<T, kDims>(v + at, vv);
}

// ------------------------------------------------------------------ eviction --
constexpr int kSelThreads = 1024;
constexpr int kSelKeys = 32;  // keys a thread keeps in registers

// One CTA per (sequence, KV head): the keys that stay, ascending. The last
// `recent` always stay; of the others the keep - recent with the largest weight
// (fp32 total order, the lowest index first on ties). The smallest weight that
// stays is found bit by bit, counting the keys that reach each candidate: 32 passes
// over registers, with one barrier each, whatever the weights' distribution (a
// histogram's bins collide on the few exponents that attention weights have).
// A thread holds consecutive keys, so one prefix sum then gives every kept key its
// place; keys beyond the first 32 of a thread (more than 32768 in all) are read
// again in every pass. 64 rows of up to 32768 keys: 39 us (histogram: 66), bound by
// the compares that the longest row's one SM issues (issue slots 68 %, ALU 63 % while
// it runs; the others are long done); 16 rows of up to 500: 9.5 us (26), the 32
// barriers.
template <int kKeys>
__device__ __forceinline__ void select_keys(const float* w, int32_t* kept, float* wo, int n, int m, int per, int (*counts)[kSelThreads / 32]);

__global__ void __launch_bounds__(kSelThreads) kv4_select_kernel(Kv4EvictArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ int counts[2][kSelThreads / 32];
  const int s = blockIdx.x / a.cache.Hkv, h = blockIdx.x % a.cache.Hkv, tid = threadIdx.x;
  const int64_t most = min(a.src_stride * kPageTokens, a.weights_stride);
  int len = a.kv_lens[s];
  if (len < 0 || len > most) {
    if (tid == 0) kv4_flag(a.cache.status, kErrBounds);
    len = int(min(max(int64_t(len), int64_t(0)), most));
  }
  const int from = a.weights_rows ? a.weights_rows[s] : s, to = a.weights_out_rows ? a.weights_out_rows[s] : s;
  const float* w = a.weights + (size_t(from) * a.cache.Hkv + h) * a.weights_stride;
  int32_t* kept = a.kept + (size_t(s) * a.cache.Hkv + h) * a.keep;
  float* wo = a.weights_out ? a.weights_out + (size_t(to) * a.cache.Hkv + h) * a.weights_out_stride : nullptr;
  const int n_new = min(len, a.keep);
  if (tid == 0 && h == 0) a.new_lens[s] = n_new;
  for (int j = n_new + tid; j < a.keep; j += kSelThreads) {
    kept[j] = -1;
    if (wo) wo[j] = 0.f;
  }
  if (len <= a.keep) {
    for (int j = tid; j < len; j += kSelThreads) {
      kept[j] = j;
      if (wo) wo[j] = w[j];
    }
    return;
  }
  const int n = len - a.recent, m = a.keep - a.recent;  // m of the first n stay
  for (int j = tid; j < a.recent; j += kSelThreads) {
    kept[m + j] = n + j;
    if (wo) wo[m + j] = w[n + j];
  }
  if (m == 0) return;
  const int per = ((n + kSelThreads - 1) / kSelThreads + 3) & ~3;
  if (per <= 4) select_keys<4>(w, kept, wo, n, m, per, counts);
  else if (per <= 16) select_keys<16>(w, kept, wo, n, m, per, counts);
  else select_keys<kSelKeys>(w, kept, wo, n, m, per, counts);
}

// m of the n keys at w; every thread has `per` of them, kKeys in registers.
template <int kKeys>
__device__ __forceinline__ void select_keys(const float* w, int32_t* kept, float* wo, int n, int m, int per, int (*counts)[kSelThreads / 32]) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // this thread's keys: [first, first + mine); a place without a key holds 0, which no candidate below counts
  const int first = min(int64_t(tid) * per, int64_t(n)), mine = min(per, n - first);
  uint32_t key[kKeys];
  const bool vec = reinterpret_cast<uintptr_t>(w) % 16 == 0;
#pragma unroll
  for (int j = 0; j < kKeys; j += 4) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (vec && j + 4 <= mine) {
      v = *reinterpret_cast<const float4*>(w + first + j);
    } else {
      if (j < mine) v.x = w[first + j];
      if (j + 1 < mine) v.y = w[first + j + 1];
      if (j + 2 < mine) v.z = w[first + j + 2];
      if (j + 3 < mine) v.w = w[first + j + 3];
    }
    key[j] = j < mine ? total_key(v.x) : 0u;
    key[j + 1] = j + 1 < mine ? total_key(v.y) : 0u;
    key[j + 2] = j + 2 < mine ? total_key(v.z) : 0u;
    key[j + 3] = j + 3 < mine ? total_key(v.w) : 0u;
  }
  auto total = [&](int mine_count, int buffer) {
    const int sum = __reduce_add_sync(0xffffffffu, mine_count);
    if (lane == 0) counts[buffer][warp] = sum;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, counts[buffer][lane]);
  };
  uint32_t bound = 0;  // the largest value that at least m keys reach
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t candidate = bound | 1u << bit;
    int c = 0;
#pragma unroll
    for (int j = 0; j < kKeys; ++j) c += key[j] >= candidate;
    for (int j = kKeys; j < mine; ++j) c += total_key(w[first + j]) >= candidate;
    if (total(c, bit & 1) >= m) bound = candidate;
  }
  int over = 0, ties = 0;
#pragma unroll
  for (int j = 0; j < kKeys; ++j) {
    over += j < mine && key[j] > bound;
    ties += j < mine && key[j] == bound;
  }
  for (int j = kKeys; j < mine; ++j) {
    const uint32_t k = total_key(w[first + j]);
    over += k > bound;
    ties += k == bound;
  }
  const int left = m - total(over, 1);  // keys equal to the bound that stay, the lowest indices first
  __syncthreads();
  // exclusive prefix sums of both over the threads
  int x = over, y = ties;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int p = __shfl_up_sync(0xffffffffu, x, o), q = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) {
      x += p;
      y += q;
    }
  }
  if (lane == 31) {
    counts[0][warp] = x;
    counts[1][warp] = y;
  }
  __syncthreads();
  const int px = __reduce_add_sync(0xffffffffu, lane < warp ? counts[0][lane] : 0);
  const int py = __reduce_add_sync(0xffffffffu, lane < warp ? counts[1][lane] : 0);
  int rank = py + y - ties, pos = px + x - over + min(rank, left);
  auto place = [&](int j, uint32_t k) {
    bool stays = k > bound;
    if (k == bound) stays = rank++ < left;
    if (stays) {
      kept[pos] = first + j;
      if (wo) wo[pos] = __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
      ++pos;
    }
  };
#pragma unroll
  for (int j = 0; j < kKeys; ++j)
    if (j < mine) place(j, key[j]);
  for (int j = kKeys; j < mine; ++j) place(j, total_key(w[first + j]));
}

// Kept keys to their new places: 16 bytes (4 or 8 for the pairs of narrow heads) a
// piece, kMovePieces per thread so that their chains of loads (kept index, page
// ids, bytes) run side by side: 64 rows of 4096 keys (76 MB both ways) in 39 us, 53
// with one piece per thread. Sources are scattered 32-byte sectors: 64 MB come from
// memory for the 19 MB of half those rows.
constexpr int kMovePieces = 4;
template <int D>
__global__ void __launch_bounds__(256) kv4_move_kernel(Kv4EvictArgs a, int row_blocks) {
  pdl_trigger();
  pdl_wait();
  using L = Kv4Layout<D>;
  constexpr int kNib = D / 32, kUnits = 2 * kNib + 2;  // of K (or V) nibbles; of a key
  const int Hkv = a.cache.Hkv;
  const int row = blockIdx.x / row_blocks, s = row / Hkv, h = row % Hkv;
  const uint32_t i0 = (blockIdx.x % row_blocks) * (256 * kMovePieces) + threadIdx.x;
  int old[kMovePieces];
  const uint8_t* src[kMovePieces];
  uint8_t* dst[kMovePieces];
#pragma unroll
  for (int k = 0; k < kMovePieces; ++k) {
    const uint32_t j = (i0 + k * 256) / kUnits;
    old[k] = j < uint32_t(a.keep) ? a.kept[size_t(row) * a.keep + j] : -1;
  }
#pragma unroll
  for (int k = 0; k < kMovePieces; ++k) {
    const uint32_t j = (i0 + k * 256) / kUnits;
    if (old[k] < 0) continue;
    const int64_t from = a.src_table[s * a.src_stride + old[k] / kPageTokens], to = a.dst_table[s * a.dst_stride + j / kPageTokens];
    if (from < 0 || to < 0 || uint64_t(from) >= a.cache.pages || uint64_t(to) >= a.cache.pages) {
      kv4_flag(a.cache.status, kErrBounds);
      old[k] = -1;
      continue;
    }
    src[k] = a.cache.block(uint64_t(from), h);
    dst[k] = a.cache.block(uint64_t(to), h);
  }
  uint4 v[kMovePieces];
  int put[kMovePieces];
#pragma unroll
  for (int k = 0; k < kMovePieces; ++k) {
    if (old[k] < 0) continue;
    const uint32_t j = (i0 + k * 256) / kUnits, u = (i0 + k * 256) % kUnits;
    const int o = old[k] % kPageTokens, p = j % kPageTokens;
    if (u < 2 * kNib) {
      constexpr int kRow = L::kChunk * 16;  // bytes of a token's run of K words
      auto at = [&](int tok) {
        const int b = u % kNib * 16;
        return u < kNib ? (b / kRow * kPageTokens + tok) * kRow + b % kRow
                        : L::kV + (b / 32 * kPageTokens + (tok & 1) * 8 + tok / 2) * 32 + b % 32;
      };
      put[k] = at(p);
      v[k] = *reinterpret_cast<const uint4*>(src[k] + at(o));
    } else {
      const int base = u == 2 * kNib ? L::kKMeta : L::kVMeta;
      put[k] = -(base + p * L::kGroups * 4);
      uint32_t pair[L::kGroups];
#pragma unroll
      for (int g = 0; g < L::kGroups; ++g) pair[g] = reinterpret_cast<const uint32_t*>(src[k] + base)[o * L::kGroups + g];
      v[k] = make_uint4(pair[0], pair[L::kGroups > 1 ? 1 : 0], pair[L::kGroups > 2 ? 2 : 0], pair[L::kGroups > 2 ? 3 : 0]);
    }
  }
#pragma unroll
  for (int k = 0; k < kMovePieces; ++k) {
    if (old[k] < 0) continue;
    if (put[k] >= 0) {
      *reinterpret_cast<uint4*>(dst[k] + put[k]) = v[k];
    } else {  // scale / bias pairs of a token: 4 bytes per group
      uint32_t* to = reinterpret_cast<uint32_t*>(dst[k] - put[k]);
      to[0] = v[k].x;
      if (L::kGroups > 1) to[1] = v[k].y;
      if (L::kGroups > 2) to[2] = v[k].z, to[3] = v[k].w;
    }
  }
}

void count_launch() { g_kernel_launches.fetch_add(1, std::memory_order_relaxed); }

template <int D, class T, class Q>
void append(const Kv4AppendArgs& a, cudaStream_t s) {
  constexpr int E = D / 32;
  const size_t align = std::min<size_t>(16, E * sizeof(T));
  auto aligned = [&](const Kv4Rows& r) {
    return !r.data || (reinterpret_cast<uintptr_t>(r.data) % align == 0 && r.token_stride * sizeof(T) % align == 0 &&
                       r.head_stride * sizeof(T) % align == 0);
  };
  const bool vec = aligned(a.q) && aligned(a.k) && aligned(a.v) && a.split_stride * sizeof(T) % align == 0 &&
                   reinterpret_cast<uintptr_t>(a.gate) % align == 0;
  // the table of the last (theta, rope) of this thread
  thread_local Frequencies freq;
  thread_local double theta = 0.0;
  thread_local int rope = 0;
  if (a.rope > 0 && (theta != a.theta || rope != a.rope)) {
    for (int j = 0; j < a.rope / 2; ++j) freq.f[j] = std::pow(a.theta, -2.0 * j / a.rope);
    theta = a.theta;
    rope = a.rope;
  }
  // few tokens: a CTA each and a warp per row; many: tokens share a CTA (their
  // sines are then made side by side) and warps take two query rows, whose loads overlap
  const int batch = std::min(kMaxBatch, (a.tokens + 591) / 592);
  const int grid = (a.tokens + batch - 1) / batch;
  const size_t smem = (sizeof(double2) + sizeof(float2)) * batch * (a.rope / 2);
  const int rows = (a.q.data ? a.cache.Hq : 0) + (a.k.data ? 2 * a.cache.Hkv : 0);
  if constexpr (std::is_same_v<T, float>) {
    if (a.gate || a.splits > 1) {
      if (batch == 1) launch_pdl(kv4_append_kernel<D, T, Q, 1, true>, grid, 32 * std::min(20, rows), smem, s, a, freq, batch, vec);
      else launch_pdl(kv4_append_kernel<D, T, Q, 2, true>, grid, 256, smem, s, a, freq, batch, vec);
      count_launch();
      return;
    }
  }
  if (batch == 1) launch_pdl(kv4_append_kernel<D, T, Q, 1, false>, grid, 32 * std::min(20, rows), smem, s, a, freq, batch, vec);
  else launch_pdl(kv4_append_kernel<D, T, Q, 2, false>, grid, 256, smem, s, a, freq, batch, vec);
  count_launch();
}

template <int D, class T>
void append_out(const Kv4AppendArgs& a, cudaStream_t s) {
  if (a.q_type == kKv4F16) append<D, T, __half>(a, s);
  else if (a.q_type == kKv4BF16) append<D, T, __nv_bfloat16>(a, s);
  else append<D, T, float>(a, s);
}

template <int D>
void append_in(const Kv4AppendArgs& a, cudaStream_t s) {
  if (a.type == kKv4F16) append_out<D, __half>(a, s);
  else if (a.type == kKv4BF16) append_out<D, __nv_bfloat16>(a, s);
  else append_out<D, float>(a, s);
}

template <int D, class T>
void read(const Kv4View& c, int64_t tokens, const int64_t* slots, void* k, void* v, cudaStream_t s) {
  const int64_t n = tokens * c.Hkv * (D * int64_t(sizeof(T)) / 16);
  const dim3 grid(unsigned((n + 255) / 256));
  if (n <= INT32_MAX) launch_pdl(kv4_read_kernel<D, T, uint32_t>, grid, 256, 0, s, c, uint32_t(tokens), slots, static_cast<T*>(k), static_cast<T*>(v));
  else launch_pdl(kv4_read_kernel<D, T, uint64_t>, grid, 256, 0, s, c, uint64_t(tokens), slots, static_cast<T*>(k), static_cast<T*>(v));
  count_launch();
}

template <int D>
void read_out(const Kv4View& c, int64_t tokens, const int64_t* slots, uint32_t type, void* k, void* v, cudaStream_t s) {
  if (type == kKv4F32) read<D, float>(c, tokens, slots, k, v, s);
  else if (type == kKv4F16) read<D, __half>(c, tokens, slots, k, v, s);
  else read<D, __nv_bfloat16>(c, tokens, slots, k, v, s);
}

}  // namespace

void launch_kv4_append(const Kv4AppendArgs& a, cudaStream_t s) {
  if (a.tokens <= 0 || (!a.q.data && !a.k.data)) return;
  if (a.cache.D == 64) append_in<64>(a, s);
  else if (a.cache.D == 128) append_in<128>(a, s);
  else append_in<256>(a, s);
}

void launch_kv4_read(const Kv4View& c, int64_t tokens, const int64_t* slots, uint32_t type, void* k, void* v,
                     cudaStream_t s) {
  if (tokens <= 0) return;
  if (c.D == 64) read_out<64>(c, tokens, slots, type, k, v, s);
  else if (c.D == 128) read_out<128>(c, tokens, slots, type, k, v, s);
  else read_out<256>(c, tokens, slots, type, k, v, s);
}

void launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t s) {
  if (a.n_seq <= 0) return;
  launch_pdl(kv4_select_kernel, a.n_seq * a.cache.Hkv, kSelThreads, 0, s, a);
  count_launch();
  const int row_blocks = int((int64_t(a.keep) * (a.cache.D / 16 + 2) + 256 * kMovePieces - 1) / (256 * kMovePieces));
  const dim3 grid(unsigned(row_blocks) * unsigned(a.n_seq * a.cache.Hkv));
  if (a.cache.D == 64) launch_pdl(kv4_move_kernel<64>, grid, 256, 0, s, a, row_blocks);
  else if (a.cache.D == 128) launch_pdl(kv4_move_kernel<128>, grid, 256, 0, s, a, row_blocks);
  else launch_pdl(kv4_move_kernel<256>, grid, 256, 0, s, a, row_blocks);
  count_launch();
}

}  // namespace qwen
