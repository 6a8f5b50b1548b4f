// 4-bit paged KV cache: append (q / k RMSNorm, partial RoPE, quantisation and
// the write into the pages in one pass), read back, and eviction by accumulated
// attention weight. The attention over the pages is in kv4_attention.cu.
#include <algorithm>
#include <atomic>

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

// Quantises a warp's row (lane l holds dims l E .. l E + E - 1, in 64 bits) and
// writes nibbles and pairs of token `tok` of `block`. A group with a value that
// is not finite gets a NaN bias: every value of it then reads back as NaN.
// The step is divided out, not multiplied by a reciprocal: inputs of few bits
// lie exactly between two nibbles often enough for the difference to show.
template <int D, bool kKey>
__device__ __forceinline__ void quantise_store(const double (&x)[D / 32], uint8_t* block, int tok, int lane) {
  using L = Kv4Layout<D>;
  constexpr int E = D / 32, kLanes = 64 / E;  // lanes of a group
  bool fine = true;
  double lo = x[0], hi = x[0];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    fine = fine && isfinite(x[e]);
    lo = fmin(lo, x[e]);
    hi = fmax(hi, x[e]);
  }
  const uint32_t group_lanes = (kLanes == 32 ? 0xffffffffu : ((1u << kLanes) - 1u) << (lane & ~(kLanes - 1)));
  fine = (__ballot_sync(0xffffffffu, fine) & group_lanes) == group_lanes;
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) {
    lo = fmin(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmax(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  __nv_bfloat16 scale = __float2bfloat16_rn(float((hi - lo) / 15.0)), bias = __float2bfloat16_rn(float(lo));
  if (!fine) {
    scale = __ushort_as_bfloat16(0);
    bias = __ushort_as_bfloat16(0x7FC0);
  }
  const double s = double(__bfloat162float(scale)), b = double(__bfloat162float(bias));
  uint32_t word = 0;
  const int e0 = lane * E % 8;  // the lane's first dim inside its word
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int n = fine && s > 0 ? int(fmin(fmax(rint((x[e] - b) / s), 0.0), 15.0)) : 0;
    const int place = kKey ? kv4_k_nibble(e0 + e) : e0 + e;
    word |= uint32_t(n) << (4 * place);
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

// One warp per head vector of token blockIdx.x; lane l owns D/32 contiguous
// dims. Queries are normalised and rotated in 32 bits (the angle in 64). Keys go
// through 64 bits up to the nibble: a key that lands next to the border between
// two nibbles is then decided by its value, not by the order of a sum, so the
// same tokens give the same cache whatever the batch around them.
template <int D, class T, class Q>
__global__ void __launch_bounds__(1024) kv4_append_kernel(Kv4AppendArgs a, bool vec) {
  pdl_trigger();
  pdl_wait();
  constexpr int E = D / 32;
  __shared__ double rot[2][D / 2];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
  const int half = a.rope / 2, Hq = a.cache.Hq, Hkv = a.cache.Hkv;
  if (half > 0) {
    const double pos = a.positions[t];
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
      double sn, cs;
      sincos(pos * pow(a.theta, -2.0 * j / a.rope), &sn, &cs);
      rot[0][j] = cs;
      rot[1][j] = sn;
    }
  }
  __syncthreads();
  const int n_q = a.q.data ? Hq : 0, n_kv = a.k.data ? Hkv : 0;
  const int64_t slot = n_kv ? a.slots[t] : -1;
  const bool in_pool = slot < 0 || uint64_t(slot) / kPageTokens < a.cache.pages;
  if (!in_pool && threadIdx.x == 0) kv4_flag(a.cache.status, kErrBounds);
  const int tok = int(uint64_t(slot) % kPageTokens);
  for (int v = warp; v < n_q + 2 * n_kv; v += nw) {
    if (v < n_q) {
      const T* src = static_cast<const T*>(a.q.data) + t * a.q.token_stride + v * a.q.head_stride;
      float val[E];
      load_parts<T, E>(src + lane * E, a.splits, a.split_stride, vec, val);
      if (a.q_norm) {
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss += val[e] * val[e];
        const float inv = rsqrtf(warp_sum(ss) / D + a.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) val[e] = val[e] * inv * a.q_norm[lane * E + e];
      }
      float rotd[E];
#pragma unroll
      for (int e = 0; e < E; ++e) rotd[e] = val[e];
      if (half > 0) {  // dim j < half turns with dim j + half, held by another lane
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int dim = lane * E + e;
          const int other = dim < half ? dim + half : dim < 2 * half ? dim - half : dim;
          float o = 0.f;
#pragma unroll
          for (int f = 0; f < E; ++f) {
            const float got = __shfl_sync(0xffffffffu, val[f], other / E);
            if (other % E == f) o = got;
          }
          if (dim < half) rotd[e] = float(double(val[e]) * rot[0][dim] - double(o) * rot[1][dim]);
          else if (dim < 2 * half) rotd[e] = float(double(o) * rot[1][dim - half] + double(val[e]) * rot[0][dim - half]);
        }
      }
      store_row<Q, E>(static_cast<Q*>(a.q_out) + (size_t(t) * Hq + v) * D + lane * E, rotd);
      if (a.gate) {
        float g[E];
        load_parts<float, E>(a.gate + t * a.q.token_stride + v * a.q.head_stride + lane * E, a.splits, a.split_stride,
                             vec, g);
        store_row<float, E>(a.gate_out + (size_t(t) * Hq + v) * D + lane * E, g);
      }
      continue;
    }
    if (slot < 0 || !in_pool) continue;
    const bool key = v < n_q + n_kv;
    const int g = v - n_q - (key ? 0 : n_kv);
    const Kv4Rows& r = key ? a.k : a.v;
    float val[E];
    load_parts<T, E>(static_cast<const T*>(r.data) + t * r.token_stride + g * r.head_stride + lane * E, a.splits,
                     a.split_stride, vec, val);
    uint8_t* block = a.cache.block(uint64_t(slot) / kPageTokens, g);
    double x[E];
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = val[e];
    if (!key) {
      quantise_store<D, false>(x, block, tok, lane);
      continue;
    }
    if (a.k_norm) {
      double ss = 0.0;
#pragma unroll
      for (int e = 0; e < E; ++e) ss += x[e] * x[e];
      const double inv = 1.0 / sqrt(warp_sum_d(ss) / D + double(a.eps));
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = x[e] * inv * double(a.k_norm[lane * E + e]);
    }
    if (half > 0) {
      double y[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int dim = lane * E + e;
        const int other = dim < half ? dim + half : dim < 2 * half ? dim - half : dim;
        double o = 0.0;
#pragma unroll
        for (int f = 0; f < E; ++f) {
          const double got = __shfl_sync(0xffffffffu, x[f], other / E);
          if (other % E == f) o = got;
        }
        y[e] = dim < half         ? x[e] * rot[0][dim] - o * rot[1][dim]
               : dim < 2 * half   ? o * rot[1][dim - half] + x[e] * rot[0][dim - half]
                                  : x[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = y[e];
    }
    quantise_store<D, true>(x, block, tok, lane);
  }
}

// One thread per (token, KV head, 8 dims): K and V values of a cached token.
template <int D, class T>
__global__ void __launch_bounds__(256) kv4_read_kernel(Kv4View c, int64_t tokens, const int64_t* __restrict__ slots,
                                                       T* k, T* v) {
  pdl_trigger();
  pdl_wait(slots);
  using L = Kv4Layout<D>;
  const int64_t i = int64_t(blockIdx.x) * blockDim.x + threadIdx.x;
  constexpr int W = D / 8;
  if (i >= tokens * c.Hkv * W) return;
  const int w = int(i % W), h = int(i / W % c.Hkv);
  const int64_t t = i / W / c.Hkv, slot = slots[t];
  float kv[8] = {}, vv[8] = {};
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
      for (int e = 0; e < 8; ++e) {
        // scale * n is exact (8 + 4 bits): one rounding, of the sum
        kv[e] = fmaf(kv4_scale(km), float((kw >> (4 * kv4_k_nibble(e))) & 15u), kv4_bias(km));
        vv[e] = fmaf(kv4_scale(vm), float((vw >> (4 * e)) & 15u), kv4_bias(vm));
      }
    }
  }
  store_row<T, 8>(k + (t * c.Hkv + h) * D + w * 8, kv);
  store_row<T, 8>(v + (t * c.Hkv + h) * D + w * 8, vv);
}

// ------------------------------------------------------------------ eviction --
constexpr int kSelThreads = 1024;

// Block-wide exclusive prefix of a packed pair of counts (two 16-bit halves).
__device__ __forceinline__ uint32_t block_prefix(uint32_t v, uint32_t* warp_sums, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint32_t before = 0, sum = 0;
  for (int w = 0; w < kSelThreads / 32; ++w) {
    const uint32_t s = warp_sums[w];
    if (w < warp) before += s;
    sum += s;
  }
  *total = sum;
  __syncthreads();
  return before + x - v;
}

// One CTA per (sequence, KV head): the keys that stay, ascending. The last
// `recent` always stay; of the others the keep - recent with the largest weight
// (fp32 total order, the lowest index first on ties) are found by a radix
// select of the order's 32-bit keys, a byte per pass, then written in index
// order by prefix sums.
__global__ void __launch_bounds__(kSelThreads) kv4_select_kernel(Kv4EvictArgs a) {
  pdl_trigger();
  pdl_wait();
  __shared__ uint32_t hist[256], warp_sums[32], pick[2];
  const int s = blockIdx.x / a.cache.Hkv, h = blockIdx.x % a.cache.Hkv, tid = threadIdx.x;
  const int64_t most = min(a.src_stride * kPageTokens, a.weights_stride);
  int len = a.kv_lens[s];
  if (len < 0 || len > most) {
    if (tid == 0) kv4_flag(a.cache.status, kErrBounds);
    len = int(min(max(int64_t(len), int64_t(0)), most));
  }
  const float* w = a.weights + (size_t(s) * a.cache.Hkv + h) * a.weights_stride;
  int32_t* kept = a.kept + (size_t(s) * a.cache.Hkv + h) * a.keep;
  float* wo = a.weights_out ? a.weights_out + (size_t(s) * a.cache.Hkv + h) * a.weights_out_stride : nullptr;
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
  uint32_t prefix = 0, mask = 0;  // the threshold's bits so far
  int left = m;                   // how many still to take at or above the prefix's bin
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSelThreads) {
      const uint32_t key = total_key(w[i]);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, bin = 255;
      for (; bin > 0 && above + int(hist[bin]) < left; --bin) above += int(hist[bin]);
      pick[0] = uint32_t(bin);
      pick[1] = uint32_t(above);
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    mask |= 255u << shift;
    left -= int(pick[1]);
    __syncthreads();
  }
  // `left` keys equal to the threshold stay, the lowest indices first
  int done = 0, ties = 0;
  for (int base = 0; base < n; base += kSelThreads) {
    const int i = base + tid;
    const uint32_t key = i < n ? total_key(w[i]) : 0u;
    const bool over = i < n && key > prefix, tie = i < n && key == prefix;
    uint32_t total;
    const uint32_t before = block_prefix(uint32_t(over) | uint32_t(tie) << 16, warp_sums, &total);
    const int tie_rank = ties + int(before >> 16);
    if (over || (tie && tie_rank < left)) {
      const int pos = done + int(before & 0xFFFFu) + min(tie_rank, left);
      kept[pos] = i;
      if (wo) wo[pos] = w[i];
    }
    done += int(total & 0xFFFFu);
    ties += int(total >> 16);
  }
}

// One warp per (sequence, kept key, KV head): its nibbles and pairs move to the
// destination page.
template <int D>
__global__ void __launch_bounds__(256) kv4_move_kernel(Kv4EvictArgs a) {
  pdl_trigger();
  pdl_wait();
  using L = Kv4Layout<D>;
  const int lane = threadIdx.x & 31, Hkv = a.cache.Hkv;
  const int64_t item = int64_t(blockIdx.x) * (blockDim.x / 32) + threadIdx.x / 32;
  if (item >= int64_t(a.n_seq) * Hkv * a.keep) return;
  const int j = int(item % a.keep), h = int(item / a.keep % Hkv), s = int(item / a.keep / Hkv);
  const int old = a.kept[(size_t(s) * Hkv + h) * a.keep + j];
  if (old < 0) return;
  const int64_t from = a.src_table[s * a.src_stride + old / kPageTokens], to = a.dst_table[s * a.dst_stride + j / kPageTokens];
  if (from < 0 || to < 0 || uint64_t(from) >= a.cache.pages || uint64_t(to) >= a.cache.pages) {
    if (lane == 0) kv4_flag(a.cache.status, kErrBounds);
    return;
  }
  const uint8_t* src = a.cache.block(uint64_t(from), h);
  uint8_t* dst = a.cache.block(uint64_t(to), h);
  const int o = old % kPageTokens, p = j % kPageTokens;
  for (int i = lane; i < D / 4 + 2 * L::kGroups; i += 32) {
    const int w = i % (D / 8), g = i - D / 4;
    const int at = i < D / 8 ? L::k_word(o, w) : i < D / 4 ? L::v_word(o, w) : g < L::kGroups ? L::k_meta(o, g) : L::v_meta(o, g - L::kGroups);
    const int put = i < D / 8 ? L::k_word(p, w) : i < D / 4 ? L::v_word(p, w) : g < L::kGroups ? L::k_meta(p, g) : L::v_meta(p, g - L::kGroups);
    *reinterpret_cast<uint32_t*>(dst + put) = *reinterpret_cast<const uint32_t*>(src + at);
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
  const int warps = (a.q.data ? a.cache.Hq : 0) + (a.k.data ? 2 * a.cache.Hkv : 0);
  launch_pdl(kv4_append_kernel<D, T, Q>, a.tokens, 32 * std::min(32, warps), 0, s, a, vec);
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

template <int D>
void read(const Kv4View& c, int64_t tokens, const int64_t* slots, uint32_t type, void* k, void* v, cudaStream_t s) {
  const int64_t n = tokens * c.Hkv * (D / 8);
  const dim3 grid(unsigned((n + 255) / 256));
  if (type == kKv4F32)
    launch_pdl(kv4_read_kernel<D, float>, grid, 256, 0, s, c, tokens, slots, static_cast<float*>(k), static_cast<float*>(v));
  else if (type == kKv4F16)
    launch_pdl(kv4_read_kernel<D, __half>, grid, 256, 0, s, c, tokens, slots, static_cast<__half*>(k), static_cast<__half*>(v));
  else
    launch_pdl(kv4_read_kernel<D, __nv_bfloat16>, grid, 256, 0, s, c, tokens, slots, static_cast<__nv_bfloat16*>(k),
               static_cast<__nv_bfloat16*>(v));
  count_launch();
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
  if (c.D == 64) read<64>(c, tokens, slots, type, k, v, s);
  else if (c.D == 128) read<128>(c, tokens, slots, type, k, v, s);
  else read<256>(c, tokens, slots, type, k, v, s);
}

void launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t s) {
  if (a.n_seq <= 0) return;
  launch_pdl(kv4_select_kernel, a.n_seq * a.cache.Hkv, kSelThreads, 0, s, a);
  count_launch();
  const int64_t items = int64_t(a.n_seq) * a.cache.Hkv * a.keep;
  const dim3 grid(unsigned((items + 7) / 8));
  if (a.cache.D == 64) launch_pdl(kv4_move_kernel<64>, grid, 256, 0, s, a);
  else if (a.cache.D == 128) launch_pdl(kv4_move_kernel<128>, grid, 256, 0, s, a);
  else launch_pdl(kv4_move_kernel<256>, grid, 256, 0, s, a);
  count_launch();
}

}  // namespace qwen
