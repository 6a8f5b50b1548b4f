// Attention over the 4-bit paged KV cache.
#include <algorithm>
#include <atomic>
#include <cfloat>

#include "kernels.h"
#include "kv4.h"

namespace qwen {

extern std::atomic<uint64_t> g_kernel_launches;

namespace {

constexpr int kWarps = 4;

// Length of sequence s, kept within the table and, when weights are written, their rows.
__device__ __forceinline__ int kv4_length(const Kv4AttentionArgs& a, int s) {
  int64_t most = a.table_stride * kPageTokens;
  if (a.weights_out) most = min(most, a.weights_stride);
  const int len = a.kv_lens[s];
  if (len < 0 || len > most) {
    if (threadIdx.x == 0) kv4_flag(a.cache.status, kErrBounds);
    return int(min(max(int64_t(len), int64_t(0)), most));
  }
  return len;
}

// Block of key `pos` of sequence s, null for a page outside the pool.
__device__ __forceinline__ const uint8_t* kv4_page(const Kv4AttentionArgs& a, int s, int pos, int head) {
  const int64_t page = a.table[s * a.table_stride + pos / kPageTokens];
  if (page < 0 || uint64_t(page) >= a.cache.pages) {
    kv4_flag(a.cache.status, kErrBounds);
    return nullptr;
  }
  return a.cache.block(uint64_t(page), head);
}

// Lane's dims lane E .. lane E + E - 1 of K (or V) of one cached token.
template <int D, bool kKey>
__device__ __forceinline__ void load_values(const uint8_t* block, int tok, int lane, float (&x)[D / 32]) {
  using L = Kv4Layout<D>;
  constexpr int E = D / 32;
  const int w = lane * E / 8;
  const uint32_t word = *reinterpret_cast<const uint32_t*>(block + (kKey ? L::k_word(tok, w) : L::v_word(tok, w)));
  const uint32_t pair = *reinterpret_cast<const uint32_t*>(block + (kKey ? L::k_meta(tok, w / 8) : L::v_meta(tok, w / 8)));
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int d = lane * E % 8 + e;
    x[e] = fmaf(kv4_scale(pair), float((word >> (4 * (kKey ? kv4_k_nibble(d) : d))) & 15u), kv4_bias(pair));
  }
}

// One CTA per (query token, query head); a warp per key.
template <int D, class T>
__global__ void __launch_bounds__(kWarps * 32) kv4_attention_kernel(Kv4AttentionArgs a) {
  pdl_trigger();
  pdl_wait();
  constexpr int E = D / 32;
  __shared__ float red[kWarps][2], acc[kWarps][D];
  const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = h / (a.cache.Hq / a.cache.Hkv);
  if (t >= a.cu_seqlens[a.n_seq] || t < a.cu_seqlens[0]) return;
  int lo = 0, hi = a.n_seq;  // the last sequence that starts at or before t
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.cu_seqlens[mid] <= t) lo = mid;
    else hi = mid;
  }
  const int s = lo, count = a.cu_seqlens[s + 1] - a.cu_seqlens[s];
  const int len = kv4_length(a, s), seen = min(len, len - count + (t - a.cu_seqlens[s]) + 1);
  const T* q = static_cast<const T*>(a.q.data) + t * a.q.token_stride + h * a.q.head_stride;
  float x[E], o[E] = {}, m = -FLT_MAX, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) x[e] = kv4_to_float(q[lane * E + e]);
  for (int p = warp; p < seen; p += kWarps) {
    const uint8_t* block = kv4_page(a, s, p, g);
    if (!block) continue;
    float k[E], v[E], dot = 0.f;
    load_values<D, true>(block, p % kPageTokens, lane, k);
    load_values<D, false>(block, p % kPageTokens, lane, v);
#pragma unroll
    for (int e = 0; e < E; ++e) dot = fmaf(x[e], k[e], dot);
    dot = warp_sum(dot) * a.scale;
    const float mn = dot > m ? dot : m, c = __expf(m - mn), w = __expf(dot - mn);
    m = mn;
    l = l * c + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * c + w * v[e];
  }
  if (lane == 0) {
    red[warp][0] = m;
    red[warp][1] = l;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) acc[warp][lane * E + e] = o[e];
  __syncthreads();
  float M = -FLT_MAX, sum = 0.f;
  for (int w = 0; w < kWarps; ++w) M = fmaxf(M, red[w][0]);
  for (int w = 0; w < kWarps; ++w) sum += red[w][1] * __expf(red[w][0] - M);
  T* out = static_cast<T*>(a.out) + t * a.out_token_stride + h * a.out_head_stride;
  for (int i = threadIdx.x; i < D; i += blockDim.x) {
    float y = 0.f;
    for (int w = 0; w < kWarps; ++w) y += acc[w][i] * __expf(red[w][0] - M);
    y = sum == 0.f ? 0.f : y / sum;
    if (a.gate.data)
      y *= sigmoidf_(static_cast<const float*>(a.gate.data)[t * a.gate.token_stride + h * a.gate.head_stride + i]);
    out[i] = kv4_from_float<T>(y);
  }
  if (a.lse && threadIdx.x == 0) a.lse[size_t(t) * a.cache.Hq + h] = sum == 0.f ? -INFINITY : M + logf(sum);
}

// One CTA per (sequence, KV head, page): what each key received from the
// sequence's query tokens and the head's group, added to what it had.
template <int D, class T>
__global__ void __launch_bounds__(kWarps * 32) kv4_weights_kernel(Kv4AttentionArgs a, const float* __restrict__ lse) {
  pdl_trigger();
  pdl_wait(lse);
  constexpr int E = D / 32;
  const int s = blockIdx.y / a.cache.Hkv, g = blockIdx.y % a.cache.Hkv, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.cache.Hq / a.cache.Hkv, first = a.cu_seqlens[s], count = a.cu_seqlens[s + 1] - first;
  const int len = kv4_length(a, s);
  for (int p = blockIdx.x * kPageTokens + warp; p < min(len, (int(blockIdx.x) + 1) * kPageTokens); p += kWarps) {
    const size_t at = (size_t(s) * a.cache.Hkv + g) * a.weights_stride + p;
    float sum = a.weights_in && p < len - count ? a.weights_in[at] : 0.f;
    const uint8_t* block = kv4_page(a, s, p, g);
    float k[E];
    if (block) {
      load_values<D, true>(block, p % kPageTokens, lane, k);
      for (int j = max(0, p - (len - count)); j < count; ++j)
        for (int h = g * G; h < (g + 1) * G; ++h) {
          const T* q = static_cast<const T*>(a.q.data) + (first + j) * a.q.token_stride + h * a.q.head_stride;
          float dot = 0.f;
#pragma unroll
          for (int e = 0; e < E; ++e) dot = fmaf(kv4_to_float(q[lane * E + e]), k[e], dot);
          sum += __expf(warp_sum(dot) * a.scale - lse[size_t(first + j) * a.cache.Hq + h]);
        }
    }
    if (lane == 0) a.weights_out[at] = sum;
  }
}

void count_launch() { g_kernel_launches.fetch_add(1, std::memory_order_relaxed); }

template <int D, class T>
void attend(const Kv4AttentionArgs& a, cudaStream_t s) {
  Kv4AttentionArgs b = a;
  if (a.weights_out && !a.lse) b.lse = static_cast<float*>(a.workspace);
  launch_pdl(kv4_attention_kernel<D, T>, dim3(a.tokens, a.cache.Hq), kWarps * 32, 0, s, b);
  count_launch();
  if (a.weights_out) {
    launch_pdl(kv4_weights_kernel<D, T>, dim3(unsigned(a.table_stride), a.n_seq * a.cache.Hkv), kWarps * 32, 0, s, b,
               static_cast<const float*>(b.lse));
    count_launch();
  }
}

}  // namespace

size_t kv4_workspace_bytes(int Hq, int Hkv, int D, size_t n_seq, size_t tokens, int sm_count) {
  (void)Hkv, (void)D, (void)n_seq, (void)sm_count;
  return std::max<size_t>(16, tokens * size_t(Hq) * 4);
}

void launch_kv4_attention(const Kv4AttentionArgs& a, cudaStream_t s) {
  if (a.tokens <= 0 || a.n_seq <= 0) return;
  const bool half = a.type == kKv4F16;
  if (a.cache.D == 64) half ? attend<64, __half>(a, s) : attend<64, __nv_bfloat16>(a, s);
  else if (a.cache.D == 128) half ? attend<128, __half>(a, s) : attend<128, __nv_bfloat16>(a, s);
  else half ? attend<256, __half>(a, s) : attend<256, __nv_bfloat16>(a, s);
}

}  // namespace qwen
