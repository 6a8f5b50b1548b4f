// Kernels of a session whose attention pages are 4-bit (rs_qwen_device_kv4): the
// step's tables, copy-on-write of a page and synthetic prefixes.
#include <atomic>

#include "kernels.h"
#include "kv4.h"

namespace qwen {

extern std::atomic<uint64_t> g_kernel_launches;

namespace {

// Per sequence: its block-table row in batch order, its cache length after the step,
// and its new tokens' slots. The attention kernels then find sequence i's pages in
// row i: one copy of a few KB a step instead of one more dependent load in every
// attention kernel of every layer. Positions count all tokens the sequence has
// been fed, cache places only those it still holds (`dropped` were evicted).
__global__ void kv4_tables_kernel(const SeqDesc* __restrict__ descs, const int32_t* __restrict__ dropped,
                                  const int32_t* __restrict__ block_table, const int32_t* __restrict__ cu_seqlens,
                                  int stride, Kv4Tables t) {
  pdl_trigger();
  pdl_wait(descs, block_table, cu_seqlens);
  const int s = blockIdx.x;
  const SeqDesc d = descs[s];
  const int at = d.position - (dropped ? dropped[s] : 0), pages = d.n_shared + d.n_new;
  const int32_t* row = block_table + size_t(d.child) * stride;
  int32_t* out = t.table + size_t(s) * t.stride;
  for (int j = threadIdx.x; j < pages; j += blockDim.x) out[j] = row[j];
  for (int i = threadIdx.x; i < d.count; i += blockDim.x) {
    const int place = at + i;
    t.slots[cu_seqlens[s] + i] =
        place / kPageTokens < pages ? int64_t(row[place / kPageTokens]) * kPageTokens + place % kPageTokens : -1;
  }
  if (threadIdx.x == 0) {
    t.kv_lens[s] = at + d.count;
    t.parents[s] = d.parent;
    t.children[s] = d.child;
  }
}

// Copy-on-write of a shared partial page: the whole page of every layer, its unused
// places included (no key behind the sequence's length is ever read).
__global__ void kv4_cow_kernel(uint8_t* pool, size_t layer_bytes, size_t page_bytes, const SeqDesc* __restrict__ descs,
                               const int32_t* __restrict__ new_pages) {
  pdl_trigger();
  pdl_wait(descs, new_pages);
  const SeqDesc d = descs[blockIdx.x];
  if (d.cow_src < 0 || d.n_new <= 0) return;
  uint8_t* base = pool + blockIdx.y * layer_bytes;
  const uint4* src = reinterpret_cast<const uint4*>(base + d.cow_src * page_bytes);
  uint4* dst = reinterpret_cast<uint4*>(base + new_pages[d.new_off] * page_bytes);
  for (size_t i = threadIdx.x; i < page_bytes / 16; i += blockDim.x) dst[i] = src[i];
}

// Synthetic keys and values [count][Hkv][D] of positions first .. first + count of
// one layer: the values that the bf16 pages hold for the same seed.
__global__ void kv4_synth_kernel(float* k, float* v, int first, int count, int Hkv, int D, int ctx, uint64_t key) {
  const float step = 1.0f / 37837.2265f;
  const int64_t per = int64_t(count) * Hkv * D;
  for (int64_t e = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; e < 2 * per; e += int64_t(gridDim.x) * blockDim.x) {
    const int sel = e >= per;
    const int64_t r = e - sel * per;
    const int i = int(r % D), g = int(r / D % Hkv);
    const int64_t pos = first + r / D / Hkv;
    const float x = synth_normal(key, ((uint64_t(sel) * Hkv + g) * ctx + pos) * D + i, step);
    (sel ? v : k)[r] = __bfloat162float(__float2bfloat16_rn(x));
  }
}

}  // namespace

void launch_kv4_tables(const SeqDesc* descs, int n_seq, const int32_t* dropped, const int32_t* block_table, int stride,
                       const int32_t* cu_seqlens, const Kv4Tables& t, cudaStream_t s) {
  launch_pdl(kv4_tables_kernel, n_seq, 256, 0, s, descs, dropped, block_table, cu_seqlens, stride, t);
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}

void launch_kv4_cow(uint8_t* pool, int layers, size_t layer_bytes, size_t page_bytes, const SeqDesc* descs, int n_seq,
                    const int32_t* new_pages, cudaStream_t s) {
  launch_pdl(kv4_cow_kernel, dim3(n_seq, layers), 256, 0, s, pool, layer_bytes, page_bytes, descs, new_pages);
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}

void launch_kv4_synth(float* k, float* v, int first, int count, int Hkv, int D, int ctx, int layer, uint64_t seed,
                      cudaStream_t s) {
  const uint64_t key = mix64(seed * 0x632BE59BD9B4E019ull ^ mix64(0x4B56000000000000ull + layer));
  kv4_synth_kernel<<<592, 256, 0, s>>>(k, v, first, count, Hkv, D, ctx, key);
  QWEN_CUDA(cudaGetLastError());
  g_kernel_launches.fetch_add(1, std::memory_order_relaxed);
}

}  // namespace qwen
