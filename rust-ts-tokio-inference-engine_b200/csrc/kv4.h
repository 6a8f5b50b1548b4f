// 4-bit paged KV cache: block layout and launch interface (all sm_100a).
#pragma once
#include <cuda_runtime.h>

#include <climits>

#include "common.cuh"

namespace qwen {

// Values of one (token, KV head) are quantised in groups of 64 dims, affine:
// value = scale * n + bias with n in 0..15, scale and bias bf16 (4.5 bits per
// value). A page holds kPageTokens tokens; of each (page, KV head) the pool
// keeps one contiguous block of 18 * D bytes, so a warp fetches a page with one
// bulk copy:
//   [0, 8D)    K nibbles        [8D, 16D)  V nibbles
//   [16D, 17D) K (scale, bias) pairs [token][D / 64]   [17D, 18D) V pairs
// The nibbles are stored as the tensor-core fragments that read them:
//   K: the 32-bit word of 8 consecutive dims holds dim e in nibble
//      e / 2 + 4 (e % 2), so (word >> 4 j) & 0x000F000F is the pair of dims
//      (2j, 2j + 1). Word r of a group belongs to lane r % 4 of the four lanes
//      that share a key row; each lane's words lie together, and the four
//      lanes' together, [chunk][token][lane][words], so a warp's loads touch
//      every bank once.
//   V: dim e in nibble e; word r of a group belongs to lane row r (the MMA's
//      row group), [lane rows][even tokens, odd tokens][lane row][group]: a
//      lane loads the two tokens of a k pair from places 8 entries apart.
template <int D>
struct Kv4Layout {
  static_assert(D == 64 || D == 128 || D == 256, "head_dim");
  static constexpr int kBlock = 18 * D;
  static constexpr int kGroups = D / 64;
  static constexpr int kLaneWords = D / 32;                        // K words of one lane and key
  static constexpr int kChunk = kLaneWords < 4 ? kLaneWords : 4;  // of them contiguous
  static constexpr int kRows = 512 / D;                            // V lane rows of a 32-byte segment
  static constexpr int kV = 8 * D, kKMeta = 16 * D, kVMeta = 17 * D;
  // byte of the word holding dims 8 w .. 8 w + 7 of token `tok`
  __host__ __device__ static constexpr int k_word(int tok, int w) {
    const int i = 2 * (w / 8) + (w % 8) / 4, lane = w % 4;
    return ((i / kChunk * kPageTokens + tok) * 4 + lane) * kChunk * 4 + i % kChunk * 4;
  }
  __host__ __device__ static constexpr int v_word(int tok, int w) {
    const int lane = w % 8, place = (tok & 1) * 8 + tok / 2;
    return kV + (lane / kRows * kPageTokens + place) * 32 + lane % kRows * (D / 16) + w / 8 * 4;
  }
  __host__ __device__ static constexpr int k_meta(int tok, int group) { return kKMeta + (tok * kGroups + group) * 4; }
  __host__ __device__ static constexpr int v_meta(int tok, int group) { return kVMeta + (tok * kGroups + group) * 4; }
};
constexpr size_t kv4_block_bytes(int D) { return size_t(18) * D; }
// Nibble holding dim e (0..7) of a K word.
__host__ __device__ __forceinline__ constexpr int kv4_k_nibble(int e) { return e / 2 + 4 * (e % 2); }

// One attention layer's pages: [page][KV head][block].
struct Kv4View {
  uint8_t* pool = nullptr;
  uint64_t pages = 0;
  int Hq = 0, Hkv = 0, D = 0;
  uint32_t* status = nullptr;  // device word for ErrorBits, may be null
  __host__ __device__ uint8_t* block(uint64_t page, int head) const {
    return pool + (page * uint64_t(Hkv) + uint64_t(head)) * (uint64_t(18) * D);
  }
};

enum Kv4Type : uint32_t { kKv4F32 = 0, kKv4F16 = 1, kKv4BF16 = 2 };

// Rows [token][head][D] of any strides (in elements; the D values contiguous).
struct Kv4Rows {
  const void* data = nullptr;
  int64_t token_stride = 0, head_stride = 0;
};

struct Kv4AppendArgs {
  Kv4View cache;
  Kv4Rows q, k, v;  // k and v both or neither
  uint32_t type = kKv4F32, q_type = kKv4F16;
  int tokens = 0;
  int splits = 1;           // fp32 rows given as split-K partials, summed in order
  size_t split_stride = 0;
  const float* q_norm = nullptr;  // null: no norm
  const float* k_norm = nullptr;
  float eps = 1e-6f;
  double theta = 1e7;
  int rope = 0;
  const int32_t* positions = nullptr;  // needed when rope > 0
  const int64_t* slots = nullptr;      // page * 16 + offset; negative: not stored
  void* q_out = nullptr;               // [token][Hq][D]
  const float* gate = nullptr;         // fp32 rows with q's strides, copied (summed) to gate_out
  float* gate_out = nullptr;
};
void launch_kv4_append(const Kv4AppendArgs& a, cudaStream_t s);

void launch_kv4_read(const Kv4View& cache, int64_t tokens, const int64_t* slots, uint32_t type, void* k, void* v,
                     cudaStream_t s);

struct Kv4AttentionArgs {
  Kv4View cache;
  Kv4Rows q, gate;  // q: `type`; gate: fp32, null data = none
  void* out = nullptr;
  int64_t out_token_stride = 0, out_head_stride = 0;
  uint32_t type = kKv4F16;  // q and out
  int n_seq = 0, tokens = 0, max_count = 0;
  const int32_t* cu_seqlens = nullptr;
  const int32_t* kv_lens = nullptr;
  const int32_t* table = nullptr;  // [n_seq][table_stride] page ids
  int64_t table_stride = 0;
  float scale = 0.f;
  float* lse = nullptr;                 // [token][Hq]
  const float* weights_in = nullptr;    // [n_seq][Hkv][weights_stride]
  float* weights_out = nullptr;
  int64_t weights_stride = 0;
  const int32_t* weights_in_rows = nullptr;   // row of each sequence (null: its own index; negative: none, zeros)
  const int32_t* weights_out_rows = nullptr;
  void* workspace = nullptr;
  size_t workspace_bytes = 0;
  int sm_count = 0;
  bool coarse = false;  // fp16 queries may run in kv4_chunk.cu: their output feeds something coarser than fp16
  int row_limit = INT_MAX;  // sequences with more query rows per KV head run in kv4_chunk.cu
};
// Throws std::invalid_argument for a call beyond the 32-bit places that its kernels
// count in, before any of them is launched (host values only; launch_kv4_attention
// checks too).
void check_kv4_attention(const Kv4AttentionArgs& a);
void check_kv4_chunk(const Kv4AttentionArgs& a);
// Sequences above row_limit, tcgen05 tiles of 128 rows (no lse, no weights).
size_t kv4_chunk_workspace_bytes(int Hq, int Hkv, int D, size_t n_seq, size_t tokens, int sm_count);
void launch_kv4_chunk(const Kv4AttentionArgs& a, void* workspace, cudaStream_t s);
size_t kv4_workspace_bytes(int Hq, int Hkv, int D, size_t n_seq, size_t tokens, int sm_count);
void launch_kv4_attention(const Kv4AttentionArgs& a, cudaStream_t s);

struct Kv4EvictArgs {
  Kv4View cache;
  int n_seq = 0;
  const int32_t* kv_lens = nullptr;
  const int32_t* src_table = nullptr;
  const int32_t* dst_table = nullptr;
  int64_t src_stride = 0, dst_stride = 0;
  const float* weights = nullptr;  // [n_seq][Hkv][weights_stride]
  int64_t weights_stride = 0;
  const int32_t* weights_rows = nullptr;  // row of each sequence (null: its own index)
  const int32_t* weights_out_rows = nullptr;
  int keep = 0, recent = 0;
  int32_t* kept = nullptr;  // [n_seq][Hkv][keep]
  int32_t* new_lens = nullptr;
  float* weights_out = nullptr;  // [n_seq][Hkv][weights_out_stride]
  int64_t weights_out_stride = 0;
};
void launch_kv4_evict(const Kv4EvictArgs& a, cudaStream_t s);

// ---- a session's 4-bit pages (kv4_session.cu) ----
struct SeqDesc;
// A step's tables, in batch order.
struct Kv4Tables {
  int32_t* kv_lens = nullptr;   // [n_seq] cache length after the step
  int32_t* table = nullptr;     // [n_seq][stride]
  int32_t* parents = nullptr;   // [n_seq] state slots
  int32_t* children = nullptr;
  int64_t* slots = nullptr;     // [tokens]
  int stride = 0;
};
// dropped: evicted keys of each sequence, null = none
void launch_kv4_tables(const SeqDesc* descs, int n_seq, const int32_t* dropped, const int32_t* block_table, int stride,
                       const int32_t* cu_seqlens, const Kv4Tables& t, cudaStream_t s);
void launch_kv4_cow(uint8_t* pool, int layers, size_t layer_bytes, size_t page_bytes, const SeqDesc* descs, int n_seq,
                    const int32_t* new_pages, cudaStream_t s);
void launch_kv4_synth(float* k, float* v, int first, int count, int Hkv, int D, int ctx, int layer, uint64_t seed,
                      cudaStream_t s);

// ---- element access by type ----
template <class T>
__device__ __forceinline__ float kv4_to_float(T v);
template <>
__device__ __forceinline__ float kv4_to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float kv4_to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float kv4_to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T>
__device__ __forceinline__ T kv4_from_float(float v);
template <>
__device__ __forceinline__ float kv4_from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half kv4_from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 kv4_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float kv4_scale(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float kv4_bias(uint32_t pair) { return __uint_as_float(pair & 0xFFFF0000u); }
__device__ __forceinline__ void kv4_flag(uint32_t* status, uint32_t bits) {
  if (status) atomicOr(status, bits);
}

}  // namespace qwen
