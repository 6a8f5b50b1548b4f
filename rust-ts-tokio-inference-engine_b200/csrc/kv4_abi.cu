// C ABI of the 4-bit KV-cache operators (include/qwen_b200.h): argument checks,
// the caller's device and stream, and the error convention.
#include <algorithm>
#include <climits>
#include <cmath>
#include <cstring>
#include <string>

#include "../../include/qwen_b200.h"
#include "kernels.h"
#include "kv4.h"

using namespace qwen;

namespace {

// 0 on success, -1 with a NUL-terminated message; no exception passes.
template <class F>
int guarded(char* error, size_t capacity, F f) noexcept {
  const char* message = "unknown native CUDA exception";
  std::string text;
  try {
    f();
    return 0;
  } catch (const std::exception& e) {
    try {
      text = e.what();
      message = text.c_str();
    } catch (...) {
    }
  } catch (...) {
  }
  if (error && capacity) {
    const size_t n = std::min(std::strlen(message), capacity - 1);
    std::memcpy(error, message, n);
    error[n] = 0;
  }
  return -1;
}

void need(bool ok, const char* message) {
  if (!ok) throw std::invalid_argument(message);
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// The cache's device for the length of a call, then the caller's again.
struct OnDevice {
  int before = 0;
  explicit OnDevice(int device) {
    QWEN_CUDA(cudaGetDevice(&before));
    if (before != device) QWEN_CUDA(cudaSetDevice(device));
    now = device;
  }
  ~OnDevice() {
    if (before != now) cudaSetDevice(before);
  }
  int now = 0;
};

void check_geometry(int q_heads, int kv_heads, int head_dim) {
  need(head_dim == 64 || head_dim == 128 || head_dim == 256, "kv4: head_dim must be 64, 128 or 256");
  need(kv_heads >= 1 && kv_heads <= 1024, "kv4: kv_heads must be 1 to 1024");
  need(q_heads >= kv_heads && q_heads % kv_heads == 0, "kv4: q_heads must be a multiple of kv_heads");
  need(q_heads / kv_heads <= 16, "kv4: at most 16 query heads per KV head");
}

Kv4View view(const rs_qwen_kv4_cache* c) {
  need(c, "kv4: null cache");
  check_geometry(c->q_heads, c->kv_heads, c->head_dim);
  need(c->pool && aligned(c->pool, 16), "kv4: the pool must be a 16-byte aligned device pointer");
  need(c->pages >= 1 && c->pages <= uint64_t(INT32_MAX), "kv4: page count must be 1 to 2^31 - 1");
  need(aligned(c->status, 4), "kv4: the status word must be 4-byte aligned");
  Kv4View v;
  v.pool = static_cast<uint8_t*>(c->pool);
  v.pages = c->pages;
  v.Hq = c->q_heads;
  v.Hkv = c->kv_heads;
  v.D = c->head_dim;
  v.status = c->status;
  return v;
}

size_t type_size(uint32_t type) { return type == RS_QWEN_F32 ? 4 : 2; }

Kv4Rows rows(const rs_qwen_kv4_rows& r, uint32_t type, const char* message) {
  need(aligned(r.data, type_size(type)), message);
  return {r.data, r.token_stride, r.head_stride};
}

}  // namespace

extern "C" {

size_t rs_qwen_kv4_page_bytes(int kv_heads, int head_dim) {
  if (kv_heads < 1 || kv_heads > 1024 || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
  return size_t(kv_heads) * kv4_block_bytes(head_dim);
}

size_t rs_qwen_kv4_workspace_bytes(const rs_qwen_kv4_cache* cache, size_t n_seq, size_t tokens) {
  size_t bytes = 0;
  char message[8];
  guarded(message, sizeof(message), [&] {
    need(cache, "");
    check_geometry(cache->q_heads, cache->kv_heads, cache->head_dim);
    need(n_seq <= size_t(INT32_MAX) && tokens <= size_t(INT32_MAX), "");
    int sms = 148;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, cache->device) != cudaSuccess) {
      cudaGetLastError();
      sms = 148;
    }
    bytes = kv4_workspace_bytes(cache->q_heads, cache->kv_heads, cache->head_dim, n_seq, tokens, sms);
  });
  return bytes;
}

int rs_qwen_kv4_append(const rs_qwen_kv4_cache* cache, const rs_qwen_kv4_append_args* args, void* stream, char* error,
                       size_t capacity) {
  return guarded(error, capacity, [&] {
    Kv4AppendArgs a;
    a.cache = view(cache);
    need(args, "kv4 append: null arguments");
    need(args->dtype <= RS_QWEN_BF16 && args->q_out_dtype <= RS_QWEN_BF16, "kv4 append: unknown dtype");
    need(args->tokens <= size_t(INT32_MAX), "kv4 append: too many tokens");
    if (!args->tokens) return;
    need(args->q.data || args->k.data, "kv4 append: neither queries nor keys");
    need(!args->k.data == !args->v.data, "kv4 append: keys and values go together");
    need(!args->q.data == !args->q_out, "kv4 append: queries and their output go together");
    need(!args->k.data || (args->slots && aligned(args->slots, 8)), "kv4 append: slots missing or not 8-byte aligned");
    need(aligned(args->q_out, 16), "kv4 append: q_out must be 16-byte aligned");
    need(aligned(args->q_norm, 4) && aligned(args->k_norm, 4), "kv4 append: norm gains must be 4-byte aligned");
    need(args->rope_dims >= 0 && args->rope_dims % 2 == 0 && args->rope_dims <= cache->head_dim,
         "kv4 append: rope_dims must be even, 0 to head_dim");
    need(!args->rope_dims || (args->positions && aligned(args->positions, 4)),
         "kv4 append: positions missing or not 4-byte aligned");
    need(!args->rope_dims || args->theta > 1.f, "kv4 append: theta must be above 1");
    need((!args->q_norm && !args->k_norm) || args->epsilon > 0.f, "kv4 append: epsilon must be positive");
    a.q = rows(args->q, args->dtype, "kv4 append: q must be aligned to its type");
    a.k = rows(args->k, args->dtype, "kv4 append: k must be aligned to its type");
    a.v = rows(args->v, args->dtype, "kv4 append: v must be aligned to its type");
    a.type = args->dtype;
    a.q_type = args->q_out_dtype;
    a.tokens = int(args->tokens);
    a.q_norm = args->q_norm;
    a.k_norm = args->k_norm;
    a.eps = args->epsilon;
    a.theta = double(args->theta);
    a.rope = args->rope_dims;
    a.positions = args->positions;
    a.slots = args->slots;
    a.q_out = args->q_out;
    OnDevice on(cache->device);
    launch_kv4_append(a, static_cast<cudaStream_t>(stream));
  });
}

int rs_qwen_kv4_read(const rs_qwen_kv4_cache* cache, size_t tokens, const int64_t* slots, uint32_t dtype, void* k,
                     void* v, void* stream, char* error, size_t capacity) {
  return guarded(error, capacity, [&] {
    const Kv4View c = view(cache);
    need(dtype <= RS_QWEN_BF16, "kv4 read: unknown dtype");
    need(tokens <= size_t(INT32_MAX), "kv4 read: too many tokens");
    if (!tokens) return;
    need(slots && aligned(slots, 8), "kv4 read: slots missing or not 8-byte aligned");
    need(k && v && aligned(k, 16) && aligned(v, 16), "kv4 read: outputs missing or not 16-byte aligned");
    need(tokens * size_t(c.Hkv) * size_t(c.D / 4) <= size_t(INT32_MAX) * 256, "kv4 read: too many tokens");
    OnDevice on(cache->device);
    launch_kv4_read(c, int64_t(tokens), slots, dtype, k, v, static_cast<cudaStream_t>(stream));
  });
}

int rs_qwen_kv4_attention(const rs_qwen_kv4_cache* cache, const rs_qwen_kv4_attention_args* args, void* stream,
                          char* error, size_t capacity) {
  return guarded(error, capacity, [&] {
    Kv4AttentionArgs a;
    a.cache = view(cache);
    need(args, "kv4 attention: null arguments");
    need(args->dtype == RS_QWEN_F16 || args->dtype == RS_QWEN_BF16, "kv4 attention: queries must be fp16 or bf16");
    need(args->n_seq <= size_t(INT32_MAX) / size_t(cache->kv_heads) &&
             args->tokens <= size_t(INT32_MAX) / size_t(cache->q_heads),
         "kv4 attention: too many sequences or tokens");
    if (!args->n_seq || !args->tokens) return;
    need(args->q.data && args->out.data, "kv4 attention: queries or output missing");
    need(args->max_count >= 1, "kv4 attention: max_count must be positive");
    need(args->cu_seqlens && args->kv_lens && args->block_table && aligned(args->cu_seqlens, 4) &&
             aligned(args->kv_lens, 4) && aligned(args->block_table, 4),
         "kv4 attention: cu_seqlens, kv_lens or block_table missing or not 4-byte aligned");
    need(args->table_stride >= 1 && args->table_stride <= INT32_MAX / kPageTokens,
         "kv4 attention: table_stride must be 1 to 2^31 / 16 pages");
    need(args->scale >= 0.f && std::isfinite(args->scale), "kv4 attention: scale must be finite and not negative");
    need(aligned(args->lse, 4) && aligned(args->weights_in, 4) && aligned(args->weights_out, 4),
         "kv4 attention: lse and weights must be 4-byte aligned");
    need(args->weights_out || !args->weights_in, "kv4 attention: weights_in needs weights_out");
    need(!args->weights_out || args->weights_stride >= 1, "kv4 attention: weights_stride must be positive");
    a.q = rows(args->q, args->dtype, "kv4 attention: q must be aligned to its type");
    a.gate = rows(args->gate, RS_QWEN_F32, "kv4 attention: the gate must be 4-byte aligned");
    rows(args->out, args->dtype, "kv4 attention: out must be aligned to its type");
    a.out = const_cast<void*>(args->out.data);
    a.out_token_stride = args->out.token_stride;
    a.out_head_stride = args->out.head_stride;
    a.type = args->dtype;
    a.n_seq = int(args->n_seq);
    a.tokens = int(args->tokens);
    a.max_count = int(std::min(args->max_count, args->tokens));
    a.cu_seqlens = args->cu_seqlens;
    a.kv_lens = args->kv_lens;
    a.table = args->block_table;
    a.table_stride = args->table_stride;
    a.scale = args->scale > 0.f ? args->scale : 1.f / std::sqrt(float(cache->head_dim));
    a.lse = args->lse;
    a.weights_in = args->weights_in;
    a.weights_out = args->weights_out;
    a.weights_stride = args->weights_stride;
    a.workspace = args->workspace;
    a.workspace_bytes = args->workspace_bytes;
    check_kv4_attention(a);
    OnDevice on(cache->device);
    QWEN_CUDA(cudaDeviceGetAttribute(&a.sm_count, cudaDevAttrMultiProcessorCount, cache->device));
    need(args->workspace && aligned(args->workspace, 16) &&
             args->workspace_bytes >= kv4_workspace_bytes(cache->q_heads, cache->kv_heads, cache->head_dim, args->n_seq,
                                                          args->tokens, a.sm_count),
         "kv4 attention: workspace missing, not 16-byte aligned or smaller than rs_qwen_kv4_workspace_bytes");
    launch_kv4_attention(a, static_cast<cudaStream_t>(stream));
  });
}

int rs_qwen_kv4_evict(const rs_qwen_kv4_cache* cache, const rs_qwen_kv4_evict_args* args, void* stream, char* error,
                      size_t capacity) {
  return guarded(error, capacity, [&] {
    Kv4EvictArgs a;
    a.cache = view(cache);
    need(args, "kv4 evict: null arguments");
    need(args->n_seq <= size_t(INT32_MAX) / size_t(cache->kv_heads), "kv4 evict: too many sequences");
    if (!args->n_seq) return;
    need(args->keep >= 1, "kv4 evict: keep must be positive");
    need(args->recent >= 0 && args->recent <= args->keep, "kv4 evict: recent must be 0 to keep");
    need(args->kv_lens && args->src_table && args->dst_table && args->weights && args->kept && args->new_lens,
         "kv4 evict: kv_lens, tables, weights, kept or new_lens missing");
    need(aligned(args->kv_lens, 4) && aligned(args->src_table, 4) && aligned(args->dst_table, 4) &&
             aligned(args->weights, 4) && aligned(args->kept, 4) && aligned(args->new_lens, 4) &&
             aligned(args->weights_out, 4),
         "kv4 evict: arrays must be 4-byte aligned");
    need(args->src_stride >= 1 && args->src_stride <= INT32_MAX / kPageTokens,
         "kv4 evict: src_stride must be 1 to 2^31 / 16 pages");
    need(args->dst_stride >= (args->keep + int64_t(kPageTokens) - 1) / kPageTokens && args->dst_stride <= INT32_MAX / kPageTokens,
         "kv4 evict: dst_stride must cover keep tokens");
    need(args->weights_stride >= 1, "kv4 evict: weights_stride must be positive");
    need(!args->weights_out || args->weights_out_stride >= args->keep, "kv4 evict: weights_out_stride must cover keep");
    need(args->weights_out != args->weights, "kv4 evict: weights_out must not be weights");
    need(args->keep <= INT32_MAX / 32 && args->n_seq * uint64_t(cache->kv_heads) * ((uint64_t(args->keep) * (cache->head_dim / 16 + 2) + 255) / 256) <=
             uint64_t(INT32_MAX), "kv4 evict: too many kept keys");
    a.n_seq = int(args->n_seq);
    a.kv_lens = args->kv_lens;
    a.src_table = args->src_table;
    a.dst_table = args->dst_table;
    a.src_stride = args->src_stride;
    a.dst_stride = args->dst_stride;
    a.weights = args->weights;
    a.weights_stride = args->weights_stride;
    a.keep = args->keep;
    a.recent = args->recent;
    a.kept = args->kept;
    a.new_lens = args->new_lens;
    a.weights_out = args->weights_out;
    a.weights_out_stride = args->weights_out_stride;
    OnDevice on(cache->device);
    launch_kv4_evict(a, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
