// serving.cuh — host side of the paged-cache operators: argument checks,
// tensor maps, workspace layout and launches. Included at the end of qb.cu
// (it uses that file's error, launch and tensor-map helpers).
#pragma once
#include "paged_decode.cuh"

namespace {

constexpr size_t kPagedZeroBytes = 8192;  // tickets: the workspace's part that must start at zero
constexpr int kPagedMaxCtas = (int)(kPagedZeroBytes / 4);

struct PagedPools {
  CUtensorMap k, v;
};

// Boxes of min(page, 64) rows x 64 dims over the pool as rows of 128 dims.
bool make_pool_map(CUtensorMap* m, const void* base, long long rows, int box_rows) {
  return make_rows_map(m, base, rows, kAttnD, box_rows);
}

int check_pages(int num_pages, int page_size, int n_kv_heads, int table_width, int n_seqs, int tokens) {
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) != 0)
    return set_err(nullptr, QB_ERR_UNSUPPORTED, "page_size must be 16, 32, 64, 128 or 256");
  if (num_pages <= 0 || (long long)num_pages * n_kv_heads * page_size > 0x7fffffffll)
    return set_err(nullptr, QB_ERR_UNSUPPORTED, "num_pages x n_kv_heads x page_size must lie in 1..2^31 - 1");
  if (n_seqs < 1 || n_seqs > kPagedMaxSeqs) return set_err(nullptr, QB_ERR_UNSUPPORTED, "1..1024 sequences");
  if (table_width < 1 || (long long)table_width * page_size > (1ll << 30))
    return set_err(nullptr, QB_ERR_UNSUPPORTED, "table_width x page_size must lie in 1..2^30");
  if (tokens < 0 || tokens > (1 << 24)) return set_err(nullptr, QB_ERR_UNSUPPORTED, "0..2^24 query rows");
  return QB_OK;
}

int check_heads(int n_heads, int n_kv_heads) {
  if (n_kv_heads <= 0 || n_heads <= 0 || n_heads % n_kv_heads != 0)
    return set_err(nullptr, QB_ERR_ARG, "n_heads must be a multiple of n_kv_heads");
  if (n_kv_heads > 64 || n_heads / n_kv_heads > 16)
    return set_err(nullptr, QB_ERR_UNSUPPORTED, "at most 64 KV heads and 16 query heads per KV head");
  return QB_OK;
}

int log2_of(int v) {
  int n = 0;
  while ((1 << n) < v) ++n;
  return n;
}

// Workspace: tickets (zero-filled by the caller once, left at zero), then the
// pieces' (m, l) and O.
struct DecodeWorkspace {
  int grid;
  size_t ml, o, bytes;
};
DecodeWorkspace decode_workspace(int sms) {
  DecodeWorkspace w;
  w.grid = std::min(sms * kPdCtasPerSm, kPagedMaxCtas);
  w.ml = kPagedZeroBytes;
  w.o = w.ml + align_up((size_t)2 * w.grid * kPdRows * 2 * sizeof(float), 256);
  w.bytes = w.o + (size_t)2 * w.grid * kPdRows * kAttnD * sizeof(float);
  return w;
}

cudaError_t launch_paged_decode(const CUtensorMap& k, const CUtensorMap& v, PagedAttnArgs a, uint8_t* ws,
                                cudaStream_t st) {
  static bool attr[kMaxDevices] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= kMaxDevices || !attr[dev]) {
    e = cudaFuncSetAttribute(paged_decode_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)pd_smem_bytes());
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) attr[dev] = true;
  }
  const DecodeWorkspace w = decode_workspace(current_sm_count());
  a.tickets = reinterpret_cast<unsigned*>(ws);
  a.part_ml = reinterpret_cast<float*>(ws + w.ml);
  a.part_o = reinterpret_cast<float*>(ws + w.o);
  return launch_ex(paged_decode_kernel, dim3(w.grid), dim3(kPdThreads), pd_smem_bytes(), st, k, v, a);
}

}  // namespace

extern "C" {

size_t qb_paged_zero_bytes(void) { return kPagedZeroBytes; }

int qb_rope_paged_append(const void* qkv, const void* q_norm, const void* k_norm, const void* rope_cos,
                         const void* rope_sin, int table_rows, float eps, void* k_pages, void* v_pages, int num_pages,
                         int page_size, const int* page_table, int table_width, const int* q_start,
                         const int* kv_lens, int n_seqs, int tokens, int first_position, int n_heads, int n_kv_heads,
                         void* q_out, int* device_status, void* stream) {
  if (!ptr_ok(k_pages) || !ptr_ok(v_pages) || !ptr_ok(rope_cos) || !ptr_ok(rope_sin) ||
      (q_norm && !ptr_ok(q_norm)) || (k_norm && !ptr_ok(k_norm)))
    return set_err(nullptr, QB_ERR_ARG, "pools, rope tables and norms must be 16-byte aligned device pointers");
  if (!page_table || !q_start || !kv_lens || !device_status)
    return set_err(nullptr, QB_ERR_ARG, "page_table, q_start, kv_lens and device_status must be device pointers");
  int rc = check_heads(n_heads, n_kv_heads);
  if (rc == QB_OK) rc = check_pages(num_pages, page_size, n_kv_heads, table_width, n_seqs, tokens);
  if (rc != QB_OK) return rc;
  if (table_rows < 1 || first_position < 0) return set_err(nullptr, QB_ERR_ARG, "rope table and first_position must not be negative");
  if (tokens == 0) return QB_OK;
  if (!ptr_ok(qkv) || !ptr_ok(q_out)) return set_err(nullptr, QB_ERR_ARG, "qkv and q_out must be 16-byte aligned device pointers");
  AppendArgs a;
  std::memset(&a, 0, sizeof(a));
  a.b.page_table = page_table;
  a.b.q_start = q_start;
  a.b.kv_lens = kv_lens;
  a.b.n_seqs = n_seqs;
  a.b.tokens = tokens;
  a.b.table_width = table_width;
  a.b.num_pages = num_pages;
  a.b.page_log2 = log2_of(page_size);
  a.b.max_queries = tokens;
  a.qkv = static_cast<const bf16*>(qkv);
  a.q_norm = static_cast<const bf16*>(q_norm);
  a.k_norm = static_cast<const bf16*>(k_norm);
  a.cos = static_cast<const bf16*>(rope_cos);
  a.sin = static_cast<const bf16*>(rope_sin);
  a.eps = eps;
  a.Hq = n_heads;
  a.Hkv = n_kv_heads;
  a.table_rows = table_rows;
  a.first_position = first_position;
  a.k_pages = static_cast<bf16*>(k_pages);
  a.v_pages = static_cast<bf16*>(v_pages);
  a.q_out = static_cast<bf16*>(q_out);
  a.err = device_status;
  cudaError_t e = launch_ex(paged_append_kernel, dim3(tokens), dim3(kAppThreads), 0, static_cast<cudaStream_t>(stream), a);
  if (e != cudaSuccess) return cuda_fail(nullptr, e, "paged append launch");
  return QB_OK;
}

int qb_paged_workspace_bytes(int max_queries, int n_heads, int n_kv_heads, size_t* bytes) {
  if (!bytes) return set_err(nullptr, QB_ERR_ARG, "bytes is NULL");
  int rc = check_heads(n_heads, n_kv_heads);
  if (rc != QB_OK) return rc;
  (void)max_queries;
  *bytes = decode_workspace(current_sm_count()).bytes;
  return QB_OK;
}

int qb_paged_attention(const void* q, const void* k_pages, const void* v_pages, int num_pages, int page_size,
                       const int* page_table, int table_width, const int* q_start, const int* kv_lens, int n_seqs,
                       int tokens, int max_queries, int n_heads, int n_kv_heads, int window, int sinks, void* out,
                       void* workspace, size_t workspace_bytes, int* device_status, void* stream) {
  if (!ptr_ok(k_pages) || !ptr_ok(v_pages) || !ptr_ok(workspace))
    return set_err(nullptr, QB_ERR_ARG, "pools and workspace must be 16-byte aligned device pointers");
  if (!page_table || !q_start || !kv_lens || !device_status)
    return set_err(nullptr, QB_ERR_ARG, "page_table, q_start, kv_lens and device_status must be device pointers");
  int rc = check_heads(n_heads, n_kv_heads);
  if (rc == QB_OK) rc = check_pages(num_pages, page_size, n_kv_heads, table_width, n_seqs, tokens);
  if (rc != QB_OK) return rc;
  if (window < 0 || sinks < 0) return set_err(nullptr, QB_ERR_ARG, "window and sinks must not be negative");
  if (max_queries < 1 && tokens > 0) return set_err(nullptr, QB_ERR_ARG, "max_queries must be at least 1");
  if (tokens == 0) return QB_OK;
  if (!ptr_ok(q) || !ptr_ok(out)) return set_err(nullptr, QB_ERR_ARG, "q and out must be 16-byte aligned device pointers");
  const int G = n_heads / n_kv_heads;
  if (max_queries > tokens) max_queries = tokens;
  size_t need = 0;
  rc = qb_paged_workspace_bytes(max_queries, n_heads, n_kv_heads, &need);
  if (rc != QB_OK) return rc;
  if (workspace_bytes < need) return set_err(nullptr, QB_ERR_ARG, "workspace smaller than qb_paged_workspace_bytes()");
  PagedAttnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.b.page_table = page_table;
  a.b.q_start = q_start;
  a.b.kv_lens = kv_lens;
  a.b.n_seqs = n_seqs;
  a.b.tokens = tokens;
  a.b.table_width = table_width;
  a.b.num_pages = num_pages;
  a.b.page_log2 = log2_of(page_size);
  a.b.max_queries = max_queries;
  a.b.window = std::min(window, 1 << 30);  // longer than any sequence: the whole of it
  a.b.sinks = std::min(sinks, 1 << 30);
  a.q = static_cast<const bf16*>(q);
  a.Hq = n_heads;
  a.Hkv = n_kv_heads;
  a.G = G;
  a.sink.out = static_cast<bf16*>(out);
  a.err = device_status;
  CUtensorMap mk, mv;
  const long long rows = (long long)num_pages * n_kv_heads * page_size;
  const int box = std::min(page_size, kPdKeys);
  if (!make_pool_map(&mk, k_pages, rows, box) || !make_pool_map(&mv, v_pages, rows, box))
    return set_err(nullptr, QB_ERR_CUDA, "cuTensorMapEncodeTiled failed for the page pools");
  if (max_queries * G > kPdRows) return set_err(nullptr, QB_ERR_UNSUPPORTED, "more than 16 query rows per KV head");
  cudaError_t e = launch_paged_decode(mk, mv, a, static_cast<uint8_t*>(workspace), static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return cuda_fail(nullptr, e, "paged attention launch");
  return QB_OK;
}

}  // extern "C"
