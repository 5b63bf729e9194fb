// serving.cuh — host side of the paged-cache operators: argument checks,
// tensor maps, workspace layout and launches. Included at the end of qb.cu
// (it uses that file's error, launch and tensor-map helpers).
#pragma once
#include "paged_attention_tc.cuh"
#include "paged_decode.cuh"
#include "sample.cuh"

namespace {

constexpr size_t kPagedZeroBytes = 8192;  // tickets: the workspace's part that must start at zero
constexpr int kPagedMaxCtas = (int)(kPagedZeroBytes / 4);

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
// cut units, the pieces' (m, l) and O of the kernel that runs, and for a shared
// prefix every row's result over the prefix.
struct PagedWorkspace {
  size_t cut, ml, o, base_lse, base, bytes;
};
PagedWorkspace paged_workspace(int grid, int rows, long long base_rows) {
  PagedWorkspace w;
  w.cut = kPagedZeroBytes;
  w.ml = w.cut + align_up((size_t)grid * sizeof(PtUnit), 256);
  w.o = w.ml + align_up((size_t)2 * grid * rows * 2 * sizeof(float), 256);
  w.base_lse = w.o + (size_t)2 * grid * rows * kAttnD * sizeof(float);
  w.base = w.base_lse + align_up((size_t)base_rows * sizeof(float), 256);
  w.bytes = w.base + (size_t)base_rows * kAttnD * sizeof(float);
  return w;
}
int decode_grid() { return std::min(current_sm_count() * kPdCtasPerSm, kPagedMaxCtas); }
int tc_grid() { return std::min(current_sm_count(), kPagedMaxTcCtas); }

// Whether the few-rows kernel takes the call: its 16 MMA rows hold every
// sequence's query rows of a KV head. Measured against the other one (32/8
// heads, pages of 64, 4 and 16 rows a head, captured): one sequence of 1000
// keys 10 and 14 against 16 us, of 32768 keys 32 and 40 against 43 us, of 131072
// keys 91 and 99 against 113 us, 32 of 4096 keys 90 and 92 against 120 us, 64 of
// 500 keys 31 and 35 against 51 us. Above 16 rows it would read the cache twice.
bool few_rows(int max_queries, int G) { return (long long)max_queries * G <= kPdRows; }

PagedWorkspace workspace_for(int max_queries, int G, int n_heads, int prefix_tokens) {
  const bool tc = !few_rows(max_queries, G) || prefix_tokens > 0;
  // the few-rows kernel's pieces fit in the other's room, which a prefix's second pass uses
  static_assert(kPdCtasPerSm * kPdRows <= kPtRows, "pieces of the few-rows kernel");
  return tc ? paged_workspace(tc_grid(), kPtRows, (long long)prefix_tokens * n_heads)
            : paged_workspace(decode_grid(), kPdRows, 0);
}

// One device's function attribute, set once.
template <typename K>
cudaError_t smem_attr(K kernel, bool (&set)[kMaxDevices], size_t bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev < kMaxDevices && set[dev])) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e == cudaSuccess && dev < kMaxDevices) set[dev] = true;
  return e;
}

cudaError_t launch_paged_decode(const CUtensorMap& k, const CUtensorMap& v, PagedAttnArgs a, uint8_t* ws,
                                const PagedWorkspace& w, cudaStream_t st) {
  static bool set[kMaxDevices] = {};
  cudaError_t e = smem_attr(paged_decode_kernel, set, pd_smem_bytes());
  if (e != cudaSuccess) return e;
  a.tickets = reinterpret_cast<unsigned*>(ws);
  a.part_ml = reinterpret_cast<float*>(ws + w.ml);
  a.part_o = reinterpret_cast<float*>(ws + w.o);
  return launch_ex(paged_decode_kernel, dim3(decode_grid()), dim3(kPdThreads), pd_smem_bytes(), st, k, v, a);
}

// Units of a launch: full ones, and one begun by each sequence.
long long tc_units(int tokens, int n_seqs, int G) { return tokens / (2 * (128 / G)) + std::min(n_seqs, tokens); }

cudaError_t launch_paged_tc(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, PagedTcArgs a,
                            uint8_t* ws, const PagedWorkspace& w, cudaStream_t st) {
  static bool set[kMaxDevices] = {};
  cudaError_t e = smem_attr(paged_tc_kernel, set, pt_smem_bytes(kPtMaxUnits));
  if (e != cudaSuccess) return e;
  a.cut = reinterpret_cast<PtUnit*>(ws + w.cut);
  a.part_ml = reinterpret_cast<float*>(ws + w.ml);
  a.part_o = reinterpret_cast<float*>(ws + w.o);
  const int grid = tc_grid();
  e = launch_ex(paged_tc_kernel, dim3(grid), dim3(kPtThreads), pt_smem_bytes(a.max_units), st, q, k, v, a);
  if (e != cudaSuccess) return e;
  return launch_ex(paged_join_kernel, dim3(grid * kPjCtasPerSm), dim3(kPjThreads), 0, st, a, grid);
}

int check_tiles(int tokens, int n_seqs, int G, int n_kv_heads, int table_width, int page_size) {
  const long long units = tc_units(tokens, n_seqs, G);
  if (units > kPtMaxUnits) return set_err(nullptr, QB_ERR_UNSUPPORTED, "more than 4096 blocks of 256 query rows per KV head");
  // sequences (or blocks of rows) x heads x key tiles: the kernels count places of the line in 32 bits
  if (std::max((long long)n_seqs, units) * ((long long)table_width * page_size / kPdKeys + 2 + kPtUnitCost) >
      0x7fffffffll / n_kv_heads)
    return set_err(nullptr, QB_ERR_UNSUPPORTED, "sequences x KV heads x 64-key tiles of the table above 2^31");
  return QB_OK;
}

// Attention of the whole call; prefix_len 0: without a shared prefix.
int run_paged_attention(const void* q, const void* k_pages, const void* v_pages, int num_pages, int page_size,
                        const int* prefix_table, int prefix_pages, int prefix_len, const int* page_table,
                        int table_width, const int* q_start, const int* kv_lens, int n_seqs, int tokens,
                        int max_queries, int n_heads, int n_kv_heads, int window, int sinks, void* out,
                        void* workspace, size_t workspace_bytes, int* device_status, void* stream) {
  if (!ptr_ok(k_pages) || !ptr_ok(v_pages) || !ptr_ok(workspace) || (reinterpret_cast<uintptr_t>(workspace) & 255) != 0)
    return set_err(nullptr, QB_ERR_ARG, "pools must be 16-byte and the workspace 256-byte aligned device pointers");
  if (!page_table || !q_start || !kv_lens || !device_status)
    return set_err(nullptr, QB_ERR_ARG, "page_table, q_start, kv_lens and device_status must be device pointers");
  int rc = check_heads(n_heads, n_kv_heads);
  if (rc == QB_OK) rc = check_pages(num_pages, page_size, n_kv_heads, table_width, n_seqs, tokens);
  if (rc != QB_OK) return rc;
  const int G = n_heads / n_kv_heads;
  if (window < 0 || sinks < 0) return set_err(nullptr, QB_ERR_ARG, "window and sinks must not be negative");
  if (prefix_len < 0 || prefix_pages < 0 || (long long)prefix_len > (long long)prefix_pages * page_size)
    return set_err(nullptr, QB_ERR_ARG, "prefix_len must lie in 0..prefix_pages x page_size");
  if (prefix_len > 0 && !prefix_table) return set_err(nullptr, QB_ERR_ARG, "prefix_table must be a device pointer");
  if (max_queries < 1 && tokens > 0) return set_err(nullptr, QB_ERR_ARG, "max_queries must be at least 1");
  if (tokens == 0) return QB_OK;
  if (!ptr_ok(q) || !ptr_ok(out) || (reinterpret_cast<uintptr_t>(out) & 31) != 0)
    return set_err(nullptr, QB_ERR_ARG, "q must be a 16-byte and out a 32-byte aligned device pointer");
  if (max_queries > tokens) max_queries = tokens;
  rc = check_tiles(tokens, n_seqs, G, n_kv_heads, table_width, page_size);
  if (rc == QB_OK && prefix_len > 0) {
    rc = check_pages(num_pages, page_size, n_kv_heads, prefix_pages, 1, tokens);
    if (rc == QB_OK) rc = check_tiles(tokens, 1, G, n_kv_heads, prefix_pages, page_size);
  }
  if (rc != QB_OK) return rc;
  const bool few = few_rows(max_queries, G);
  const PagedWorkspace w = workspace_for(max_queries, G, n_heads, prefix_len > 0 ? tokens : 0);
  if (workspace_bytes < w.bytes) return set_err(nullptr, QB_ERR_ARG, "workspace smaller than qb_paged_workspace_bytes()");
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  cudaStream_t st = static_cast<cudaStream_t>(stream);

  PagedBatch b;
  std::memset(&b, 0, sizeof(b));
  b.page_table = page_table;
  b.q_start = q_start;
  b.kv_lens = kv_lens;
  b.n_seqs = n_seqs;
  b.tokens = tokens;
  b.table_width = table_width;
  b.num_pages = num_pages;
  b.page_log2 = log2_of(page_size);
  b.max_queries = max_queries;
  b.window = std::min(window, 1 << 30);  // longer than any sequence: the whole of it
  b.sinks = std::min(sinks, 1 << 30);
  RowSink sink;
  std::memset(&sink, 0, sizeof(sink));
  sink.out = static_cast<bf16*>(out);

  const long long rows = (long long)num_pages * n_kv_heads * page_size;
  CUtensorMap mq, mk, mv;
  if (!few || prefix_len > 0) {
    const int box = std::min(page_size, kPtKeys);
    if (!make_q3_map(&mq, q, tokens, n_heads, G, 128 / G) || !make_rows_map(&mk, k_pages, rows, kAttnD, box) ||
        !make_rows_map(&mv, v_pages, rows, kAttnD, box))
      return set_err(nullptr, QB_ERR_CUDA, "cuTensorMapEncodeTiled failed for q or the page pools");
    PagedTcArgs a;
    std::memset(&a, 0, sizeof(a));
    a.Hq = n_heads;
    a.Hkv = n_kv_heads;
    a.G = G;
    a.err = device_status;
    if (prefix_len > 0) {  // the prefix once for all rows, as one sequence whose rows see every key
      a.b = b;
      a.b.page_table = prefix_table;
      a.b.q_start = nullptr;
      a.b.kv_lens = nullptr;
      a.b.n_seqs = 1;
      a.b.table_width = prefix_pages;
      a.b.kv_all = prefix_len;
      a.b.window = a.b.sinks = 0;
      a.max_units = (int)tc_units(tokens, 1, G);
      a.sink.out32 = reinterpret_cast<float*>(ws + w.base);
      a.sink.lse32 = reinterpret_cast<float*>(ws + w.base_lse);
      cudaError_t e = launch_paged_tc(mq, mk, mv, a, ws, w, st);
      if (e != cudaSuccess) return cuda_fail(nullptr, e, "shared prefix launch");
      sink.base32 = a.sink.out32;
      sink.base_lse = a.sink.lse32;
    }
    if (!few) {
      a.b = b;
      a.max_units = (int)tc_units(tokens, n_seqs, G);
      a.sink = sink;
      cudaError_t e = launch_paged_tc(mq, mk, mv, a, ws, w, st);
      if (e != cudaSuccess) return cuda_fail(nullptr, e, "paged attention launch");
      return QB_OK;
    }
  }
  const int box = std::min(page_size, kPdKeys);
  if (!make_rows_map(&mk, k_pages, rows, kAttnD, box) || !make_rows_map(&mv, v_pages, rows, kAttnD, box))
    return set_err(nullptr, QB_ERR_CUDA, "cuTensorMapEncodeTiled failed for the page pools");
  PagedAttnArgs a;
  std::memset(&a, 0, sizeof(a));
  a.b = b;
  a.q = static_cast<const bf16*>(q);
  a.Hq = n_heads;
  a.Hkv = n_kv_heads;
  a.G = G;
  a.sink = sink;
  a.err = device_status;
  cudaError_t e = launch_paged_decode(mk, mv, a, ws, w, st);
  if (e != cudaSuccess) return cuda_fail(nullptr, e, "paged attention launch");
  return QB_OK;
}

template <typename T>
cudaError_t launch_sample(SampleArgs a, int rows, cudaStream_t st) {
  static bool set[kMaxDevices] = {};
  a.slice = (int)align_up((a.vocab + kSmCluster - 1) / kSmCluster, kSmWarps * 8);
  cudaError_t e = smem_attr(sample_kernel<T>, set, sample_smem_bytes(kSmMaxVocab / kSmCluster, sizeof(T)));
  if (e != cudaSuccess) return e;
  return launch_ex(sample_kernel<T>, dim3((unsigned)rows * kSmCluster), dim3(kSmThreads),
                   sample_smem_bytes(a.slice, sizeof(T)), st, a);
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

int qb_paged_workspace_bytes(int max_queries, int n_heads, int n_kv_heads, int prefix_tokens, size_t* bytes) {
  if (!bytes) return set_err(nullptr, QB_ERR_ARG, "bytes is NULL");
  if (prefix_tokens < 0 || prefix_tokens > (1 << 24)) return set_err(nullptr, QB_ERR_UNSUPPORTED, "0..2^24 query rows");
  int rc = check_heads(n_heads, n_kv_heads);
  if (rc != QB_OK) return rc;
  *bytes = workspace_for(max_queries, n_heads / n_kv_heads, n_heads, prefix_tokens).bytes;
  return QB_OK;
}

int qb_paged_attention(const void* q, const void* k_pages, const void* v_pages, int num_pages, int page_size,
                       const int* page_table, int table_width, const int* q_start, const int* kv_lens, int n_seqs,
                       int tokens, int max_queries, int n_heads, int n_kv_heads, int window, int sinks, void* out,
                       void* workspace, size_t workspace_bytes, int* device_status, void* stream) {
  return run_paged_attention(q, k_pages, v_pages, num_pages, page_size, nullptr, 0, 0, page_table, table_width, q_start,
                             kv_lens, n_seqs, tokens, max_queries, n_heads, n_kv_heads, window, sinks, out, workspace,
                             workspace_bytes, device_status, stream);
}

int qb_shared_prefix_attention(const void* q, const void* k_pages, const void* v_pages, int num_pages, int page_size,
                               const int* prefix_table, int prefix_pages, int prefix_len, const int* page_table,
                               int table_width, const int* q_start, const int* kv_lens, int n_seqs, int tokens,
                               int max_queries, int n_heads, int n_kv_heads, void* out, void* workspace,
                               size_t workspace_bytes, int* device_status, void* stream) {
  return run_paged_attention(q, k_pages, v_pages, num_pages, page_size, prefix_table, prefix_pages, prefix_len,
                             page_table, table_width, q_start, kv_lens, n_seqs, tokens, max_queries, n_heads, n_kv_heads,
                             0, 0, out, workspace, workspace_bytes, device_status, stream);
}

int qb_sample_token(const void* logits, int fp32, int rows, int vocab, const float* uniforms, const float* temperature,
                    float temperature_all, const int* top_k, int top_k_all, const float* top_p, float top_p_all,
                    const float* min_p, float min_p_all, int64_t* token_out, int* device_status, void* stream) {
  if (rows < 0 || rows > (1 << 24)) return set_err(nullptr, QB_ERR_UNSUPPORTED, "0..2^24 rows");
  if (vocab < 1 || vocab > kSmMaxVocab) return set_err(nullptr, QB_ERR_UNSUPPORTED, "vocab must lie in 1..262144");
  if (rows == 0) return QB_OK;
  if (!logits || (reinterpret_cast<uintptr_t>(logits) & (fp32 ? 3 : 1)) != 0 || !uniforms || !token_out || !device_status)
    return set_err(nullptr, QB_ERR_ARG, "logits, uniforms, token_out and device_status must be device pointers");
  SampleArgs a;
  std::memset(&a, 0, sizeof(a));
  a.logits = logits;
  a.uniforms = uniforms;
  a.temperature = temperature;
  a.top_k = top_k;
  a.top_p = top_p;
  a.min_p = min_p;
  a.temperature_all = temperature_all;
  a.top_k_all = top_k_all;
  a.top_p_all = top_p_all;
  a.min_p_all = min_p_all;
  a.vocab = vocab;
  a.out = token_out;
  a.err = device_status;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = fp32 ? launch_sample<float>(a, rows, st) : launch_sample<bf16>(a, rows, st);
  if (e != cudaSuccess) return cuda_fail(nullptr, e, "sample launch");
  return QB_OK;
}

}  // extern "C"
