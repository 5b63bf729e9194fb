// paged.cuh — what the operators over a paged K/V cache share: the batch
// description, its checks on the device, and the append kernel.
//
// K and V live in pools [num_pages][Hkv][page][128] (bf16). Key c of sequence
// b is slot c % page of page page_table[b][c / page]; a (page, head) slab is
// contiguous. The queries of a batch are packed: sequence b owns rows
// q_start[b] .. q_start[b + 1] - 1, its last query sits at position
// kv_lens[b] - 1. The lengths and tables are device memory, so a captured
// graph follows them as they change; everything a kernel reads from them is
// checked against the sizes the host passed before it becomes an address.
//
// The reference keeps one contiguous cache per sequence
// (dryft/engine/decode.py:25-46); it has no counterpart of the pages.
#pragma once
#include "attention.cuh"

namespace qb {

constexpr int kPagedMaxSeqs = 1024;

struct PagedBatch {
  const int* page_table;  // [n_seqs][table_width]
  const int* q_start;     // [n_seqs + 1]; NULL: one sequence of `tokens` queries that all see kv_all keys
  const int* kv_lens;     // [n_seqs]
  int n_seqs, tokens, table_width, num_pages, page_log2;
  int max_queries;        // longest sequence the launch handles
  int window, sinks;      // window 0: none
  int kv_all;
};

// 16 bytes through the coherent path: what the previous kernel of the stream
// may have written while this grid was already resident is no read-only data.
__device__ __forceinline__ uint4 ld128(const void* p) { return *reinterpret_cast<const uint4*>(p); }

struct SeqSpan {
  int q0, n, kv;  // first query row, queries, cached keys (the queries' own included)
};

// Sequence s; one whose numbers lie outside the call's sizes is reported and
// becomes empty.
__device__ __forceinline__ SeqSpan paged_seq(const PagedBatch& b, int s, int* err) {
  if (b.q_start == nullptr) return SeqSpan{0, b.tokens, b.kv_all};
  SeqSpan r;
  r.q0 = b.q_start[s];
  const int q1 = b.q_start[s + 1];
  r.kv = b.kv_lens[s];
  r.n = q1 - r.q0;
  if (r.q0 < 0 || q1 < r.q0 || q1 > b.tokens || r.n > b.max_queries || r.kv < 0 ||
      r.kv > (b.table_width << b.page_log2)) {
    report_error(err, DEV_BAD_BATCH);
    return SeqSpan{0, 0, 0};
  }
  return r;
}

// The key tiles of KEYS keys that hold a key some query at positions
// p_first .. hi - 1 sees: n_sink tiles from 0, then tiles from lo_tile. Rows
// that see nothing (hi <= 0) keep one tile, in which every key is masked, so
// that their output is written.
struct TileSpan {
  int n_sink, lo_tile, count, lo;  // lo: first key of the window
};
template <int KEYS>
__device__ __forceinline__ TileSpan tile_span(int p_first, int hi, int window, int sinks) {
  TileSpan t;
  t.lo = window > 0 ? max(0, p_first - window + 1) : 0;
  if (hi <= 0) return TileSpan{0, 0, 1, 0};
  t.lo_tile = t.lo / KEYS;
  t.n_sink = window > 0 ? min((min(sinks, hi) + KEYS - 1) / KEYS, t.lo_tile) : 0;
  t.count = t.n_sink + (hi + KEYS - 1) / KEYS - t.lo_tile;
  return t;
}

// ------------------------------------------------------------------- append
struct AppendArgs {
  PagedBatch b;
  const bf16* qkv;     // [tokens][Hq*D + 2*Hkv*D]
  const bf16* q_norm;  // NULL: no norm
  const bf16* k_norm;
  const bf16* cos;     // [table_rows][D]
  const bf16* sin;
  float eps;
  int Hq, Hkv, table_rows, first_position;
  bf16* k_pages;
  bf16* v_pages;
  bf16* q_out;         // [tokens][Hq][D]
  int* err;
};

constexpr int kAppThreads = 256;
constexpr int kAppHeads = 4;  // heads that a half-warp holds at once: 64 of a token

// One CTA per token: 16 half-warps take the token's Hq + 2 Hkv heads in turn,
// lane j of a half-warp the dims [8j, 8j + 8) of its heads (one 16-byte access
// each way; the rotation's partner dim d +- 64 is lane j ^ 8). Bound by bytes:
// the token's heads are on their way before its sequence, position and page are
// looked up (three dependent reads).
//   y = x * rsqrt(mean(x^2) + eps) * gain,  out = y * cos + rot_half(y) * sin
// in fp32 with one rounding at the end (rope_attention rounds every product,
// as the reference does; the cache rows of the two may differ by an ulp).
__global__ void __launch_bounds__(kAppThreads) paged_append_kernel(const AppendArgs a) {
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x;
  const int hw = threadIdx.x >> 4, j = threadIdx.x & 15;
  const int heads = a.Hq + 2 * a.Hkv;
  const bf16* row = a.qkv + (size_t)t * heads * kAttnD + 8 * j;
  uint4 xv[kAppHeads];
  auto load = [&](int h0) {
#pragma unroll
    for (int i = 0; i < kAppHeads; ++i) {
      const int h = h0 + 16 * i + hw;
      xv[i] = h < heads ? ld128(row + (size_t)h * kAttnD) : make_uint4(0, 0, 0, 0);
    }
  };
  load(0);
  // the sequence that holds token t: the count of starts (from the second) at or below t
  int seq = 0;
  for (int s0 = 0; s0 < a.b.n_seqs; s0 += kAppThreads) {
    const int s = s0 + threadIdx.x;
    seq += __syncthreads_count(s < a.b.n_seqs && a.b.q_start[s + 1] <= t);
  }
  if (seq >= a.b.n_seqs) return;  // a row behind the last sequence
  const SeqSpan sp = paged_seq(a.b, seq, a.err);
  if (t < sp.q0 || t >= sp.q0 + sp.n) return;
  const int pos = sp.kv - sp.n + (t - sp.q0);
  const long long angle = (long long)pos + a.first_position;
  if (pos < 0 || angle >= a.table_rows) {
    if (threadIdx.x == 0) report_error(a.err, DEV_BAD_POSITION);
    return;
  }
  const uint4 cv = ld128(a.cos + (size_t)angle * kAttnD + 8 * j);
  uint4 sv = ld128(a.sin + (size_t)angle * kAttnD + 8 * j);
  const uint32_t sign = j < 8 ? 0x80008000u : 0u;  // the first half takes minus the second
  sv.x ^= sign; sv.y ^= sign; sv.z ^= sign; sv.w ^= sign;
  const int page = a.b.page_table[(size_t)seq * a.b.table_width + (pos >> a.b.page_log2)];
  const bool page_ok = page >= 0 && page < a.b.num_pages;
  if (!page_ok && threadIdx.x == 0) report_error(a.err, DEV_BAD_PAGE);
  const int slot = pos & ((1 << a.b.page_log2) - 1);
  const uint32_t c2[4] = {cv.x, cv.y, cv.z, cv.w}, s2[4] = {sv.x, sv.y, sv.z, sv.w};
  for (int h0 = 0; h0 < heads; h0 += 16 * kAppHeads) {
    if (h0 > 0) load(h0);
#pragma unroll
    for (int i = 0; i < kAppHeads; ++i) {
      const int h = h0 + 16 * i + hw;
      if (h0 + 16 * i >= heads) break;
      const bool turn = h < a.Hq + a.Hkv;
      const bf16* gain = h < a.Hq ? a.q_norm : a.k_norm;
      float x[8] = {bf_lo(xv[i].x), bf_hi(xv[i].x), bf_lo(xv[i].y), bf_hi(xv[i].y),
                    bf_lo(xv[i].z), bf_hi(xv[i].z), bf_lo(xv[i].w), bf_hi(xv[i].w)};
      float o[8];
      if (__any_sync(0xffffffffu, turn)) {  // a warp of V heads only copies
        float ss = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, d);
        if (turn && gain != nullptr) {
          const float inv = rsqrtf(ss * (1.0f / kAttnD) + a.eps);  // within 2^-22; the one rounding at the end is 2^-8
          const uint4 gv = ld128(gain + 8 * j);
          const uint32_t g2[4] = {gv.x, gv.y, gv.z, gv.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[2 * e] = x[2 * e] * inv * bf_lo(g2[e]);
            x[2 * e + 1] = x[2 * e + 1] * inv * bf_hi(g2[e]);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float other = __shfl_xor_sync(0xffffffffu, x[e], 8);
          const float c = (e & 1) ? bf_hi(c2[e >> 1]) : bf_lo(c2[e >> 1]);
          const float s = (e & 1) ? bf_hi(s2[e >> 1]) : bf_lo(s2[e >> 1]);
          o[e] = fmaf(x[e], c, other * s);  // s carries the sign
        }
      }
      if (h >= heads) continue;
      const uint4 ov = turn ? make_uint4(pack_bf16(o[0], o[1]), pack_bf16(o[2], o[3]), pack_bf16(o[4], o[5]),
                                         pack_bf16(o[6], o[7]))
                            : xv[i];
      bf16* dst;
      if (h < a.Hq) {
        dst = a.q_out + ((size_t)t * a.Hq + h) * kAttnD;
      } else {
        if (!page_ok) continue;
        const int kh = turn ? h - a.Hq : h - a.Hq - a.Hkv;
        bf16* pool = turn ? a.k_pages : a.v_pages;
        dst = pool + ((((size_t)page * a.Hkv + kh) << a.b.page_log2) + slot) * kAttnD;
      }
      *reinterpret_cast<uint4*>(dst + 8 * j) = ov;
    }
  }
}

}  // namespace qb
