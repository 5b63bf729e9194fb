// paged_decode.cuh — attention of few query rows over a paged cache (decode
// and short verify rows: at most 16 query rows per KV head and sequence).
//
//   o_r = sum_c 2^(s_rc - m) v_c / sum_c 2^(s_rc - m),
//   s_rc = (q_r . k_c) log2(e) / sqrt(128) over the keys c that row r sees:
//   c <= p_r and (no window, or c > p_r - window, or c < sinks)
//
// Bound by the bytes of K and V: 64 sequences of 130 to 16384 keys (1.8 GB)
// take 279 us, the copy rate. Work = 64-key tiles of every (sequence, KV head),
// laid out in one line of `total` places, two of them without a tile before each
// unit (sequence, head) for its start and end (120 sequences of up to 900 keys: 65
// us without them, 49 with two, 51 with four); CTA i of E takes the places
// [i total / E, (i + 1) total / E), so ragged lengths cost no balance: a CTA
// finishes one unit and goes on with the next. A unit cut by
// a CTA border leaves (m, l, O) of each piece in the workspace, and the CTA
// that draws the unit's last ticket joins them in order; a CTA has at most two
// such pieces, its first and its last, which bounds the workspace whatever the
// batch.
//  * warp 4: TMA. A tile's K and V come as boxes of min(page, 64) rows x 64
//    dims (128-byte swizzle), one per lane, into a 3-slot ring of 32 KB; boxes
//    without a key that some row sees are not read (their pages may have been
//    given back), and their V rows are cleared, since 0 * NaN is NaN.
//  * warps 0-3: scores of 16 keys each (rows on the MMA's M = 16: one code path
//    for every group size), maximum over the warps through shared memory, P
//    (bf16) to shared memory, then O of 32 dims each over all 64 keys, so that
//    a unit's end needs no exchange of O between the warps.
// fp32 scores, statistics and O; P is rounded to bf16 for its product, as on
// the framework's other attention paths (its error averages out over the keys).
#pragma once
#include "paged.cuh"
#include "verify_attention.cuh"

namespace qb {

constexpr int kPdKeys = 64;
constexpr int kPdRows = 16;
constexpr int kPdStages = 3;
constexpr int kPdWarps = 4;
constexpr int kPdThreads = (kPdWarps + 1) * 32;
constexpr int kPdStageBytes = 4 * kAttnSubTile;  // K lo, K hi, V lo, V hi
constexpr int kPdPStride = kPdKeys * 2 + 16;     // bytes of a P row; 16 more keep ldmatrix free of conflicts
constexpr int kPdCtasPerSm = 2;
constexpr int kPdMinTiles = 1;                   // fewest tiles of a CTA: 1 of 16 in 24 us, 2 in 29, 4 in 40 (six short rows)

constexpr int kPdUnitCost = 2;  // what beginning and ending a unit takes, in key tiles: its place in the line

// Where a finished row goes: out (bf16), or out32 / lse32 (normalised fp32 and
// log-sum-exp in base 2, for a later join); base32 / base_lse: a part of the
// row's keys already attended to, joined in.
struct RowSink {
  bf16* out;
  float* out32;
  float* lse32;
  const float* base32;
  const float* base_lse;
};

struct PagedAttnArgs {
  PagedBatch b;
  const bf16* q;  // [tokens][Hq][128]
  int Hq, Hkv, G;
  RowSink sink;
  float* part_o;      // [2 CTAs][rows][128]
  float* part_ml;     // [2 CTAs][rows][2]
  unsigned* tickets;  // one per CTA: of the unit that its last piece begins
  int* err;
};

// Factors that turn a row's unnormalised O (maximum m, sum l) into its result:
// result = O * own + base * other; a row that saw nothing gives 0.
struct RowScale {
  float own, other, lse;
};
__device__ __forceinline__ RowScale row_scale(float m, float l, bool has_base, float base_lse) {
  RowScale r;
  if (!has_base || base_lse == -INFINITY) {
    r.own = l > 0.f ? 1.0f / l : 0.f;
    r.other = 0.f;
    r.lse = l > 0.f ? m + log2f(l) : -INFINITY;
    return r;
  }
  const float lse = l > 0.f ? m + log2f(l) : -INFINITY;
  const float top = fmaxf(lse, base_lse);
  const float wo = exp2f(lse - top), wb = exp2f(base_lse - top);
  r.own = l > 0.f ? wo / (l * (wo + wb)) : 0.f;
  r.other = wb / (wo + wb);
  r.lse = top + log2f(wo + wb);
  return r;
}

__device__ __forceinline__ bool named_barrier_and(int id, int threads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.and.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(threads), "r"((uint32_t)v)
      : "memory");
  return r != 0;
}

// The CTA of E that owns tile x of `total`, and the first tile of CTA i.
__device__ __forceinline__ int tile_owner(long long x, long long total, int E) {
  return (int)(((x + 1) * E - 1) / total);
}
__device__ __forceinline__ long long tile_begin(int i, long long total, int E) { return (long long)i * total / E; }

// Joins the pieces that CTAs cf .. cl left of a unit, in order, and writes its
// rows: warp w the rows w, w + 4, ..., R of them at once, a lane 4 dims. Bound by
// the latency of the loads (L2), so 8 / R pieces are loaded at a time.
template <int R>
__device__ __forceinline__ void join_pieces(const PagedAttnArgs& a, int warp, int lane, int rows, int cf, int cl,
                                            int first_slot, int q0, int g) {
  constexpr int U = 8 / R;
  auto piece = [&](int c, int i) {
    return (size_t)(2 * c + (c == cf ? first_slot : 0)) * kPdRows + warp + kPdWarps * i;  // the later ones are their CTAs' first
  };
  float top[R], lsum[R];
  float4 acc[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    top[i] = -INFINITY;
    lsum[i] = 0.f;
    acc[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  for (int c = cf + lane; c <= cl; c += 32)
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (warp + kPdWarps * i < rows) top[i] = fmaxf(top[i], __ldcg(a.part_ml + piece(c, i) * 2));
#pragma unroll
  for (int i = 0; i < R; ++i) top[i] = warp_max(top[i]);
  for (int c0 = cf; c0 <= cl; c0 += U) {
    float2 ml[U][R];
    float4 ov[U][R];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const bool in = c0 + u <= cl && warp + kPdWarps * i < rows;
        ml[u][i] = in ? __ldcg(reinterpret_cast<const float2*>(a.part_ml + piece(c0 + u, i) * 2)) : make_float2(-INFINITY, 0.f);
        ov[u][i] = in ? __ldcg(reinterpret_cast<const float4*>(a.part_o + piece(c0 + u, i) * kAttnD + 4 * lane))
                      : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const float w = exp2f(ml[u][i].x - (top[i] == -INFINITY ? 0.f : top[i]));
        lsum[i] = fmaf(ml[u][i].y, w, lsum[i]);
        acc[i].x = fmaf(ov[u][i].x, w, acc[i].x);
        acc[i].y = fmaf(ov[u][i].y, w, acc[i].y);
        acc[i].z = fmaf(ov[u][i].z, w, acc[i].z);
        acc[i].w = fmaf(ov[u][i].w, w, acc[i].w);
      }
  }
  const bool has_base = a.sink.base32 != nullptr;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = warp + kPdWarps * i;
    if (r >= rows) continue;
    const size_t row = (size_t)(q0 + r / a.G) * a.Hq + g * a.G + r % a.G;
    const RowScale rs = row_scale(top[i], lsum[i], has_base, has_base ? a.sink.base_lse[row] : 0.f);
    float4 v = make_float4(acc[i].x * rs.own, acc[i].y * rs.own, acc[i].z * rs.own, acc[i].w * rs.own);
    if (has_base) {
      const float4 bv = *reinterpret_cast<const float4*>(a.sink.base32 + row * kAttnD + 4 * lane);
      v.x = fmaf(bv.x, rs.other, v.x);
      v.y = fmaf(bv.y, rs.other, v.y);
      v.z = fmaf(bv.z, rs.other, v.z);
      v.w = fmaf(bv.w, rs.other, v.w);
    }
    uint2 ob;
    ob.x = pack_bf16(v.x, v.y);
    ob.y = pack_bf16(v.z, v.w);
    *reinterpret_cast<uint2*>(a.sink.out + row * kAttnD + 4 * lane) = ob;
  }
}

__host__ inline size_t pd_smem_bytes() {
  return 1024 + (size_t)kPdStages * kPdStageBytes + kPdRows * kPdPStride + 2 * kPdWarps * kPdRows * 4 +
         2 * kPdStages * 8 + 64 + (kPagedMaxSeqs + 1) * 4 + 4 + kPagedMaxSeqs * 8;
}

// Sum of v over the block.
__device__ __forceinline__ int block_count(int v, int* warp_tot) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) warp_tot[threadIdx.x >> 5] = v;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) all += warp_tot[w];
  return all;
}

__global__ void __launch_bounds__(kPdThreads, kPdCtasPerSm)
    paged_decode_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                        const PagedAttnArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ps = ring + kPdStages * kPdStageBytes;                        // P [16][64]
  float* wmax = reinterpret_cast<float*>(ps + kPdRows * kPdPStride);     // [warp][row]
  float* wsum = wmax + kPdWarps * kPdRows;                               // [warp][row]
  uint64_t* full = reinterpret_cast<uint64_t*>(wsum + kPdWarps * kPdRows);
  uint64_t* empty = full + kPdStages;
  int* flag = reinterpret_cast<int*>(empty + kPdStages);                 // [0]: this CTA joins the unit's pieces
  int* warp_tot = flag + 1;                                              // [5]
  int* pref = flag + 16;                                                 // [n_seqs + 1] tiles before each sequence
  // First row and queries (at most 16) in one word, and keys, of each sequence: a new one costs no trip to memory.
  int2* seqs = reinterpret_cast<int2*>(pref + kPagedMaxSeqs + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const PagedBatch& b = a.b;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPdStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kPdWarps);
    }
    fence_mbar_init();
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
  }
  pdl_wait();
  pdl_trigger();

  // Tiles of every sequence, summed up (each CTA for itself).
  int carry = 0, live = 0;  // live: this thread's sequences with rows
  for (int s0 = 0; s0 < b.n_seqs; s0 += kPdThreads) {
    const int s = s0 + threadIdx.x;
    int cnt = 0;
    if (s < b.n_seqs) {
      const SeqSpan sp = paged_seq(b, s, a.err);
      seqs[s] = make_int2(sp.q0 | sp.n << 25, sp.kv);
      if (sp.n > 0) {
        cnt = tile_span<kPdKeys>(sp.kv - sp.n, sp.kv, b.window, b.sinks).count + kPdUnitCost;
        ++live;
      }
    }
    int v = cnt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) warp_tot[warp] = v;
    __syncthreads();
    int before = carry, all = 0;
#pragma unroll
    for (int w = 0; w < kPdThreads / 32; ++w) {
      if (w < warp) before += warp_tot[w];
      all += warp_tot[w];
    }
    if (s < b.n_seqs) pref[s + 1] = before + v;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) pref[0] = 0;
  __syncthreads();

  const int total = carry * a.Hkv;  // the host keeps the line below 2^31 places
  const int tiles = carry - kPdUnitCost * block_count(live, warp_tot);
  const int E = min((int)gridDim.x, max(1, tiles * a.Hkv / kPdMinTiles));
  const int me = blockIdx.x;
  if (me >= E || total == 0) return;
  const int t_begin = (int)tile_begin(me, total, E), t_end = (int)tile_begin(me + 1, total, E);
  int seq0;  // the sequence of tile t_begin: the last with pref[seq] * Hkv <= t_begin and tiles of its own
  {
    int lo = 0, hi = b.n_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (pref[mid + 1] * a.Hkv > t_begin) hi = mid;
      else lo = mid + 1;
    }
    seq0 = lo;
  }
  const int br = min(1 << b.page_log2, kPdKeys);  // rows of a box

  if (warp == kPdWarps) {
    // ---------------------------------------------------------------- producer
    const int kind = lane & 3, box = lane >> 2;
    const int nbox = kPdKeys / br;
    int issued = 0;
    bool ok = true;
    int seq = seq0;
    for (int t = t_begin; t < t_end && ok; ++seq) {
      const int places = pref[seq + 1] - pref[seq];  // of one head in the line
      if (places == 0) continue;
      const SeqSpan sp = {seqs[seq].x & 0x1ffffff, seqs[seq].x >> 25, seqs[seq].y};
      const TileSpan ts = tile_span<kPdKeys>(sp.kv - sp.n, sp.kv, b.window, b.sinks);
      const int base = pref[seq] * a.Hkv;
      const int stop = min(t_end, base + places * a.Hkv);
      // page of this lane's box of the tile at k, or -1
      auto page_of = [&](int k) {
        const int c0 = (k < ts.n_sink ? k : k - ts.n_sink + ts.lo_tile) * kPdKeys + box * br;
        if (box >= nbox || c0 >= sp.kv || !(b.window == 0 || c0 + br > ts.lo || c0 < b.sinks)) return -1;
        const int page = b.page_table[(size_t)seq * b.table_width + (c0 >> b.page_log2)];
        if (page < 0 || page >= b.num_pages) {
          report_error(a.err, DEV_BAD_PAGE);
          return -1;
        }
        return page;
      };
      int k = max(0, (t - base) % places - kPdUnitCost);
      int page = page_of(k);
      while (t < stop && ok) {
        const int g = (t - base) / places;
        const int x0 = t - base - g * places, x1 = min(places, x0 + (t_end - t));
        const int k1 = max(0, x1 - kPdUnitCost);
        for (k = max(0, x0 - kPdUnitCost); k < k1; ++k) {
          const int c0 = (k < ts.n_sink ? k : k - ts.n_sink + ts.lo_tile) * kPdKeys + box * br;
          const int s = issued % kPdStages;
          const int now = page;
          page = page_of(k + 1 == places - kPdUnitCost ? 0 : k + 1);  // its load runs while the slot is waited for
          if (issued >= kPdStages)
            ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], ((issued / kPdStages) - 1) & 1, a.err, DEV_TIMEOUT_ATTN_EMPTY));
          if (!ok) break;
          const uint32_t need = __ballot_sync(0xffffffffu, now >= 0);
          if (lane == 0) mbar_arrive_expect_tx(&full[s], (uint32_t)__popc(need) * br * 128);
          __syncwarp();
          if (now >= 0) {
            const int y = ((now * a.Hkv + g) << b.page_log2) + (c0 & ((1 << b.page_log2) - 1));
            tma_load_2d(ring + s * kPdStageBytes + kind * kAttnSubTile + box * br * 128, kind < 2 ? &tmk : &tmv,
                        64 * (kind & 1), y, &full[s]);
          }
          ++issued;
        }
        t += x1 - x0;
      }
    }
    // keep shared memory alive until every issued copy has landed
    for (int i = max(0, issued - kPdStages); i < issued; ++i) mbar_wait(&full[i % kPdStages], (i / kPdStages) & 1, nullptr, 0);
    return;
  }

  // ------------------------------------------------------------------ consumers
  const int r_lo = lane >> 2, cq = (lane & 3) * 2;  // this lane's rows r_lo, r_lo + 8 and column pair
  const float scale = kLog2e * 0.08838834764831845f;  // log2(e) / sqrt(128)
  int used = 0;
  int seq = seq0;
  for (int t = t_begin; t < t_end; ++seq) {
    const int places = pref[seq + 1] - pref[seq], n_tiles = places - kPdUnitCost;
    if (places == 0) continue;
    const SeqSpan sp = {seqs[seq].x & 0x1ffffff, seqs[seq].x >> 25, seqs[seq].y};
    const TileSpan ts = tile_span<kPdKeys>(sp.kv - sp.n, sp.kv, b.window, b.sinks);
    const int base = pref[seq] * a.Hkv;
    const int stop = min(t_end, base + places * a.Hkv);
    const int rows = sp.n * a.G;
    int pos[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) pos[h] = r_lo + 8 * h < rows ? sp.kv - sp.n + (r_lo + 8 * h) / a.G : -1;
    const int p_first = sp.kv - sp.n;
    while (t < stop) {
      const int g = (t - base) / places;
      const int u0 = base + g * places;  // the unit's place in the line: first those without a tile
      const int x0 = t - u0, x1 = min(places, x0 + (t_end - t));
      const int k0 = max(0, x0 - kPdUnitCost), k1 = max(0, x1 - kPdUnitCost);
      if (k0 == k1) {
        t += x1 - x0;
        continue;
      }
      // Q as the MMA's A operand, straight from memory
      uint32_t qa[8][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = r_lo + 8 * h;
        const bf16* src = a.q + ((size_t)(sp.q0 + r / a.G) * a.Hq + g * a.G + r % a.G) * kAttnD + cq;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          qa[ks][h] = r < rows ? *reinterpret_cast<const uint32_t*>(src + 16 * ks) : 0u;
          qa[ks][2 + h] = r < rows ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 8) : 0u;
        }
      }
      float o[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

      for (int k = k0; k < k1; ++k, ++used) {
        const int s = used % kPdStages;
        uint8_t* st = ring + s * kPdStageBytes;
        const int c0 = (k < ts.n_sink ? k : k - ts.n_sink + ts.lo_tile) * kPdKeys;
        const bool landed = mbar_wait(&full[s], (used / kPdStages) & 1, a.err, DEV_TIMEOUT_ATTN_FULL);
        // scores of keys c0 + 16 warp .. + 15
        float sc[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][e] = 0.f;
        const int key = 16 * warp + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          uint32_t kb[4];
          const int ch = ((ks & 3) << 1) + ((lane >> 3) & 1);
          ldsm_x4(kb, st + (ks >> 2) * kAttnSubTile + swz(key, ch));
          mma_bf16_16816(sc[0], qa[ks], kb[0], kb[1]);
          mma_bf16_16816(sc[1], qa[ks], kb[2], kb[3]);
        }
        // Only tiles at an edge hold keys that some row does not see.
        const bool edge = !(c0 + kPdKeys - 1 <= p_first &&
                            (b.window == 0 || (long long)c0 > (long long)sp.kv - 1 - b.window || c0 + kPdKeys <= b.sinks));
        if (edge) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int c = c0 + 16 * warp + 8 * i + cq + (e & 1), p = pos[e >> 1];
              const bool seen = c <= p && (b.window == 0 || (long long)c > (long long)p - b.window || c < b.sinks);
              sc[i][e] = seen ? sc[i][e] : -INFINITY;
            }
          // V rows that no row sees: P is 0 there, and they must not be NaN
          const int vr = threadIdx.x >> 1, c = c0 + vr;
          if (c >= sp.kv || (b.window > 0 && c < ts.lo && c >= b.sinks)) {
            uint8_t* vt = st + (2 + (threadIdx.x & 1)) * kAttnSubTile + vr * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(vt + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        float mx[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mx[h] = fmaxf(fmaxf(sc[0][2 * h], sc[0][2 * h + 1]), fmaxf(sc[1][2 * h], sc[1][2 * h + 1]));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
          mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        }
        if ((lane & 3) == 0) {
          wmax[warp * kPdRows + r_lo] = mx[0];
          wmax[warp * kPdRows + r_lo + 8] = mx[1];
        }
        if (!named_barrier_and(1, kPdWarps * 32, landed)) return;  // every warp leaves together
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float top = m[h];
#pragma unroll
          for (int w = 0; w < kPdWarps; ++w) top = fmaxf(top, wmax[w * kPdRows + r_lo + 8 * h] * scale);
          const float mu = top == -INFINITY ? 0.f : top;  // a row that has seen nothing yet
          const float corr = exp2f(m[h] - mu);            // 2^-inf = 0
          m[h] = top;
          float p[4];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 2; ++e) p[2 * i + e] = exp2f(fmaf(sc[i][2 * h + e], scale, -mu));
          l[h] = l[h] * corr + ((p[0] + p[1]) + (p[2] + p[3]));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            o[i][2 * h] *= corr;
            o[i][2 * h + 1] *= corr;
          }
          uint8_t* pr = ps + (r_lo + 8 * h) * kPdPStride + (16 * warp + cq) * 2;
          *reinterpret_cast<uint32_t*>(pr) = pack_bf16(p[0], p[1]);
          *reinterpret_cast<uint32_t*>(pr + 16) = pack_bf16(p[2], p[3]);
        }
        named_barrier(1, kPdWarps * 32);
        // O of dims 32 warp .. + 31 over the tile's 64 keys
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          uint32_t pa[4];
          ldsm_x4(pa, ps + (lane & 15) * kPdPStride + ks * 32 + (lane >> 4) * 16);
#pragma unroll
          for (int dp = 0; dp < 2; ++dp) {
            uint32_t vb[4];
            const int vkey = 16 * ks + (lane & 15);
            const int dch = warp * 4 + dp * 2 + (lane >> 4);  // 8-dim chunk
            ldsm_x4_t(vb, st + (2 + (dch >> 3)) * kAttnSubTile + swz(vkey, dch & 7));
            mma_bf16_16816(o[2 * dp], pa, vb[0], vb[1]);
            mma_bf16_16816(o[2 * dp + 1], pa, vb[2], vb[3]);
          }
        }
        if (edge) fence_proxy_async_smem();  // the cleared rows, before the next copy into the slot
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }

      // ---- the piece's row sums, then the rows themselves
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      }
      if ((lane & 3) == 0) {
        wsum[warp * kPdRows + r_lo] = l[0];
        wsum[warp * kPdRows + r_lo + 8] = l[1];
      }
      named_barrier(1, kPdWarps * 32);
      const bool whole = k0 == 0 && k1 == n_tiles;
      const int slot = 2 * me + (t == t_begin ? 0 : 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = r_lo + 8 * h;
        if (r >= rows) continue;
        const float lsum = (wsum[r] + wsum[kPdRows + r]) + (wsum[2 * kPdRows + r] + wsum[3 * kPdRows + r]);
        if (whole) {
          const size_t row = (size_t)(sp.q0 + r / a.G) * a.Hq + g * a.G + r % a.G;
          const bool has_base = a.sink.base32 != nullptr;
          const RowScale rs = row_scale(m[h], lsum, has_base, has_base ? a.sink.base_lse[row] : 0.f);
          const int d = 32 * warp + cq;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x = o[i][2 * h] * rs.own, y = o[i][2 * h + 1] * rs.own;
            if (has_base) {
              const float2 bv = *reinterpret_cast<const float2*>(a.sink.base32 + row * kAttnD + d + 8 * i);
              x = fmaf(bv.x, rs.other, x);
              y = fmaf(bv.y, rs.other, y);
            }
            *reinterpret_cast<uint32_t*>(a.sink.out + row * kAttnD + d + 8 * i) = pack_bf16(x, y);
          }
        } else {
          float* po = a.part_o + ((size_t)slot * kPdRows + r) * kAttnD + 32 * warp + cq;
#pragma unroll
          for (int i = 0; i < 4; ++i) *reinterpret_cast<float2*>(po + 8 * i) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
          if (warp == 0 && (lane & 3) == 0) {
            a.part_ml[((size_t)slot * kPdRows + r) * 2] = m[h];
            a.part_ml[((size_t)slot * kPdRows + r) * 2 + 1] = lsum;
          }
        }
      }
      if (!whole) {
        const int cf = tile_owner(u0 + kPdUnitCost, total, E), cl = tile_owner(u0 + places - 1, total, E);
        named_barrier(1, kPdWarps * 32);
        if (threadIdx.x == 0) {
          const unsigned old = atomic_add_acq_rel_gpu(&a.tickets[cf], 1u);
          const bool last = old == (unsigned)(cl - cf);
          if (last) a.tickets[cf] = 0u;
          flag[0] = last;
        }
        named_barrier(1, kPdWarps * 32);
        if (flag[0]) {
          const int slot0 = tile_begin(cf, total, E) >= u0 ? 0 : 1;
          // one, two or four rows a warp at once: eight pieces' loads on their way either way
          if (rows <= kPdWarps) join_pieces<1>(a, warp, lane, rows, cf, cl, slot0, sp.q0, g);
          else if (rows <= 2 * kPdWarps) join_pieces<2>(a, warp, lane, rows, cf, cl, slot0, sp.q0, g);
          else join_pieces<4>(a, warp, lane, rows, cf, cl, slot0, sp.q0, g);
        }
      }
      t += x1 - x0;
    }
  }
}

}  // namespace qb
