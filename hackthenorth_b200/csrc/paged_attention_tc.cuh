// paged_attention_tc.cuh — attention of many query rows over a paged cache on
// the tcgen05 tensor cores: prompts, chunks of prompts, verify rows, mixed
// batches, and the pass over a prefix that a whole batch shares.
//
// The formula and the masks are those of paged_decode.cuh. A unit is up to 256
// query rows of one sequence (two M = 128 tiles of 128 / G tokens with the G
// query heads of one KV head) against the 64-key tiles that some of its rows
// see. As there, the units' tiles form one line which is cut evenly over the
// CTAs (one per SM), a unit's own start and end counted as four tiles (without
// that the CTAs with many short units of a causal prompt finished last: 746 us
// for 8100 tokens of 32/8 heads at the power cap, 618 with two tiles, 582 with
// four, 588 with seven). A cut
// unit leaves (m, l, O) of its pieces in the workspace, and paged_join_kernel
// joins them: with 256 rows a piece is 128 KB, too much for one CTA to join
// behind the others.
//
// Bound, where every key tile meets 256 rows, by the softmax and the MMAs
// together (about 2000 cycles a key tile; the MMAs alone take 1280: 384 for S,
// whose operands come from shared memory, and 256 for P.V of each M tile), and
// by the cache's bytes below that. 8100 prompt tokens: 545 us (0.99 PFLOP/s) with
// pauses between the calls, 578 (0.93) call after call, at the power cap.
//  * warp 0: TMA. Q tiles (3D map, 128-byte swizzle) and K and V tiles of
//    16 KB, a box per page, into four slots each.
//  * warps 1 and 3: the MMAs of M tile 0 and 1. S_t = Q_t . K^T goes to one of
//    two buffers of 64 TMEM columns in turn, so that the softmax finds the next
//    one ready; P_t (bf16) comes back over the first half of its S, and O_t +=
//    P_t . V reads it from there into columns 256 + 128 t. S_t of the tile after
//    next follows P_t . V into the same buffer: issue order is the order of
//    execution.
//  * warps 4-7 and 8-11: softmax of M tile 0 and 1, a thread per row. The
//    reference maximum only moves when a row's maximum grows by more than 8 (P
//    stays below 2^8 and keeps its relative precision), so O is seldom rescaled.
//    Both groups tend to reach their exponentials together, so every fourth
//    pair is computed on the FMA pipe, to the MUFU's precision: 545 us for the
//    8100 tokens against 568 without it, 556 and 552 with every third and fifth
//    pair; at the power cap 578 to 581 without, with every fourth and fifth.
//  * warp 2: walks the CTA's pieces of units ahead of the others and hands them
//    over through a ring of 4 (the lookups and divisions of a new piece took 3 us
//    of every role's time when each made them itself); and waits for K and V on
//    the MMA warps' behalf.
// Every wait is bounded; on failure an error is recorded, the roles stop, and
// TMEM is released after the MMAs that were issued.
#pragma once
#include "paged_decode.cuh"
#include "prefill_attention_tc.cuh"

namespace qb {

constexpr int kPtKeys = 64;
constexpr int kPtRows = 256;
constexpr int kPtThreads = 12 * 32;
constexpr int kPtTile = 128 * 128 * 2;         // a Q tile: 32 KB, dims 0-63 then 64-127
constexpr int kPtKvTile = kPtKeys * 128 * 2;   // a K or V tile: 16 KB, likewise
constexpr int kPtSlots = 4;                    // ring slots of each
constexpr int kPtMaxUnits = 4096;
constexpr int kPagedMaxTcCtas = 1024;
constexpr int kPtMinTiles = 2;
constexpr int kPtUnitCost = 4;  // what beginning and ending a unit takes, in key tiles: its place in the line

constexpr int kPtPieces = 4;
constexpr int kPtPolyEvery = 4;  // every fourth pair of P comes from exp2_poly, the rest from the MUFU

// What a CTA does next: the key tiles [k0, k1) of a unit (a role's whole state).
struct PtPiece {
  int seq, token0, tokens, p_first, hi, lo_tile, n_sink, lo;
  int head, k0, k1;
  int whole;  // the unit in one piece
  int first;  // the CTA's first piece: its workspace slot is the first
  int last;   // of a cut unit's first piece: the CTA of the last one; else -1
  int pad[2];
};
static_assert(sizeof(PtPiece) == 64, "read as four 16-byte words");

struct PtUnit {  // a cut unit, for the join
  int token0, tokens, head, last, first_slot, valid;
};

struct PagedTcArgs {
  PagedBatch b;
  int Hq, Hkv, G, max_units;
  RowSink sink;
  float* part_o;   // [2 CTAs][256][128]
  float* part_ml;  // [2 CTAs][256][2]
  PtUnit* cut;     // [CTAs]
  int* err;
};

__host__ inline size_t pt_smem_bytes(int max_units) {
  return 1024 + 2 * (size_t)kPtTile + 2 * kPtSlots * (size_t)kPtKvTile + 512 + kPtPieces * sizeof(PtPiece) + (size_t)(4 * kPagedMaxSeqs + 1 + max_units + 1) * 4;
}

// The MMAs as the whole warp runs them: `lead` (one lane) issues. Kept free of
// divergence, descriptors and addresses stay in uniform registers, which the
// instruction takes its operands from; in a lane's own branch every operand is
// moved there anew.
__device__ __forceinline__ bool elect_lane() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void tc_mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, l;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 l, %5, 0;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, l;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 l, %5, 0;\n\t"
      "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void tc_commit_by(uint32_t lead, uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred l;\n\tsetp.ne.b32 l, %1, 0;\n\t"
      "@l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}
// 32 columns of this warp's lanes without the wait (tc_ld_wait follows).
__device__ __forceinline__ void tc_ld32_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tc_st32_async(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tc_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The wait, and a use of the registers after it, so that no use moves above.
template <int N>
__device__ __forceinline__ void tc_ld_wait(uint32_t (&r)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

// 32 bytes to a 32-byte aligned address in one store.
__device__ __forceinline__ void st_global_32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// mbar_wait with a short path for the polls that the kernel's rarer roles make:
// their code is fetched anew each time, so its length counts.
__device__ __forceinline__ bool pt_wait(uint64_t* bar, uint32_t parity, int* err, int code) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_timer_ns();
#pragma unroll 1
  while (!mbar_try_wait(bar, parity))
    if (global_timer_ns() - t0 > kWaitLimitNs) {
      report_error(err, code);
      return false;
    }
  return true;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// Two fp32 values in one register pair, for sm_100's packed arithmetic.
__device__ __forceinline__ uint64_t f32x2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x of two values (below 2^7) on the FMA pipe: x = n + f with n the nearest
// integer, 2^f on [-1/2, 1/2] by 1 + f q(f) with a quartic q (fitted to the least
// largest relative error: 2^-22.5 as evaluated in fp32, and none at whole x),
// times 2^n from n's bits. The multiplication, unlike an addition to the
// exponent, keeps a NaN, and gives exactly 0 for x at or below -127, where 2^n's
// bits are 0: a masked key's V may be 2^128, so any rest of its weight would show.
__device__ __forceinline__ void exp2_poly(uint64_t x, float& p0, float& p1) {
  constexpr float kC1 = 0.69314700f, kC2 = 0.24022242f, kC3 = 0.055507336f, kC4 = 0.0096715130f, kC5 = 0.0013264727f;
  constexpr float kRound = 12582912.f + 127.f;  // 1.5 * 2^23, and the exponent's bias: the sum's low bits are n + 127
  float a, b;
  unpack_f32x2(x, a, b);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(a) : "f"(-127.f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(b) : "f"(-127.f));
  x = f32x2(a, b);
  const uint64_t n = add_f32x2(x, f32x2(kRound, kRound));
  const uint64_t f = add_f32x2(x, fma_f32x2(n, f32x2(-1.f, -1.f), f32x2(kRound, kRound)));
  uint64_t p = fma_f32x2(f, f32x2(kC5, kC5), f32x2(kC4, kC4));
  p = fma_f32x2(p, f, f32x2(kC3, kC3));
  p = fma_f32x2(p, f, f32x2(kC2, kC2));
  p = fma_f32x2(p, f, f32x2(kC1, kC1));
  p = fma_f32x2(p, f, f32x2(1.f, 1.f));
  float n0, n1;
  unpack_f32x2(n, n0, n1);
  const float s0 = __int_as_float(__float_as_int(n0) << 23), s1 = __int_as_float(__float_as_int(n1) << 23);
  unpack_f32x2(mul_f32x2(p, f32x2(s0, s1)), p0, p1);
}

// A word with its lowest n bits set (n clamped to 0..32).
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Unit u of the launch: its sequence, tokens and key tiles.
struct TcUnit {
  int seq, token0, tokens, p_first, kv, hi;  // p_first: position of token0; hi: one past the last key a row sees
  TileSpan ts;
};
__device__ __forceinline__ TcUnit tc_unit(const PagedBatch& b, const SeqSpan* seqs, const int* seq_unit, int u,
                                          int per_unit) {
  int lo = 0, hi = b.n_seqs - 1;
  while (lo < hi) {  // the sequence of unit u: the first with seq_unit[seq + 1] > u
    const int mid = (lo + hi) >> 1;
    if (seq_unit[mid + 1] > u) hi = mid;
    else lo = mid + 1;
  }
  const SeqSpan sp = seqs[lo];
  TcUnit r;
  r.seq = lo;
  const int i0 = (u - seq_unit[lo]) * per_unit;
  r.token0 = sp.q0 + i0;
  r.tokens = min(per_unit, sp.n - i0);
  r.kv = sp.kv;
  if (b.q_start == nullptr) {  // every row sees all keys
    r.p_first = sp.kv - 1;
    r.hi = sp.kv;
  } else {
    r.p_first = sp.kv - sp.n + i0;
    r.hi = r.p_first + r.tokens;
  }
  r.ts = tile_span<kPtKeys>(r.p_first, r.hi, b.window, b.sinks);
  return r;
}

// Inclusive sum of v over the block's threads on top of carry (updated).
__device__ __forceinline__ int block_scan(int v, int* warp_tot, int& carry) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  if (lane == 31) warp_tot[warp] = v;
  __syncthreads();
  int before = carry, all = 0;
  for (int w = 0; w < (int)blockDim.x / 32; ++w) {
    if (w < warp) before += warp_tot[w];
    all += warp_tot[w];
  }
  carry += all;
  __syncthreads();
  return before + v;
}

__global__ void __launch_bounds__(kPtThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                    const __grid_constant__ CUtensorMap tmv, const PagedTcArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* qs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* kring = qs + 2 * kPtTile;
  uint8_t* vring = kring + kPtSlots * kPtKvTile;
  uint64_t* bars = reinterpret_cast<uint64_t*>(vring + kPtSlots * kPtKvTile);
  uint64_t* kv_full = bars;            // [2][slots]: K, V
  uint64_t* kv_empty = bars + 8;       // [2][slots]
  uint64_t* q_full = bars + 16;        // [2]
  uint64_t* q_empty = bars + 18;       // [2]
  uint64_t* s_full = bars + 20;        // [2 M tiles][2 buffers]
  // of S's buffers too: P may be a tile ahead of its MMAs, which are then two phases of one barrier behind
  uint64_t* p_full = bars + 24;        // [2][2]
  uint64_t* o_done = bars + 28;        // [2][2]
  uint64_t* done = bars + 32;          // [2]
  uint64_t* piece_full = bars + 34;    // [4]
  uint64_t* piece_empty = bars + 38;   // [4]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 42);
  volatile int* flags = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* warp_tot = reinterpret_cast<int*>(tmem_slot + 2);  // [12]
  PtPiece* pieces = reinterpret_cast<PtPiece*>(bars + 64);
  SeqSpan* seqs = reinterpret_cast<SeqSpan*>(pieces + kPtPieces);
  int* seq_unit = reinterpret_cast<int*>(seqs + kPagedMaxSeqs);  // [n_seqs + 1] units before each sequence
  int* unit_tile = seq_unit + kPagedMaxSeqs + 1;          // [units + 1] the line before each unit (of one head)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const PagedBatch& b = a.b;
  const int RH = 128 / a.G;  // tokens per M tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2 * kPtSlots; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 2);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      for (int i = 2 * t; i < 2 * t + 2; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&p_full[i], 5);
        mbar_init(&o_done[i], 1);
      }
      mbar_init(&done[t], 1);
    }
    for (int i = 0; i < kPtPieces; ++i) {
      mbar_init(&piece_full[i], 1);
      mbar_init(&piece_empty[i], 12);  // producer, 2 MMA warps, warp 2, 8 softmax warps
    }
    fence_mbar_init();
    flags[0] = 0;
    seq_unit[0] = 0;
    unit_tile[0] = 0;
    prefetch_tensormap(&tmq);
    prefetch_tensormap(&tmk);
    prefetch_tensormap(&tmv);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  pdl_trigger();

  // ---- the line of tiles
  int units = 0;
  for (int s0 = 0; s0 < b.n_seqs; s0 += kPtThreads) {
    const int s = s0 + threadIdx.x;
    const SeqSpan sp = s < b.n_seqs ? paged_seq(b, s, a.err) : SeqSpan{0, 0, 0};
    const int v = block_scan((sp.n + 2 * RH - 1) / (2 * RH), warp_tot, units);
    if (s < b.n_seqs) {
      seqs[s] = sp;
      seq_unit[s + 1] = v;
    }
  }
  __syncthreads();
  if (units > a.max_units) {  // sequences that overlap
    if (threadIdx.x == 0) report_error(a.err, DEV_BAD_BATCH);
    units = a.max_units;
  }
  int tiles = 0;
  for (int u0 = 0; u0 < units; u0 += kPtThreads) {
    const int u = u0 + threadIdx.x;
    const int v = block_scan(u < units ? tc_unit(b, seqs, seq_unit, u, 2 * RH).ts.count + kPtUnitCost : 0, warp_tot, tiles);
    if (u < units) unit_tile[u + 1] = v;
  }
  __syncthreads();
  const long long total = (long long)tiles * a.Hkv;
  const int E = (int)min((long long)gridDim.x, max(1ll, (total - (long long)units * a.Hkv * kPtUnitCost) / kPtMinTiles));
  const int me = blockIdx.x;
  const bool busy = me < E && total > 0;
  const long long t_begin = busy ? tile_begin(me, total, E) : 0, t_end = busy ? tile_begin(me + 1, total, E) : 0;
  if (threadIdx.x == 0) a.cut[me].valid = 0;
  __syncthreads();

  // Every role takes the same pieces in turn: f(piece), until an empty one. Lane 0 frees the entry.
  auto walk = [&](auto&& f, auto&& gave_up) {
    for (int i = 0;; ++i) {
      const int e = i % kPtPieces;
      if (!__all_sync(0xffffffffu, mbar_wait(&piece_full[e], (i / kPtPieces) & 1, a.err, DEV_TIMEOUT_ATTN_FULL))) {
        gave_up();
        return;
      }
      union {
        uint4 w[4];
        PtPiece p;
      } u;
#pragma unroll
      for (int j = 0; j < 4; ++j) u.w[j] = reinterpret_cast<const uint4*>(&pieces[e])[j];
      __syncwarp();
      if (lane == 0) mbar_arrive(&piece_empty[e]);
      if (u.p.k0 == u.p.k1 || !f(u.p)) return;
    }
  };
  auto tile_key = [&](const PtPiece& p, int k) { return (k < p.n_sink ? k : k - p.n_sink + p.lo_tile) * kPtKeys; };

  if (warp < 4) {
    if (warp == 0) {
      // -------------------------------------------------------------- producer
      const int br = min(1 << b.page_log2, kPtKeys), nbox = kPtKeys / br;
      const int kind = lane & 3, box = lane >> 2;
      int issued = 0, quse[2] = {0, 0};
      bool ok = true;
      walk([&](const PtPiece& un) {
        const int g = un.head, k0 = un.k0, k1 = un.k1;
        auto page_of = [&](int k) {
          const int c0 = tile_key(un, k) + box * br;
          if (k >= k1 || box >= nbox || c0 >= un.hi || !(b.window == 0 || c0 + br > un.lo || c0 < b.sinks)) return -1;
          const int page = b.page_table[(size_t)un.seq * b.table_width + (c0 >> b.page_log2)];
          if (page < 0 || page >= b.num_pages) {
            report_error(a.err, DEV_BAD_PAGE);
            return -1;
          }
          return page;
        };
        int page = page_of(k0);
        for (int t = 0; t < (un.tokens > RH ? 2 : 1) && ok; ++t) {
          if (quse[t] > 0) ok = __all_sync(0xffffffffu, mbar_wait(&q_empty[t], (quse[t] - 1) & 1, a.err, DEV_TIMEOUT_ATTN_EMPTY));
          if (!ok) break;
          ++quse[t];
          if (lane == 0) {
            mbar_arrive_expect_tx(&q_full[t], (uint32_t)RH * a.G * 256);
            for (int h = 0; h < 2; ++h)
              tma_load_3d(qs + t * kPtTile + h * (kPtTile / 2), &tmq, 64 * h, g * a.G, un.token0 + t * RH, &q_full[t]);
          }
        }
        for (int k = k0; k < k1 && ok; ++k) {
          const int c0 = tile_key(un, k) + box * br;
          const int now = page;
          page = page_of(k + 1);  // its load runs while the slots are waited for
          const int y = ((now * a.Hkv + g) << b.page_log2) + (c0 & ((1 << b.page_log2) - 1));
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, now >= 0 && kind < 2)) * br * 128;
          const int slot = issued % kPtSlots, parity = ((issued / kPtSlots) - 1) & 1;
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            uint64_t* full = &kv_full[kv * kPtSlots + slot];
            if (issued >= kPtSlots)
              ok = ok && __all_sync(0xffffffffu, mbar_wait(&kv_empty[kv * kPtSlots + slot], parity, a.err, DEV_TIMEOUT_ATTN_EMPTY));
            if (!ok) break;
            if (lane == 0) mbar_arrive_expect_tx(full, bytes);
            __syncwarp();
            if (now >= 0 && (kind >> 1) == kv)
              tma_load_2d((kv ? vring : kring) + slot * kPtKvTile + (kind & 1) * (kPtKvTile / 2) + box * br * 128,
                          kv ? &tmv : &tmk, 64 * (kind & 1), y, full);
          }
          if (ok) ++issued;
        }
        if (flags[0] != 0) ok = false;
        return ok;
      }, [&] { ok = false; });
      if (!ok) flags[0] = 1;
      // keep shared memory alive until every issued copy has landed (after a failure a K tile may have no V: the
      // waits are bounded)
      for (int t = 0; t < 2; ++t)
        if (quse[t] > 0) mbar_wait(&q_full[t], (quse[t] - 1) & 1, nullptr, 0);
      for (int i = max(0, issued - kPtSlots); i < issued + (ok ? 0 : 1); ++i)
        for (int kv = 0; kv < 2; ++kv) mbar_wait(&kv_full[kv * kPtSlots + i % kPtSlots], (i / kPtSlots) & 1, nullptr, 0);
    } else if (warp == 2) {
      // ----------------------------------------------- scheduler and gatekeeper
      int u = 0;
      for (int hi = max(0, units - 1); u < hi;) {  // the unit of tile t_begin
        const int mid = (u + hi) >> 1;
        if ((long long)unit_tile[mid + 1] * a.Hkv > t_begin) hi = mid;
        else u = mid + 1;
      }
      long long at = t_begin, base = 0;
      TcUnit un;
      int n = 0, fresh = -1, made = 0;  // fresh: the unit that `un` describes
      bool more = true, ok = true;
      auto hand_over = [&] {  // the next piece into the ring
        const int e = made % kPtPieces;
        PtPiece p;
        p.k0 = p.k1 = 0;  // the end of the CTA's work
        while (at < t_end && p.k0 == p.k1) {
          if (fresh != u) {
            un = tc_unit(b, seqs, seq_unit, u, 2 * RH);
            n = unit_tile[u + 1] - unit_tile[u];
            base = (long long)unit_tile[u] * a.Hkv;
            fresh = u;
          }
          const int g = (int)((at - base) / n);
          const long long u0 = base + (long long)g * n;
          p.seq = un.seq;
          p.token0 = un.token0;
          p.tokens = un.tokens;
          p.p_first = un.p_first;
          p.hi = un.hi;
          p.lo_tile = un.ts.lo_tile;
          p.n_sink = un.ts.n_sink;
          p.lo = un.ts.lo;
          p.head = g;
          const int x0 = (int)(at - u0), x1 = (int)min((long long)n, x0 + (t_end - at));
          p.k0 = max(0, x0 - kPtUnitCost);  // its first places hold no tile
          p.k1 = max(0, x1 - kPtUnitCost);
          p.whole = p.k0 == 0 && x1 == n;
          p.first = at == t_begin;
          p.last = p.k0 == 0 && !p.whole ? tile_owner(u0 + n - 1, total, E) : -1;
          at += x1 - x0;
          if (g == a.Hkv - 1 && x1 == n) ++u;
        }
        if (made >= kPtPieces)
          ok = __all_sync(0xffffffffu, mbar_wait(&piece_empty[e], ((made / kPtPieces) - 1) & 1, a.err, DEV_TIMEOUT_ATTN_EMPTY));
        if (!ok) return;
        if (lane == 0) {
          pieces[e] = p;
          mbar_arrive(&piece_full[e]);
        }
        ++made;
        more = p.k0 != p.k1;
      };
      while (more && made < kPtPieces) hand_over();
      // The gatekeeper waits for the K and V tiles that a step's MMAs read and
      // joins P's barrier for them: an MMA warp's own waits take 280 cycles each
      // even where nothing is to be waited for, a quarter of its step.
      int J = 0;
      uint32_t phase = 0;  // bit 2 t + buffer
      walk([&](const PtPiece& pc) {
        const int steps = pc.k1 - pc.k0, nt = pc.tokens > RH ? 2 : 1;
        for (int k = 0; k < steps && ok; ++k, ++J) {
          ok = mbar_wait(&kv_full[kPtSlots + J % kPtSlots], (J / kPtSlots) & 1, a.err, DEV_TIMEOUT_ATTN_FULL);
          if (ok && k + 2 < steps) ok = mbar_wait(&kv_full[(J + 2) % kPtSlots], ((J + 2) / kPtSlots) & 1, a.err, DEV_TIMEOUT_ATTN_FULL);
          for (int t = 0; t < nt && ok; ++t) {
            const int i = 2 * t + (J & 1);
            ok = mbar_wait(&p_full[i], ((phase >> i) & 1) ^ 1, a.err, DEV_TIMEOUT_ATTN_FULL);  // the tile before it is through
            if (ok && lane == 0) mbar_arrive(&p_full[i]);
            phase ^= 1u << i;
          }
          ok = __all_sync(0xffffffffu, ok);
        }
        if (ok && more) hand_over();
        return ok && flags[0] == 0;
      }, [] {});
    } else if (warp == 1 || warp == 3) {
      // ------------------------------------------------------------ MMA issuer
      const uint32_t idesc_s = pg_idesc(128, kPtKeys);
      const uint32_t idesc_o = pg_idesc(128, 128) | (1u << 16);  // B (V) MN-major
      // descriptors made once; an offset of x bytes adds x >> 4 (the addresses stay below 2^18)
      const uint64_t qd = ft_desc(qs, 16, 1024), kd = ft_desc(kring, 16, 1024);
      const uint64_t vd = ft_desc(vring, kPtKvTile / 2, 1024);
      const uint32_t lead = elect_lane() ? 1u : 0u;
      const int t = warp == 1 ? 0 : 1;
      auto uniform = [](int v) { return __shfl_sync(0xffffffffu, v, 0); };
      auto wait = [&](uint64_t* bar, int parity) {
        return __all_sync(0xffffffffu, pt_wait(bar, parity, a.err, DEV_TIMEOUT_ATTN_FULL)) != 0;
      };
      const uint64_t qt = qd + (uint64_t)(t * (kPtTile >> 4));
      const uint32_t sd = tmem + (uint32_t)(128 * t), od = tmem + (uint32_t)(256 + 128 * t);
      int J = 0, qphase = 0, pphase = 0;
      bool ok = true;
      walk([&](const PtPiece& un) {
        const int n = uniform(un.k1 - un.k0);
        const bool both = uniform(un.tokens > RH) != 0;
        if (t == 1 && !both) {
          J += n;
          return true;
        }
        auto k_full = [&](int j) { return wait(&kv_full[j % kPtSlots], (j / kPtSlots) & 1); };
        // a slot is free after both M tiles' MMAs; of a lone tile it is released twice
        auto release = [&](int kv, int j) {
          tc_commit_by(lead, &kv_empty[kv * kPtSlots + j % kPtSlots]);
          if (!both) tc_commit_by(lead, &kv_empty[kv * kPtSlots + j % kPtSlots]);
        };
        auto issue_s = [&](int j) {  // S_t of key tile j of this CTA into buffer j & 1: 16 dims a step
          const uint64_t kt = kd + (uint64_t)((j % kPtSlots) * (kPtKvTile >> 4));
#pragma unroll
          for (int k = 0; k < 8; ++k)
            tc_mma_ss(lead, sd + (uint32_t)(64 * (j & 1)), qt + (k >> 2) * (kPtTile >> 5) + (k & 3) * 2,
                      kt + (k >> 2) * (kPtKvTile >> 5) + (k & 3) * 2, idesc_s, k > 0 ? 1u : 0u);
          tc_commit_by(lead, &s_full[2 * t + (j & 1)]);
          release(0, j);
        };
        ok = wait(&q_full[t], qphase) && k_full(J);
        if (!ok) return false;
        qphase ^= 1;
        tc_fence_after();
        issue_s(J);
        if (n > 1) {
          ok = k_full(J + 1);
          if (!ok) return false;
          tc_fence_after();
          issue_s(J + 1);
        }
        if (n <= 2) tc_commit_by(lead, &q_empty[t]);
#pragma unroll 1
        for (int k = 0; k < n && ok; ++k, ++J) {
          ok = wait(&p_full[2 * t + (J & 1)], (pphase >> (J & 1)) & 1);  // P, and K and V (warp 2)
          if (!ok) break;
          pphase ^= 1 << (J & 1);
          tc_fence_after();
          // O_t += P_t . V: 16 keys a step, P in the first half of S's buffer
          const uint64_t vt = vd + (uint64_t)((J % kPtSlots) * (kPtKvTile >> 4));
#pragma unroll
          for (int i = 0; i < 4; ++i)
            tc_mma_ts(lead, od, sd + (uint32_t)(64 * (J & 1) + 8 * i), vt + i * 128, idesc_o, i > 0 || k > 0 ? 1u : 0u);
          tc_commit_by(lead, &o_done[2 * t + (J & 1)]);
          release(1, J);
          if (k + 2 < n) {
            issue_s(J + 2);  // over P's buffer: runs after P . V, as issued
            if (k + 3 == n) tc_commit_by(lead, &q_empty[t]);
          }
        }
        return ok;
      }, [&] { ok = false; });
      if (!ok) flags[0] = 1;
      tc_commit_by(lead, &done[t]);  // TMEM is released below only after every MMA issued here has completed
      mbar_wait(&done[t], 0, nullptr, 0);
    }
  } else {
    // ----------------------------------------------------------------- softmax
    const int t = (warp - 4) >> 2;  // M tile
    const int qrow = (warp & 3) * 32 + lane;
    const int qi = qrow / a.G, hj = qrow - qi * a.G;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + 128 * t, o_col = tmem + lanes + 256 + 128 * t;
    const float scale = kLog2e * 0.08838834764831845f;  // log2(e) / sqrt(128)
    int J = 0;
    uint32_t sphase = 0;  // of S's two buffers: the phase of their next use
    // O_t with key tile j, the last one whose S was read in its buffer, added
    auto pv_done = [&](int j) {
      return mbar_wait(&o_done[2 * t + (j & 1)], ((sphase >> (j & 1)) & 1) ^ 1, a.err, DEV_TIMEOUT_ATTN_FULL);
    };
    walk([&](const PtPiece& un) {
      const int k0 = un.k0, k1 = un.k1;
      if (t * RH >= un.tokens) {
        J += k1 - k0;
        return true;
      }
      const int token = t * RH + qi;  // of the unit
      const bool valid = qi < RH && token < un.tokens;
      const int pos = !valid ? -1 : b.q_start == nullptr ? un.hi - 1 : un.p_first + token;
      float m_ref = -INFINITY, l = 0.f;
      for (int k = k0; k < k1; ++k, ++J) {
        const int c0 = tile_key(un, k);
        const uint32_t buf = s_col + 64 * (J & 1);
        bool ok = pt_wait(&s_full[2 * t + (J & 1)], (sphase >> (J & 1)) & 1, a.err, DEV_TIMEOUT_ATTN_FULL);
        if (!__all_sync(0xffffffffu, ok)) return false;
        sphase ^= 1u << (J & 1);
        tc_fence_after();
        uint32_t sr[64];
        tc_ld32_async(buf, sr);
        tc_ld32_async(buf + 32, sr + 32);
        tc_ld_wait(sr);
        // keys [lo, hi) and [0, first) of the tile are visible to this row
        const int hi = pos - c0 + 1;
        const int lo = b.window > 0 ? pos - b.window + 1 - c0 : 0;
        const int first = b.sinks - c0;
        if (!__all_sync(0xffffffffu, hi >= kPtKeys && (lo <= 0 || first >= kPtKeys))) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {  // one bit a key, so that each score costs a test and a select
            const uint32_t seen = bits_below(hi - 32 * w) & (~bits_below(lo - 32 * w) | bits_below(first - 32 * w));
#pragma unroll
            for (int c = 0; c < 32; ++c)  // -inf where unseen, whatever the score was
              sr[32 * w + c] = (seen >> c) & 1u ? sr[32 * w + c] : 0xff800000u;
          }
        }
        float mx[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = fmaxf(__uint_as_float(sr[e]), __uint_as_float(sr[e + 4]));
#pragma unroll
        for (int c = 8; c < 64; c += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(sr[c + e]), __uint_as_float(sr[c + e + 4]));
        const float m_new = scale * fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        // A row that has seen nothing has O = l = 0: its reference moves freely.
        if (m_ref == -INFINITY) m_ref = m_new;
        if (__any_sync(0xffffffffu, m_new > m_ref + 8.f)) {
          ok = pv_done(J - 1);
          if (!__all_sync(0xffffffffu, ok)) return false;
          tc_fence_after();
          const float top = fmaxf(m_ref, m_new);
          const float corr = m_ref == -INFINITY ? 1.f : exp2f(m_ref - top);
#pragma unroll 1
          for (int c = 0; c < 128; c += 8) {
            float ov[8];
            tc_ld8(o_col + c, ov);
            asm volatile(
                "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(o_col + c),
                "r"(__float_as_uint(ov[0] * corr)), "r"(__float_as_uint(ov[1] * corr)),
                "r"(__float_as_uint(ov[2] * corr)), "r"(__float_as_uint(ov[3] * corr)),
                "r"(__float_as_uint(ov[4] * corr)), "r"(__float_as_uint(ov[5] * corr)),
                "r"(__float_as_uint(ov[6] * corr)), "r"(__float_as_uint(ov[7] * corr))
                : "memory");
          }
          tc_st_wait();
          l *= corr;
          m_ref = top;
        }
        if (c0 + kPtKeys > un.hi || (b.window > 0 && c0 < un.lo && c0 + kPtKeys > b.sinks)) {
          // V rows that no row of the unit sees may hold anything: their P is 0, but 0 * NaN is NaN. A warp
          // clears 16 keys, four rows of a 64-dim half at a time.
          ok = mbar_wait(&kv_full[kPtSlots + J % kPtSlots], (J / kPtSlots) & 1, a.err, DEV_TIMEOUT_ATTN_FULL);
          if (!__all_sync(0xffffffffu, ok)) return false;
          uint8_t* vt = vring + (J % kPtSlots) * kPtKvTile + (lane & 7) * 16;
#pragma unroll 1
          for (int i = 0; i < 4; ++i) {
            const int r = (warp & 3) * 16 + i * 4 + (lane >> 3), c = c0 + r;
            if (c >= un.hi || (b.window > 0 && c < un.lo && c >= b.sinks)) {
              *reinterpret_cast<uint4*>(vt + r * 128) = make_uint4(0u, 0u, 0u, 0u);
              *reinterpret_cast<uint4*>(vt + r * 128 + kPtKvTile / 2) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_proxy_async_smem();
        }
        // P over S's own registers, two bf16 in one, and over the first half of the buffer.
        const float mu = m_ref == -INFINITY ? 0.f : m_ref;
        const uint64_t scale2 = f32x2(scale, scale), mu2 = f32x2(-mu, -mu);
        uint64_t rs[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 64; c += 2) {
          const uint64_t x = fma_f32x2(f32x2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), scale2, mu2);
          float p0, p1;
          if ((c >> 1) % kPtPolyEvery == kPtPolyEvery - 1) {
            exp2_poly(x, p0, p1);
          } else {
            unpack_f32x2(x, p0, p1);
            p0 = ex2_approx(p0);
            p1 = ex2_approx(p1);
          }
          rs[(c >> 1) & 1] = add_f32x2(rs[(c >> 1) & 1], f32x2(p0, p1));
          sr[c >> 1] = pack_bf16(p0, p1);
        }
        tc_st32_async(buf, sr);
        tc_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * t + (J & 1)]);
        float r0, r1;
        unpack_f32x2(add_f32x2(rs[0], rs[1]), r0, r1);
        l += r0 + r1;
      }
      // ---- the piece's rows
      const bool ok = pv_done(J - 1);
      if (!__all_sync(0xffffffffu, ok)) return false;
      tc_fence_after();
      const bool whole = un.whole != 0;
      const int slot = 2 * me + (un.first ? 0 : 1);
      const size_t row = (size_t)(un.token0 + token) * a.Hq + un.head * a.G + hj;
      const bool has_base = a.sink.base32 != nullptr;
      RowScale rs = {1.f, 0.f, 0.f};
      if (whole && valid) rs = row_scale(m_ref, l, has_base, has_base ? a.sink.base_lse[row] : 0.f);
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        float ov[32];
        tc_ld32(o_col + 32 * c, ov);
        if (!valid) continue;
#pragma unroll
        for (int e = 0; e < 32; ++e) ov[e] *= rs.own;
        if (!whole || a.sink.out32 != nullptr) {
          float* dst = whole ? a.sink.out32 + row * kAttnD + 32 * c
                             : a.part_o + ((size_t)slot * kPtRows + t * 128 + qrow) * kAttnD + 32 * c;
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(ov[e + i]);
            st_global_32(dst + e, w);
          }
        } else {
          if (has_base) {
            const float* bv = a.sink.base32 + row * kAttnD + 32 * c;
#pragma unroll
            for (int e = 0; e < 32; e += 4) {
              const float4 x = *reinterpret_cast<const float4*>(bv + e);
              ov[e] = fmaf(x.x, rs.other, ov[e]);
              ov[e + 1] = fmaf(x.y, rs.other, ov[e + 1]);
              ov[e + 2] = fmaf(x.z, rs.other, ov[e + 2]);
              ov[e + 3] = fmaf(x.w, rs.other, ov[e + 3]);
            }
          }
          bf16* dst = a.sink.out + row * kAttnD + 32 * c;
#pragma unroll
          for (int e = 0; e < 32; e += 16) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = pack_bf16(ov[e + 2 * i], ov[e + 2 * i + 1]);
            st_global_32(dst + e, w);
          }
        }
      }
      if (valid) {
        if (!whole) {
          float* ml = a.part_ml + ((size_t)slot * kPtRows + t * 128 + qrow) * 2;
          ml[0] = m_ref;
          ml[1] = l;
        } else if (a.sink.lse32 != nullptr) {
          a.sink.lse32[row] = rs.lse;
        }
      }
      if (un.last >= 0 && t == 0 && qrow == 0) {
        PtUnit* c = &a.cut[me];
        c->token0 = un.token0;
        c->tokens = un.tokens;
        c->head = un.head;
        c->last = un.last;
        c->first_slot = un.first ? 0 : 1;
        c->valid = 1;
      }
      tc_fence_before();  // O_t is read before the next unit's MMAs write it (through p_full)
      return true;
    }, [] {});
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// Joins the pieces of the units that paged_tc_kernel cut: a warp a row, a lane
// 4 dims, the rows of all cut units dealt out to the grid's warps. Bound by the
// latency of its loads (the pieces lie in L2), so a row's are issued eight
// pieces at a time.
constexpr int kPjThreads = 256;
constexpr int kPjCtasPerSm = 8;
__global__ void __launch_bounds__(kPjThreads) paged_join_kernel(const PagedTcArgs a, int ctas) {
  __shared__ int cut_of[kPagedMaxTcCtas];
  __shared__ int warp_cuts[kPjThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_trigger();
  int cuts = 0;
  for (int c0 = 0; c0 < ctas; c0 += kPjThreads) {  // the CTAs whose last piece begins a cut unit
    const int c = c0 + threadIdx.x;
    const bool is = c < ctas && a.cut[c].valid != 0;
    const unsigned who = __ballot_sync(0xffffffffu, is);
    if (lane == 0) warp_cuts[warp] = __popc(who);
    __syncthreads();
    int at = cuts;
    for (int w = 0; w < kPjThreads / 32; ++w) {
      if (w < warp) at += warp_cuts[w];
      cuts += warp_cuts[w];
    }
    if (is) cut_of[at + __popc(who & ((1u << lane) - 1u))] = c;
    __syncthreads();
  }
  const int RH = 128 / a.G;
  const bool has_base = a.sink.base32 != nullptr;
  for (int i = blockIdx.x * (kPjThreads / 32) + warp; i < cuts * kPtRows; i += gridDim.x * (kPjThreads / 32)) {
    const int first = cut_of[i / kPtRows];
    const PtUnit un = a.cut[first];
    const int r = i % kPtRows, t = r >> 7, qrow = r & 127;
    const int qi = qrow / a.G, token = t * RH + qi;
    if (qi >= RH || token >= un.tokens) continue;
    auto piece = [&](int c) { return (size_t)(2 * c + (c == first ? un.first_slot : 0)) * kPtRows + r; };
    float top = -INFINITY;
    for (int c = first + lane; c <= un.last; c += 32) top = fmaxf(top, a.part_ml[piece(c) * 2]);
    top = warp_max(top);
    const float mu = top == -INFINITY ? 0.f : top;
    float lsum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c0 = first; c0 <= un.last; c0 += 8) {
      float2 ml[8];
      float4 ov[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool in = c0 + j <= un.last;
        ml[j] = in ? *reinterpret_cast<const float2*>(a.part_ml + piece(c0 + j) * 2) : make_float2(-INFINITY, 0.f);
        ov[j] = in ? *reinterpret_cast<const float4*>(a.part_o + piece(c0 + j) * kAttnD + 4 * lane)
                   : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float w = exp2f(ml[j].x - mu);
        lsum = fmaf(ml[j].y, w, lsum);
        acc.x = fmaf(ov[j].x, w, acc.x);
        acc.y = fmaf(ov[j].y, w, acc.y);
        acc.z = fmaf(ov[j].z, w, acc.z);
        acc.w = fmaf(ov[j].w, w, acc.w);
      }
    }
    const size_t row = (size_t)(un.token0 + token) * a.Hq + un.head * a.G + qrow % a.G;
    const RowScale rs = row_scale(top, lsum, has_base, has_base ? a.sink.base_lse[row] : 0.f);
    acc.x *= rs.own; acc.y *= rs.own; acc.z *= rs.own; acc.w *= rs.own;
    if (has_base) {
      const float4 bv = *reinterpret_cast<const float4*>(a.sink.base32 + row * kAttnD + 4 * lane);
      acc.x = fmaf(bv.x, rs.other, acc.x);
      acc.y = fmaf(bv.y, rs.other, acc.y);
      acc.z = fmaf(bv.z, rs.other, acc.z);
      acc.w = fmaf(bv.w, rs.other, acc.w);
    }
    if (a.sink.out32 != nullptr) {
      *reinterpret_cast<float4*>(a.sink.out32 + row * kAttnD + 4 * lane) = acc;
      if (lane == 0 && a.sink.lse32 != nullptr) a.sink.lse32[row] = rs.lse;
    } else {
      uint2 ob;
      ob.x = pack_bf16(acc.x, acc.y);
      ob.y = pack_bf16(acc.z, acc.w);
      *reinterpret_cast<uint2*>(a.sink.out + row * kAttnD + 4 * lane) = ob;
    }
  }
}

}  // namespace qb
