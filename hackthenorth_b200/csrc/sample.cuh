// sample.cuh — drawing a token from a row of logits with temperature, top-k,
// top-p and min-p, from a given uniform number (the sampled counterpart of the
// greedy head, dryft/engine/kernels/greedy.py:13-60; the reference only takes
// the argmax).
//
//   w_i = exp((x_i - max x) / T);  tokens ranked by falling x, then rising index
//   top-k: the first k ranks; top-p: of these, the ranks before which less than
//   p of their mass lies; min-p: of these, the ones with w_i >= min_p
//   token = the first index at which the running mass of the kept tokens, in
//   index order, exceeds u times their mass
//
// Masses are integers (w 2^44, so a sum of up to 2^18 tokens fits 64 bits), which
// makes every sum exact and the result independent of the order of the atomics.
//
// A cluster of 8 CTAs holds the row in shared memory, so it is read once.
// Bound by latency: a chain of a few cluster barriers and of code that runs once
// (one row of 151936: 8 us on the device, 192 rows 150 us, 37 of them at a time,
// beside 18 us for their bytes). So the work is cut down step by step:
//  1. the largest token of every lane and warp, and of the row with its lowest
//     index: the answer of greedy rows (T = 0)
//  2. what cannot be kept is dropped without being counted: the first top_k
//     warps' maxima (or as many as hold top-p's mass) are that many tokens, so
//     nothing below the last of them ranks among the first top_k; where the
//     warps' 128 are too few, the same with the lanes' 4096, in bins
//  3. up to 4096 tokens are left: put in a list in index order, and one CTA finds
//     the border, of up to 256 by counting each one's betters (sorting or a
//     search by bits took 20 us more), of more by 1024 bins and the border's bin
//     token by token
//  4. else (wide nuclei, flat rows): all tokens counted and weighed in 1024 bins
//     of equal width in (max - x) / T (1/32 each, the last takes the rest:
//     monotone in x, and unlike bins of x's own bits not a handful of crowded
//     ones), each CTA summing its share over the cluster; the border's bin again
//     in 1024 sub-bins, a sub-bin of unequal tokens by 8 bits of their pattern at
//     a time; then the kept mass of every warp's stretch of indexes, the stretch
//     that the target falls in, and the token in it (without any filter: this alone)
#pragma once
#include "attention.cuh"

namespace qb {

constexpr int kSmThreads = 512;
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kSmBins = 1024;
constexpr int kSmCluster = 8;
constexpr int kSmMaxVocab = 1 << 18;
constexpr float kSmBinsPerUnit = 32.f;
constexpr float kSmOne = 17592186044416.f;  // 2^44: weight 1

struct SampleArgs {
  const void* logits;  // [rows][vocab]
  const float* uniforms;
  const float* temperature;  // per row, or NULL: the value below
  const int* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_all, top_p_all, min_p_all;
  int top_k_all;
  int vocab, slice;  // slice: tokens a CTA holds, a multiple of 128
  int64_t* out;
  int* err;
};

struct SampleBorder {  // the slot that holds the last kept rank
  unsigned long long before_mass, mass;  // of what ranks before the slot, of its own tokens
  unsigned before_count, count;
  unsigned slot;
  unsigned key_or, key_and;  // of its tokens' ordered patterns (where asked for)
  unsigned found;
};

constexpr int kSmList = 4096;  // tokens of a list
constexpr int kSmShort = 256;  // of one whose ranks are counted token by token

struct alignas(16) SampleShared {
  union {
    struct {
      unsigned cnt[kSmBins], lo[kSmBins], hi[kSmBins], kor[kSmBins], kand[kSmBins];
    };
    struct {
      unsigned list_key[kSmList], list_token[kSmList];
      unsigned long long short_mass[kSmShort];
    };
  };
  unsigned long long warp_mass[kSmCluster * kSmWarps];  // every warp of the cluster
  unsigned warp_ties[kSmCluster * kSmWarps];
  unsigned long long seg_mass[kSmCluster];  // of every CTA's bins
  unsigned seg_cnt[kSmCluster];
  unsigned long long warp_top[kSmCluster * kSmWarps];  // (ordered value, inverted index) of every warp's maximum
  unsigned long long scan_mass[kSmWarps];
  unsigned scan_cnt[kSmWarps];
  SampleBorder border;
};

// For a list that is not short, in the row's place once the list is made.
struct SampleLong {
  unsigned cnt[kSmBins], lo[kSmBins], hi[kSmBins];
  unsigned long long mass[kSmShort];  // of the border bin's tokens
  unsigned key[kSmShort], place[kSmShort];
  unsigned members, cut_key, cut_place;
  unsigned long long cut_mass;  // up to the cut, its token included
};

// Values as unsigned numbers in the same order; -0 counts as 0, and what cannot
// be drawn (NaN, -inf) as 0.
__device__ __forceinline__ unsigned sample_key(float x) {
  if (!(x > -INFINITY)) return 0u;
  const unsigned u = __float_as_uint(x + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float sample_value(unsigned key) {
  return __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

__device__ __forceinline__ unsigned cluster_addr(const void* p, unsigned rank) { return map_shared_rank(p, rank); }
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, unsigned v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ unsigned ld_cluster_u32(uint32_t addr) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ void sample_load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void sample_load8<bf16>(const bf16* p, float (&x)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  x[0] = bf_lo(v.x); x[1] = bf_hi(v.x); x[2] = bf_lo(v.y); x[3] = bf_hi(v.y);
  x[4] = bf_lo(v.z); x[5] = bf_hi(v.z); x[6] = bf_lo(v.w); x[7] = bf_hi(v.w);
}
template <>
__device__ __forceinline__ void sample_load8<float>(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
  x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ T sample_lowest();
template <>
__device__ __forceinline__ bf16 sample_lowest<bf16>() { return __ushort_as_bfloat16(0xff80); }
template <>
__device__ __forceinline__ float sample_lowest<float>() { return -INFINITY; }

__host__ inline size_t sample_smem_bytes(int slice, int item) {
  const size_t row = (size_t)slice * item;
  return sizeof(SampleShared) + 16 + (row > sizeof(SampleLong) ? row : sizeof(SampleLong));
}

template <typename T>
__global__ void __cluster_dims__(kSmCluster, 1, 1) __launch_bounds__(kSmThreads, 2) sample_kernel(const SampleArgs a) {
  extern __shared__ uint8_t smem_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>((reinterpret_cast<uintptr_t>(smem_raw) + 15) & ~uintptr_t(15));
  T* xs = reinterpret_cast<T*>(reinterpret_cast<uint8_t*>(&sh) + sizeof(SampleShared));
  constexpr int C = kSmCluster;
  const int rank = (int)cluster_ctarank(), row = blockIdx.x / C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int base = rank * a.slice;                           // first token of this CTA
  const int seg = a.slice / kSmWarps;                        // tokens of a warp, a multiple of 8
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  pdl_wait();
  pdl_trigger();

  // A warp owns a stretch of the tokens, a lane 8 of each 256 of it.
  auto each = [&](auto&& f) {  // f(tokens i .. i + 7 of the slice, i)
    for (int i = warp * seg + 8 * lane; i < (warp + 1) * seg; i += 256) {
      float x[8];
      sample_load8<T>(xs + i, x);
      f(x, i);
    }
  };

  // ---- the row's slice into shared memory (filled up with -inf), and the largest token of every lane and warp
  const T* src = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.vocab + base;
  const int live = max(0, min(a.slice, a.vocab - base));
  const bool aligned = (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  float mine = -INFINITY;
  int mine_at = 0;  // of its first place, the eight tokens it is among
#pragma unroll 4
  for (int i = warp * seg + 8 * lane; i < (warp + 1) * seg; i += 256) {
    alignas(16) T v[8];
    if (aligned && i + 8 <= live) {
#pragma unroll
      for (int j = 0; j < (int)sizeof(T) / 2; ++j)
        reinterpret_cast<uint4*>(v)[j] = __ldcs(reinterpret_cast<const uint4*>(src + i) + j);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = i + j < live ? src[i + j] : sample_lowest<T>();
    }
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4*>(xs + i)[j] = reinterpret_cast<uint4*>(v)[j];
    float m = (float)v[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) m = fmaxf(m, (float)v[j]);  // drops NaN
    if (m > mine) {
      mine = m;
      mine_at = i;
    }
  }
  unsigned long long best = 0ull;
  if (mine > -INFINITY) {
    while (!((float)xs[mine_at] == mine)) ++mine_at;
    best = ((unsigned long long)sample_key(mine) << 32) | (unsigned)~(unsigned)(base + mine_at);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
    best = other > best ? other : best;
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // every CTA runs: its memory may be written
  if (lane < C) st_cluster_u64(cluster_addr(&sh.warp_top[rank * kSmWarps + warp], lane), best);
  cluster_sync_all();
  constexpr int kTops = C * kSmWarps / 32;
  unsigned long long tops[kTops];  // a lane's share of the warps' largest
  best = 0ull;
#pragma unroll
  for (int j = 0; j < kTops; ++j) {
    tops[j] = sh.warp_top[lane + 32 * j];
    best = tops[j] > best ? tops[j] : best;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
    best = other > best ? other : best;
  }
  const unsigned top_key = (unsigned)(best >> 32);
  const float top = sample_value(top_key);

  float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
  if (top_key == 0u || !(temperature > 0.f)) {  // nothing to draw, or greedy
    if (rank == 0 && threadIdx.x == 0) {
      if (top_key == 0u) report_error(a.err, DEV_BAD_LOGITS);
      a.out[row] = top_key == 0u ? -1 : (int64_t)(unsigned)~(unsigned)best;
    }
    return;  // the same for the whole cluster, and no CTA's memory is read after the barrier
  }
  if (top == INFINITY) temperature = 1.f;  // an infinite logit takes all the mass at any temperature, infinity too
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  const float min_p = fminf(a.min_p ? a.min_p[row] : a.min_p_all, 1.f);
  temperature = fmaxf(temperature, 1.17549435e-38f);  // 2^-126: below it 1 / T passes fp32
  const float inv_t = 1.f / temperature;
  const float mend_below = inv_t > 0.f ? 128.f : 0.f;  // T infinite: the quotient 0 is exact, and T * 0 no number

  // (max - x) / T for the bins (0 at the maximum, infinite ones too), and the weight, of the same corrected to a
  // rounding or two of 2^-24: its error would be the weight's.
  auto depth = [&](float x) { return x == top ? 0.f : fminf(top - x, 3.402823466e38f) * inv_t; };
  auto weight = [&](float x, float y) {
    if (y < mend_below) y = fmaf(fmaf(-y, temperature, x == top ? 0.f : top - x), inv_t, y);
    return expf(-y);
  };
  auto mass_of = [](float w) { return (unsigned long long)__float2ull_rn(w * kSmOne); };
  auto bin_of = [](float y) { return (int)fminf(y * kSmBinsPerUnit, (float)(kSmBins - 1)); };
  auto sub_of = [](float y, int bin) {
    const float f = (fminf(y, 64.f) * kSmBinsPerUnit - (float)bin) * (float)kSmBins;
    return (int)fminf(fmaxf(f, 0.f), (float)(kSmBins - 1));
  };

  const bool by_mass = top_p < 1.f;

  auto every_token = [&](auto&& f) {
    each([&](const float (&x)[8], int) {
#pragma unroll
      for (int j = 0; j < 8; ++j) f(x[j]);
    });
  };
  auto lane_tops = [&](auto&& f) { f(mine); };

  // Tokens of the cluster counted (and weighed) in `bins` slots: member(x, y,
  // slot) says whether a token counts, and where. Thread i < bins / 8 comes back
  // with slot rank * bins / 8 + i: its sums over the cluster and what lies before.
  struct Slot {
    unsigned long long mass, before_mass;
    unsigned count, before_count, key_or, key_and;
  };
  unsigned long long all_mass = 0ull;  // of the last histogram
  auto histogram = [&](int bins, bool masses, bool keys, auto&& tokens, auto&& member) {
    __syncthreads();  // everyone has read the last border
    for (int i = threadIdx.x; i < bins; i += kSmThreads) {
      sh.cnt[i] = sh.lo[i] = sh.hi[i] = 0u;
      if (keys) {
        sh.kor[i] = 0u;
        sh.kand[i] = 0xffffffffu;
      }
    }
    if (threadIdx.x == 0) sh.border.found = 0u;
    __syncthreads();
    tokens([&](float x) {
      int slot;
      if (!(x > -INFINITY)) return;
      const float y = depth(x);
      if (!member(x, y, slot)) return;
      atomicAdd(&sh.cnt[slot], 1u);
      if (masses) {
        const unsigned long long q = mass_of(weight(x, y));
        const unsigned ql = (unsigned)q;
        unsigned qh = (unsigned)(q >> 32);
        if (ql != 0u) qh += atomicAdd(&sh.lo[slot], ql) + ql < ql;  // the carry
        if (qh != 0u) atomicAdd(&sh.hi[slot], qh);
      }
      if (keys) {
        atomicOr(&sh.kor[slot], sample_key(x));
        atomicAnd(&sh.kand[slot], sample_key(x));
      }
    });
    cluster_sync_all();
    const int share = bins / C, i = rank * share + threadIdx.x;
    Slot s = {0ull, 0ull, 0u, 0u, 0u, 0xffffffffu};
    if (threadIdx.x < share)
#pragma unroll
      for (int c = 0; c < kSmCluster; ++c) {
        s.count += ld_cluster_u32(cluster_addr(&sh.cnt[i], c));
        s.mass += ((unsigned long long)ld_cluster_u32(cluster_addr(&sh.hi[i], c)) << 32) + ld_cluster_u32(cluster_addr(&sh.lo[i], c));
        if (keys) {
          s.key_or |= ld_cluster_u32(cluster_addr(&sh.kor[i], c));
          s.key_and &= ld_cluster_u32(cluster_addr(&sh.kand[i], c));
        }
      }
    // sums before each slot: within the share, then the shares before it
    unsigned n = s.count;
    unsigned long long q = s.mass;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned un = __shfl_up_sync(0xffffffffu, n, o);
      const unsigned long long uq = __shfl_up_sync(0xffffffffu, q, o);
      if (lane >= o) {
        n += un;
        q += uq;
      }
    }
    if (lane == 31) {
      sh.scan_cnt[warp] = n;
      sh.scan_mass[warp] = q;
    }
    __syncthreads();
    unsigned long long total = 0ull;
    unsigned total_n = 0;
    s.before_count = n - s.count;
    s.before_mass = q - s.mass;
    for (int w = 0; w < (share + 31) / 32; ++w) {
      if (w < warp) {
        s.before_count += sh.scan_cnt[w];
        s.before_mass += sh.scan_mass[w];
      }
      total_n += sh.scan_cnt[w];
      total += sh.scan_mass[w];
    }
    if (threadIdx.x < C) {
      st_cluster_u32(cluster_addr(&sh.seg_cnt[rank], threadIdx.x), total_n);
      st_cluster_u64(cluster_addr(&sh.seg_mass[rank], threadIdx.x), total);
    }
    cluster_sync_all();
    all_mass = 0ull;
    for (int c = 0; c < C; ++c) {
      if (c < rank) {
        s.before_count += sh.seg_cnt[c];
        s.before_mass += sh.seg_mass[c];
      }
      all_mass += sh.seg_mass[c];
    }
    return s;
  };
  // The slot in which the running count reaches `count` (mass: reaches `mass`);
  // found 0 if none does. The same answer in every thread of the cluster.
  auto search = [&](const Slot& s, int bins, bool mass_wanted, unsigned count, unsigned long long mass) {
    const int share = bins / C;
    const bool hit = mass_wanted ? s.before_mass < mass && s.before_mass + s.mass >= mass
                                 : s.before_count < count && s.before_count + s.count >= count;
    if (threadIdx.x < share && hit) {
      for (int c = 0; c < C; ++c) {
        const uint32_t b = cluster_addr(&sh.border, c);
        st_cluster_u64(b + offsetof(SampleBorder, before_mass), s.before_mass);
        st_cluster_u64(b + offsetof(SampleBorder, mass), s.mass);
        st_cluster_u32(b + offsetof(SampleBorder, before_count), s.before_count);
        st_cluster_u32(b + offsetof(SampleBorder, count), s.count);
        st_cluster_u32(b + offsetof(SampleBorder, slot), rank * share + threadIdx.x);
        st_cluster_u32(b + offsetof(SampleBorder, key_or), s.key_or);
        st_cluster_u32(b + offsetof(SampleBorder, key_and), s.key_and);
        st_cluster_u32(b + offsetof(SampleBorder, found), 1u);
      }
    }
    cluster_sync_all();
    return sh.border;
  };

  // The drawn token is the first at which the running mass exceeds this.
  auto target_of = [&](unsigned long long total) {
    const double u = (double)a.uniforms[row];
    const unsigned long long t = u > 0.0 ? (unsigned long long)(fmin(u, 1.0) * (double)total) : 0ull;
    return t >= total ? total - 1ull : t;  // the maximum's own weight keeps total above 0
  };

  constexpr int kLowBits = 32 - 8 * (int)sizeof(T);  // bits of the pattern that a bf16 does not have
  // Sum over the warp of masses below 2^59, in three parts whose sums fit 32 bits.
  auto warp_sum64 = [](unsigned long long v) {
    const unsigned long long s0 = __reduce_add_sync(0xffffffffu, (unsigned)(v & 0x3fffffu));
    const unsigned long long s1 = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 22 & 0x3fffffu));
    const unsigned long long s2 = __reduce_add_sync(0xffffffffu, (unsigned)(v >> 44));
    return s0 + (s1 << 22) + (s2 << 44);
  };
  // Mass that top-p keeps of `whole`: ranks before which less than it lies.
  auto wanted = [&](unsigned long long whole) {
    return max(1ull, (unsigned long long)ceil((double)fmaxf(top_p, 0.f) * (double)whole));
  };

  // What is kept: tokens of a bin before bin1, and of bin1 (unless all of it) of
  // a sub-bin before bin2, and of bin2 (unless all of it) those above `key` and
  // the first `ties` of those equal to it.
  int bin1 = kSmBins, bin2 = kSmBins;
  unsigned key = 0u, ties = 0u;
  unsigned long long kept_mass = 0ull;
  // Sets them to the last rank of bin b1 whose count (mass) before it is below the wanted one.
  auto refine = [&](const SampleBorder& b1, bool mass_wanted, unsigned count, unsigned long long mass) {
    bin1 = (int)b1.slot;
    bin2 = kSmBins;
    ties = 0u;
    kept_mass = b1.before_mass + b1.mass;
    if (!mass_wanted && b1.before_count + b1.count == count) return;  // the whole bin
    unsigned need = count - b1.before_count;
    unsigned long long need_mass = mass - b1.before_mass;
    const int want1 = bin1;
    SampleBorder b = search(histogram(kSmBins, by_mass, true, every_token, [&](float, float y, int& slot) {
                              if (bin_of(y) != want1) return false;
                              slot = sub_of(y, want1);
                              return true;
                            }), kSmBins, mass_wanted, need, need_mass);
    bin2 = (int)b.slot;
    kept_mass = b1.before_mass + b.before_mass;
    need -= b.before_count;
    need_mass -= b.before_mass;
    if (b.key_or != b.key_and) {  // different values within 2^-15 of one another: by their bits, 8 at a time
      const int want2 = bin2;
      unsigned head = 0u;
      for (int shift = 24; shift >= 0; shift -= 8) {
        b = search(histogram(256, by_mass, true, every_token, [&](float x, float y, int& slot) {
                     const unsigned k = sample_key(x);
                     if (bin_of(y) != want1 || sub_of(y, want1) != want2 || (shift < 24 && k >> (shift + 8) != head))
                       return false;
                     slot = 255 - (int)(k >> shift & 255u);
                     return true;
                   }), 256, mass_wanted, need, need_mass);
        head = head << 8 | (255u - b.slot);
        kept_mass += b.before_mass;
        need -= b.before_count;
        need_mass -= b.before_mass;
      }
    }
    key = b.key_and;
    const unsigned long long one = b.count > 0u ? b.mass / b.count : 0ull;  // equal tokens weigh the same
    ties = mass_wanted ? (unsigned)min((unsigned long long)b.count, one > 0ull ? (need_mass + one - 1ull) / one : 1ull) : need;
    kept_mass += one * ties;
  };
  // The tokens at or above `least` and in the bins up to `last`, if they are few
  // enough: put in a list in index order, and the rest is up to the first CTA.
  // They have to be a first stretch of the ranks that holds all that is kept;
  // whole: the mass that top-p refers to, 0 for that of the list after top-k.
  auto finish_in_list = [&](float least, int last, bool cut_count, unsigned long long whole) {
    auto in = [&](float x) { return x >= least && x > -INFINITY && (last >= kSmBins || bin_of(depth(x)) <= last); };
    const bool some = __any_sync(0xffffffffu, in(mine));  // most warps have none
    unsigned n = 0;
    if (some)
      each([&](const float (&x)[8], int) {
#pragma unroll
        for (int j = 0; j < 8; ++j) n += in(x[j]);
      });
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane < C) st_cluster_u32(cluster_addr(&sh.warp_ties[rank * kSmWarps + warp], lane), n);
    cluster_sync_all();
    unsigned at = 0, all = 0;
    for (int w = lane; w < C * kSmWarps; w += 32) {
      const unsigned v = sh.warp_ties[w];
      all += v;
      if (w < rank * kSmWarps + warp) at += v;
    }
    at = __reduce_add_sync(0xffffffffu, at);
    all = __reduce_add_sync(0xffffffffu, all);
    if (all > kSmList) {
      cluster_sync_all();  // the counts are read before they are written again
      return false;
    }
    if (n > 0)
      for (int i0 = warp * seg; i0 < (warp + 1) * seg; i0 += 256) {
        const int i = i0 + 8 * lane;
        float x[8];
        unsigned is = 0u;
        if (i < (warp + 1) * seg) {
          sample_load8<T>(xs + i, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) is |= in(x[j]) ? 1u << j : 0u;
        }
        if (!__any_sync(0xffffffffu, is != 0u)) continue;
        unsigned upto = __popc(is);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += v;
        }
        for (unsigned p = at + upto - __popc(is); is != 0u; is &= is - 1u, ++p) {
          const int j = __ffs(is) - 1;
          st_cluster_u32(cluster_addr(&sh.list_key[p], 0), sample_key((float)xs[i + j]));
          st_cluster_u32(cluster_addr(&sh.list_token[p], 0), (unsigned)(base + i + j));
        }
        at += __shfl_sync(0xffffffffu, upto, 31);
      }
    cluster_sync_all();  // the last access to another CTA's memory is before it
    if (rank != 0) return true;
    if (all <= kSmShort) {
      // Short: a thread a token counts what ranks ahead of it. (The bit-by-bit search below takes two dozen barriers.)
      const unsigned p = threadIdx.x;
      unsigned k = 0u, ahead = 0u;
      unsigned long long q = 0ull, ahead_mass = 0ull;
      float w = 0.f;
      if (p < all) {
        k = sh.list_key[p];
        w = weight(sample_value(k), depth(sample_value(k)));
        q = mass_of(w);
        sh.short_mass[p] = q;
      }
      __syncthreads();
      if (p < all)
#pragma unroll 4
        for (unsigned j = 0; j < all; ++j) {
          const unsigned o = sh.list_key[j];
          if (o > k || (o == k && j < p)) {
            ++ahead;
            ahead_mass += sh.short_mass[j];
          }
        }
      const bool counted = p < all && (!cut_count || ahead < (unsigned)top_k);
      if (by_mass) {
        if (whole == 0ull) {  // of what top-k has left: known to its last rank
          if (p < all && ahead == min(cut_count ? (unsigned)top_k : all, all) - 1u) sh.seg_mass[0] = ahead_mass + q;
          __syncthreads();
          whole = sh.seg_mass[0];
        }
      }
      if (!counted || (by_mass && ahead_mass >= wanted(whole)) || !(w >= min_p)) q = 0ull;
      unsigned long long upto = q;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) sh.scan_mass[warp] = upto;
      __syncthreads();
      unsigned long long before = upto - q, total = 0ull;
#pragma unroll
      for (int v = 0; v < kSmShort / 32; ++v) {
        if (v < warp) before += sh.scan_mass[v];
        total += sh.scan_mass[v];
      }
      const unsigned long long target = target_of(total);
      if (target >= before && target < before + q) a.out[row] = sh.list_token[p];
      return true;
    }
    constexpr int kEach = kSmList / kSmThreads;
    unsigned key_of[kEach];
    unsigned long long mass[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const unsigned p = threadIdx.x * kEach + j;
      key_of[j] = p < all ? sh.list_key[p] : 0u;
      mass[j] = 0ull;
      if (p < all) {
        const float x = sample_value(key_of[j]);
        mass[j] = mass_of(weight(x, depth(x)));
      }
    }
    int turn = 0;
    // Count or mass over the list: two buffers, so that one barrier a call is enough.
    auto block_sum = [&](unsigned long long v) {
      v = warp_sum64(v);
      unsigned long long* buf = sh.warp_mass + 32 * (turn++ & 1);
      if (lane == 0) buf[warp] = v;
      __syncthreads();
      unsigned long long t = 0ull;
#pragma unroll
      for (int w = 0; w < kSmWarps; ++w) t += buf[w];
      return t;
    };
    auto over = [&](unsigned least, bool weigh) {  // tokens at or above it
      unsigned long long v = 0ull;
#pragma unroll
      for (int j = 0; j < kEach; ++j) v += key_of[j] >= least ? (weigh ? mass[j] : 1ull) : 0ull;
      return v;
    };
    // Of the tokens kept so far, those behind the rank whose count or mass reaches `want` go. Bit by bit, each with a
    // barrier: for many (nearly) equal tokens.
    auto cut = [&](bool weigh, unsigned long long want) {
      unsigned border = 0u;
      for (int bit = 31; bit >= kLowBits; --bit) {
        const unsigned c = border | 1u << bit;
        if (block_sum(over(c, weigh)) >= want) border = c;
      }
      const unsigned above = border + (1u << kLowBits);  // 0 only past the largest pattern, which no value has
      const unsigned long long rest = want - block_sum(over(above, weigh));
      unsigned eq = 0;
      unsigned long long one = 0ull;
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (key_of[j] >= border && key_of[j] < above) {
          ++eq;
          one = mass[j];
        }
      // equal tokens in index order: those of the threads before, then this one's
      unsigned upto = eq;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) sh.scan_cnt[warp] = upto;
      __syncthreads();
      unsigned r = upto - eq;
      for (int w = 0; w < warp; ++w) r += sh.scan_cnt[w];
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kEach; ++j) {
        bool keep = key_of[j] >= above;
        if (key_of[j] >= border && key_of[j] < above) {
          keep = weigh ? r * one < rest : r < rest;
          ++r;
        }
        if (!keep) {
          mass[j] = 0ull;
          key_of[j] = 0u;
        }
      }
    };
    // The list in bins of equal width in (max - x) / T, counted and weighed; a thread has two of them.
    SampleLong& big = *reinterpret_cast<SampleLong*>(xs);
    const float per_unit = (kSmBins - 1) / fmaxf(least > -INFINITY ? depth(least) : (float)(last + 1) / kSmBinsPerUnit, 1e-20f);
    auto slot_of = [&](unsigned k) { return (int)fminf(depth(sample_value(k)) * per_unit, (float)(kSmBins - 1)); };
    for (int i = threadIdx.x; i < kSmBins; i += kSmThreads) big.cnt[i] = big.lo[i] = big.hi[i] = 0u;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (key_of[j] != 0u) {
        const int i = slot_of(key_of[j]);
        atomicAdd(&big.cnt[i], 1u);
        const unsigned l = (unsigned)mass[j];
        const unsigned h = (unsigned)(mass[j] >> 32) + (l != 0u && atomicAdd(&big.lo[i], l) + l < l);
        if (h != 0u) atomicAdd(&big.hi[i], h);
      }
    __syncthreads();
    unsigned bin_n[2];
    unsigned long long bin_q[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = 2 * threadIdx.x + h;
      bin_n[h] = big.cnt[i];
      bin_q[h] = ((unsigned long long)big.hi[i] << 32) + big.lo[i];
    }
    unsigned n_upto = bin_n[0] + bin_n[1];
    unsigned long long q_upto = bin_q[0] + bin_q[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned un = __shfl_up_sync(0xffffffffu, n_upto, o);
      const unsigned long long uq = __shfl_up_sync(0xffffffffu, q_upto, o);
      if (lane >= o) {
        n_upto += un;
        q_upto += uq;
      }
    }
    if (lane == 31) {
      sh.scan_cnt[warp] = n_upto;
      sh.scan_mass[warp] = q_upto;
    }
    __syncthreads();
    for (int w = 0; w < warp; ++w) {
      n_upto += sh.scan_cnt[w];
      q_upto += sh.scan_mass[w];
    }
    // As cut(), by the bins: the border's bin, and in it, where it is short, token by token. Gives the mass up to the cut.
    auto cut_by_bins = [&](bool weigh, unsigned long long want) {
      unsigned n = n_upto - bin_n[0] - bin_n[1];
      unsigned long long q = q_upto - bin_q[0] - bin_q[1];
      if (threadIdx.x == 0) {
        sh.border.found = 0u;
        big.members = 0u;
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (weigh ? q < want && q + bin_q[h] >= want : n < want && n + bin_n[h] >= want) {
          sh.border.before_count = n;
          sh.border.before_mass = q;
          sh.border.count = bin_n[h];
          sh.border.slot = 2 * threadIdx.x + h;
          sh.border.found = 1u;
        }
        n += bin_n[h];
        q += bin_q[h];
      }
      __syncthreads();
      const SampleBorder b = sh.border;
      if (!b.found) return 0ull;  // nothing to cut
      if (b.count > kSmShort) {
        cut(weigh, want);
        unsigned long long v = 0ull;
#pragma unroll
        for (int j = 0; j < kEach; ++j) v += mass[j];
        return block_sum(v);
      }
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (key_of[j] != 0u && slot_of(key_of[j]) == (int)b.slot) {
          const unsigned p = atomicAdd(&big.members, 1u);
          big.key[p] = key_of[j];
          big.place[p] = threadIdx.x * kEach + j;
          big.mass[p] = mass[j];
        }
      __syncthreads();
      const unsigned members = big.members;
      if (threadIdx.x < members) {
        const unsigned k = big.key[threadIdx.x], place = big.place[threadIdx.x];
        const unsigned long long m = big.mass[threadIdx.x];
        unsigned long long count = b.before_count, ahead = b.before_mass;
#pragma unroll 4
        for (unsigned j = 0; j < members; ++j) {
          const unsigned o = big.key[j];
          if (o > k || (o == k && big.place[j] < place)) {
            ++count;
            ahead += big.mass[j];
          }
        }
        // the last kept rank: what lies before it is below the wanted, what lies up to it is not
        if (weigh ? ahead < want && ahead + m >= want : count + 1ull == want) {
          big.cut_key = k;
          big.cut_place = place;
          big.cut_mass = ahead + m;
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kEach; ++j)
        if (key_of[j] < big.cut_key || (key_of[j] == big.cut_key && threadIdx.x * kEach + j > big.cut_place)) {
          key_of[j] = 0u;
          mass[j] = 0ull;
        }
      return big.cut_mass;
    };
    if (cut_count) {
      const unsigned long long v = cut_by_bins(false, (unsigned long long)top_k);
      if (whole == 0ull) whole = v;
    }
    if (by_mass) {
      if (whole == 0ull) {  // of the list
        unsigned long long v = 0ull;
#pragma unroll
        for (int j = 0; j < kEach; ++j) v += mass[j];
        whole = block_sum(v);
      }
      cut_by_bins(true, wanted(whole));
    }
    unsigned long long v = 0ull;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      if (key_of[j] != 0u) {
        const float x = sample_value(key_of[j]);
        if (!(weight(x, depth(x)) >= min_p)) mass[j] = 0ull;
      }
      v += mass[j];
    }
    unsigned long long upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long w = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += w;
    }
    if (lane == 31) sh.scan_mass[warp] = upto;
    __syncthreads();
    unsigned long long before = upto - v, total = 0ull;
    for (int w = 0; w < kSmWarps; ++w) {
      if (w < warp) before += sh.scan_mass[w];
      total += sh.scan_mass[w];
    }
    const unsigned long long target = target_of(total);
    if (target < before || target >= before + v) return true;
    int pick = -1;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      before += mass[j];
      if (pick < 0 && before > target) pick = j;
    }
    a.out[row] = sh.list_token[threadIdx.x * kEach + pick];
    return true;
  };

  if (top_k > 0 || by_mass) {
    auto all_bins = [&](float, float y, int& slot) {
      slot = bin_of(y);
      return true;
    };
    SampleBorder b;
    unsigned long long whole = 0ull;  // mass of all tokens: what top-p refers to without top-k
    if (top_k <= 0) {
      double sum = 0.0;  // integers below 2^53: exact
      every_token([&](float x) {
        if (x > -INFINITY) sum += (double)rintf(weight(x, depth(x)) * kSmOne);
      });
      unsigned long long q = (unsigned long long)sum;
      q = warp_sum64(q);
      if (lane < C) st_cluster_u64(cluster_addr(&sh.warp_mass[rank * kSmWarps + warp], lane), q);
      cluster_sync_all();
      for (int w = lane; w < C * kSmWarps; w += 32) whole += sh.warp_mass[w];
      whole = warp_sum64(whole);
    }
    // A cheap first stretch of the ranks: as many warps' maxima as top_k asks
    // for, or of the mass that top_p asks for, are that many tokens, so
    // everything ranked after them all is dropped. Then the same with the lanes' maxima.
    if (a.vocab <= kSmShort) {
      finish_in_list(-INFINITY, kSmBins, top_k > 0 && top_k < a.vocab, whole);
      return;
    }
    const unsigned long long want = top_k > 0 ? 0ull : wanted(whole);
    if (top_k <= kSmWarps * C / 2) {
      // found by one warp: all sixteen at it would take the issue slots of the SM's other rows
      if (warp == 0) {
        unsigned border = 0u;
        if (top_k > 0) {
          for (int bit = 31; bit >= kLowBits; --bit) {
            const unsigned c = border | 1u << bit;
            unsigned v = 0u;
#pragma unroll
            for (int j = 0; j < kTops; ++j) v += (unsigned)(tops[j] >> 32) >= c;
            if (__reduce_add_sync(0xffffffffu, v) >= (unsigned)top_k) border = c;
          }
        } else {
          unsigned long long q[kTops];
#pragma unroll
          for (int j = 0; j < kTops; ++j) {
            const float x = sample_value((unsigned)(tops[j] >> 32));
            q[j] = tops[j] != 0ull ? mass_of(weight(x, depth(x))) : 0ull;
          }
          for (int bit = 31; bit >= kLowBits; --bit) {
            const unsigned c = border | 1u << bit;
            unsigned long long v = 0ull;
#pragma unroll
            for (int j = 0; j < kTops; ++j) v += (unsigned)(tops[j] >> 32) >= c ? q[j] : 0ull;
            if (warp_sum64(v) >= want) border = c;
          }
        }
        if (lane == 0) sh.scan_cnt[0] = border;
      }
      __syncthreads();
      const unsigned border = sh.scan_cnt[0];
      // every value at or above the border's pattern (its low bits lack where bf16 has none: not above the value)
      if (border != 0u && finish_in_list(sample_value(border), kSmBins, top_k > 0, whole)) return;
    }
    if (top_k <= kSmList) {
      b = search(histogram(kSmBins, top_k <= 0, false, lane_tops, all_bins), kSmBins, top_k <= 0, (unsigned)top_k, want);
      if (b.found && finish_in_list(-INFINITY, (int)b.slot, top_k > 0, whole)) return;
    }
    const Slot s = histogram(kSmBins, by_mass, false, every_token, all_bins);
    kept_mass = all_mass;
    if (top_k > 0) {
      b = search(s, kSmBins, false, (unsigned)top_k, 0ull);
      if (b.found) refine(b, false, (unsigned)top_k, 0ull);
    }
    if (by_mass) {
      const unsigned long long mass = wanted(kept_mass);
      __syncthreads();
      if (threadIdx.x == 0) sh.border.found = 0u;
      cluster_sync_all();
      b = search(s, kSmBins, true, 0u, mass);
      if (b.found && finish_in_list(-INFINITY, (int)b.slot, false, kept_mass)) return;
      if (b.found) refine(b, true, 0u, mass);
    }
  }

  // ---- the kept tokens' mass, warp by warp in index order
  // 1 kept, 0 not, 2 equal to the border's value (kept if among its first `ties`)
  auto state_of = [&](float x, float y, float w) {
    if (!(x > -INFINITY) || !(w >= min_p)) return 0;
    if (bin1 == kSmBins) return 1;
    const int b = bin_of(y);
    if (b != bin1 || bin2 == kSmBins) return b <= bin1 ? 1 : 0;
    const int c = sub_of(y, bin1);
    if (c != bin2) return c < bin2 ? 1 : 0;
    const unsigned k = sample_key(x);
    return k != key ? (k > key ? 1 : 0) : 2;
  };
  unsigned ties_before = 0u;  // equal to the border's value and before this warp's tokens
  if (bin2 != kSmBins) {
    unsigned n = 0;
    each([&](const float (&x)[8], int) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = depth(x[j]);
        n += state_of(x[j], y, weight(x[j], y)) == 2;
      }
    });
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane < C) st_cluster_u32(cluster_addr(&sh.warp_ties[rank * kSmWarps + warp], lane), n);
    cluster_sync_all();
    for (int w = lane; w < rank * kSmWarps + warp; w += 32) ties_before += sh.warp_ties[w];
    ties_before = __reduce_add_sync(0xffffffffu, ties_before);
  }
  // f(masses of this lane's 8 tokens, the first one's index) over the warp's tokens, 256 at a time, until it says so
  auto kept = [&](auto&& f) {
    unsigned seen = ties_before;
    for (int i0 = warp * seg; i0 < (warp + 1) * seg; i0 += 256) {
      const int i = i0 + 8 * lane;
      unsigned long long q[8];
      unsigned tie = 0u;  // bit j: token j equals the border's value
      if (i < (warp + 1) * seg) {
        float x[8];
        sample_load8<T>(xs + i, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y = depth(x[j]), w = weight(x[j], y);
          const int st = state_of(x[j], y, w);
          q[j] = st != 0 ? mass_of(w) : 0ull;
          tie |= st == 2 ? 1u << j : 0u;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = 0ull;
      }
      if (__any_sync(0xffffffffu, tie != 0u)) {
        const unsigned mine = __popc(tie);
        unsigned n = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const unsigned u = __shfl_up_sync(0xffffffffu, n, o);
          if (lane >= o) n += u;
        }
        unsigned r = seen + n - mine;
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (tie >> j & 1u) {
            if (r >= ties) q[j] = 0ull;
            ++r;
          }
        seen += __shfl_sync(0xffffffffu, n, 31);
      }
      if (f(q, base + i)) return;
    }
  };
  unsigned long long sum = 0ull;
  kept([&](const unsigned long long (&q)[8], int) {
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += q[j];
    return false;
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane < C) st_cluster_u64(cluster_addr(&sh.warp_mass[rank * kSmWarps + warp], lane), sum);
  cluster_sync_all();  // the last access to another CTA's memory is before it
  unsigned long long before = 0ull, total = 0ull;
  for (int w = lane; w < C * kSmWarps; w += 32) {
    const unsigned long long m = sh.warp_mass[w];
    total += m;
    if (w < rank * kSmWarps + warp) before += m;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    total += __shfl_xor_sync(0xffffffffu, total, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
  const unsigned long long target = target_of(total);
  if (target < before || target >= before + sum) return;
  kept([&](const unsigned long long (&q)[8], int i) {
    unsigned long long m = 0ull;
#pragma unroll
    for (int j = 0; j < 8; ++j) m += q[j];
    unsigned long long upto = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + upto > target);
    if (past != 0u) {
      if (lane == __ffs(past) - 1) {
        unsigned long long run = before + upto - m;
        int pick = -1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          run += q[j];
          if (pick < 0 && run > target) pick = j;
        }
        a.out[row] = i + pick;
      }
      return true;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
    return false;
  });
}

}  // namespace qb
