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
// No sort: the last kept rank is found by a histogram. Masses are integers
// (w 2^44, so a sum of up to 2^18 tokens fits 64 bits), which makes every sum
// exact and the result independent of the order of the atomics.
//
// A cluster of 8 CTAs holds the row in shared memory, so it is read once.
// Bound by latency for few rows (a dozen passes over 20 thousand shared-memory
// values a CTA, each ended by a cluster barrier), by bytes for many.
//  1. (maximum, its lowest index): the answer of greedy rows (T = 0)
//  2. tokens counted and weighed in 1024 bins of equal width in (max - x) / T,
//     1/32 each (the last takes the rest): monotone in x, and unlike bins of
//     x's own bits not a handful of crowded ones. Each CTA sums its share of the
//     bins over the cluster and finds whether the border lies there.
//  3. the border's bin again in 1024 sub-bins; a sub-bin whose tokens are not
//     all equal is split by 8 bits of the value's ordered pattern at a time
//  4. the kept mass of every warp's stretch of indexes, the stretch that the
//     target falls in, the token in it
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

struct alignas(16) SampleShared {
  unsigned cnt[kSmBins], lo[kSmBins], hi[kSmBins], kor[kSmBins], kand[kSmBins];
  unsigned long long warp_mass[kSmCluster * kSmWarps];  // every warp of the cluster
  unsigned warp_ties[kSmCluster * kSmWarps];
  unsigned long long seg_mass[kSmCluster];  // of every CTA's bins
  unsigned seg_cnt[kSmCluster];
  unsigned long long top[kSmCluster];  // (ordered value, inverted index) of every CTA's maximum
  unsigned long long scan_mass[kSmWarps];
  unsigned scan_cnt[kSmWarps];
  SampleBorder border;
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
  return sizeof(SampleShared) + 16 + (size_t)slice * item;
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
  pdl_wait();
  pdl_trigger();

  // ---- the row's slice into shared memory (filled up with -inf), and its maximum
  const T* src = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.vocab + base;
  const int live = max(0, min(a.slice, a.vocab - base));
  constexpr int kPer = 16 / sizeof(T);
  const int vec = (reinterpret_cast<uintptr_t>(src) & 15) == 0 ? live / kPer : 0;
  for (int i = threadIdx.x; i < vec; i += kSmThreads) reinterpret_cast<uint4*>(xs)[i] = __ldcs(reinterpret_cast<const uint4*>(src) + i);
  for (int i = vec * kPer + threadIdx.x; i < a.slice; i += kSmThreads) xs[i] = i < live ? src[i] : sample_lowest<T>();
  __syncthreads();

  auto each = [&](auto&& f) {  // f(tokens 8 lane .. + 7 of the warp's next 256, the first one's place in the slice)
    for (int i = warp * seg + 8 * lane; i < (warp + 1) * seg; i += 256) {
      float x[8];
      sample_load8<T>(xs + i, x);
      f(x, i);
    }
  };
  unsigned long long best = 0ull;
  each([&](const float (&x)[8], int i) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const unsigned long long k = ((unsigned long long)sample_key(x[j]) << 32) | (unsigned)~(unsigned)(base + i + j);
      best = k > best ? k : best;
    }
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
    best = other > best ? other : best;
  }
  if (lane == 0) sh.scan_mass[warp] = best;
  __syncthreads();
  if (threadIdx.x < C) {
    for (int w = 0; w < kSmWarps; ++w) best = sh.scan_mass[w] > best ? sh.scan_mass[w] : best;
    st_cluster_u64(cluster_addr(&sh.top[rank], threadIdx.x), best);
  }
  cluster_sync_all();
  for (int c = 0; c < C; ++c) best = sh.top[c] > best ? sh.top[c] : best;
  const unsigned top_key = (unsigned)(best >> 32);
  const float top = sample_value(top_key);

  const float temperature = a.temperature ? a.temperature[row] : a.temperature_all;
  if (top_key == 0u || !(temperature > 0.f)) {  // nothing to draw, or greedy
    if (rank == 0 && threadIdx.x == 0) {
      if (top_key == 0u) report_error(a.err, DEV_BAD_LOGITS);
      a.out[row] = top_key == 0u ? -1 : (int64_t)(unsigned)~(unsigned)best;
    }
    return;  // the same for the whole cluster, and no CTA's memory is read after the barrier
  }
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all;
  const float min_p = fminf(a.min_p ? a.min_p[row] : a.min_p_all, 1.f);
  const float inv_t = fminf(1.f / temperature, 3.402823466e38f);

  // (max - x) / T, correctly rounded but for rare last bits; weights of it.
  auto depth = [&](float x) {
    if (x == top) return 0.f;
    const float d = fminf(top - x, 3.402823466e38f);
    const float y = d * inv_t;
    return y < 128.f ? fmaf(fmaf(-y, temperature, d), inv_t, y) : y;
  };
  auto weight = [&](float y) { return expf(-y); };
  auto mass_of = [](float w) { return (unsigned long long)__float2ull_rn(w * kSmOne); };
  auto bin_of = [](float y) { return (int)fminf(y * kSmBinsPerUnit, (float)(kSmBins - 1)); };
  auto sub_of = [](float y, int bin) {
    const float f = (fminf(y, 64.f) * kSmBinsPerUnit - (float)bin) * (float)kSmBins;
    return (int)fminf(fmaxf(f, 0.f), (float)(kSmBins - 1));
  };

  const bool by_mass = top_p < 1.f;

  // Tokens of the cluster counted (and weighed) in `bins` slots: member(x, y,
  // slot) says whether a token counts, and where. Thread i < bins / 8 comes back
  // with slot rank * bins / 8 + i: its sums over the cluster and what lies before.
  struct Slot {
    unsigned long long mass, before_mass;
    unsigned count, before_count, key_or, key_and;
  };
  unsigned long long all_mass = 0ull;  // of the last histogram
  auto histogram = [&](int bins, bool keys, auto&& member) {
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
    each([&](const float (&x)[8], int) {
      int at = -1;
      unsigned n = 0;
      unsigned long long q = 0ull;
      auto flush = [&] {
        if (at < 0) return;
        atomicAdd(&sh.cnt[at], n);
        const unsigned ql = (unsigned)q;
        unsigned qh = (unsigned)(q >> 32);
        if (ql != 0u) qh += atomicAdd(&sh.lo[at], ql) + ql < ql;  // the carry
        if (qh != 0u) atomicAdd(&sh.hi[at], qh);
      };
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!(x[j] > -INFINITY)) continue;
        const float y = depth(x[j]);
        int slot;
        if (!member(x[j], y, slot)) continue;
        if (slot != at) {  // equal neighbours add up first
          flush();
          at = slot;
          n = 0;
          q = 0ull;
        }
        ++n;
        if (by_mass) q += mass_of(weight(y));
        if (keys) {
          atomicOr(&sh.kor[slot], sample_key(x[j]));
          atomicAnd(&sh.kand[slot], sample_key(x[j]));
        }
      }
      flush();
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
    SampleBorder b = search(histogram(kSmBins, true, [&](float, float y, int& slot) {
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
        b = search(histogram(256, true, [&](float x, float y, int& slot) {
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
  if (top_k > 0 || by_mass) {
    const Slot s = histogram(kSmBins, false, [&](float, float y, int& slot) {
      slot = bin_of(y);
      return true;
    });
    kept_mass = all_mass;
    if (top_k > 0) {
      const SampleBorder b = search(s, kSmBins, false, (unsigned)top_k, 0ull);
      if (b.found) refine(b, false, (unsigned)top_k, 0ull);
    }
    if (by_mass) {
      const unsigned long long want = max(1ull, (unsigned long long)ceil((double)fmaxf(top_p, 0.f) * (double)kept_mass));
      __syncthreads();
      if (threadIdx.x == 0) sh.border.found = 0u;
      cluster_sync_all();
      const SampleBorder b = search(s, kSmBins, true, 0u, want);
      if (b.found) refine(b, true, 0u, want);
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
        n += state_of(x[j], y, weight(y)) == 2;
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
          const float y = depth(x[j]), w = weight(y);
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
  const double u = (double)a.uniforms[row];
  unsigned long long target = u > 0.0 ? (unsigned long long)(fmin(u, 1.0) * (double)total) : 0ull;
  if (target >= total) target = total - 1ull;  // the maximum's own weight keeps total above 0
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
