// Choice of a token from a row of logits with given random numbers: temperature, top-k, top-p, min-p.
//
//   weight   w_i = exp((l_i - max l) / temperature)
//   order    larger logits first, equal ones by index
//   top-k    the first k tokens of that order
//   top-p    of those, every token before which less than p of their total weight lies
//   min-p    of those, the tokens with w_i >= min_p (w of the likeliest is 1)
//   draw     the lowest index i at which the running sum of the kept weights, in index order, exceeds u * total
//
// Weights are held as integers, round(w * 2^44).  Integer sums are exact in any order and split, so the drawn
// token does not depend on how a row is divided over threads and CTAs, nor on the order of the shared-memory
// atomics, and two runs agree.  2^-45 of the likeliest token's weight is far below what a random number of 24
// bits can tell apart, and 2^18 weights of up to 2^44 stay within 64 bits.  The exponentials are fp64 for the same
// reason: with 10^5 tokens in play an fp32 running sum puts the border between two tokens off by more than a
// rare token's width.
//
// Nothing is sorted.  The first k and the shortest prefix are thresholds in the order -- a logit and, among the
// tokens of that very logit, a number of them -- and a histogram over bins of 1/64 below the maximum tells in
// which bin a threshold lies and how much lies before it.
//   - When the bins down to it hold few tokens (the usual case of a peaked distribution or a small k), these are
//     listed, and one CTA finishes on the list by comparing its tokens pairwise.
//   - Otherwise the threshold is found within its bin: by comparing the bin's tokens pairwise, or, where they are too
//     many, by histograms over ever finer ranges of the order-preserving key.  A last pass sums what is kept, per
//     warp segment of the row; the segment that holds u * total is scanned for the token.
//
// A cluster of C CTAs holds a row in its shared memory, so the logits are read from memory once.
#pragma once

#include "norm_common.cuh"
#include "norm_stage.cuh"

namespace b200norm {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;  // four a thread
constexpr int kSampleMaxVocab = 1 << 18;
constexpr int kSampleMaxCluster = 8;
constexpr float kSampleBinsPerUnit = 64.f;
// Tokens that are compared pairwise: all that may be drawn from, or those of a threshold's bin.  512^2 comparisons are
// 1024 a thread, about as long as two further histograms.
constexpr int kSampleFinish = 256, kSampleList = 512;

struct SampleParams {
  const void* logits;
  int64_t stride;        // elements
  const float* uniform;  // (M,)
  const float *temperature_v, *top_p_v, *min_p_v;  // (M,) each, or null: the scalars below
  const int* top_k_v;
  float temperature, top_p, min_p;
  int top_k;
  int64_t* tokens;  // (M,)
  int64_t M;
  int V;
  int chunk;  // tokens of a row that a CTA holds: a multiple of 16 bytes
};

using u64 = unsigned long long;

// Order-preserving integer of a storage type's number; -0 counts as +0.
template <typename T>
__device__ __forceinline__ uint32_t token_key(T v) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t b = __float_as_uint(static_cast<float>(v) + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
  } else {
    uint32_t b = reinterpret_cast<const uint16_t&>(v);
    if (b == 0x8000u) b = 0u;
    return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
  }
}
template <typename T>
__device__ __forceinline__ float key_logit(uint32_t k) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
  } else {
    const uint16_t b = static_cast<uint16_t>((k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu));
    return to_f32(reinterpret_cast<const T&>(b));
  }
}

// round(2^44 exp((x - top) / temperature)).  With y = 16 log2(e) (x - top) / temperature = n + g, n whole and |g| <= 1/2:
// 2^(y / 16) = 2^(n / 16) 2^(g / 16), the first factor from a table of the sixteen 2^(i / 16) and an exponent, the second by
// the polynomial of degree 5 that meets it at six Chebyshev points (within 5e-15).  Logits further than 42 temperatures
// below the maximum weigh less than 2^-60, which rounds to 0, like -inf.
struct Weigh {
  double top, scale;    // y = (x - top) * scale: exactly 0 at the maximum, whose weight is exactly 2^44
  float least;          // logits down from here weigh nothing
  const double* table;  // 2^(i / 16)

  __device__ __forceinline__ u64 operator()(float x) const {
    const double y = x > least ? (static_cast<double>(x) - top) * scale : -976.;
    constexpr double kMagic = 6755399441055744.;  // 1.5 * 2^52: adding it rounds to an integer
    const double t = y + kMagic;
    const int n = __double2loint(t);
    const double g = y - (t - kMagic);
    double e = 1.2716085030349987e-09;
    e = fma(e, g, 1.467644462189871e-07);
    e = fma(e, g, 1.355080777749983e-05);
    e = fma(e, g, 0.000938384792486206);
    e = fma(e, g, 0.04332169878499661);
    e = fma(e, g, 1.0000000000000044);
    e *= table[n & 15];
    const double w = __hiloint2double(__double2hiint(e) + ((n >> 4) << 20), __double2loint(e));
    // 256 has an ulp of 2^-44: the sum's fraction field is the rounded weight
    return static_cast<u64>(__double_as_longlong(w + 256.)) & ((1ull << 52) - 1);
  }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 warp_scan64(u64 v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 a = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += a;
  }
  return v;
}

template <int C>
struct SampleShared {
  uint32_t lo[kSampleBins], hi[kSampleBins];  // a bin's weight (64 bits in two words) or, in lo, its count
  double table[16];
  u64 warp_total[kSampleWarps];
  float top[C];                  // per CTA: the largest logit
  u64 weight[C * kSampleWarps];  // per warp segment of the row: weight above the threshold ...
  uint32_t ties[C * kSampleWarps];  // ... and number of tokens at it
  u64 list[kSampleList];            // this CTA's listed tokens: key, index
  u64 item[kSampleList], amount[kSampleList];  // the row's listed tokens
  float pending[kSampleWarps][64];             // kept logits a warp has yet to weigh
  u64 found_above, rest;
  uint32_t found_key;
  int found_bin, down_to, inside, segment, budget, listed;
};

template <int C>
__device__ __forceinline__ void row_sync() {
  if constexpr (C == 1) __syncthreads();
  else cluster_sync_all();
}

__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint4 ld_cluster16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ u64 ld_cluster_u64(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ int ld_cluster_i32(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Exclusive prefix over the CTA's threads.
__device__ __forceinline__ u64 block_scan64(u64 v, u64* totals, int warp, int lane) {
  const u64 inc = warp_scan64(v, lane);
  __syncthreads();  // the previous use of `totals` is over
  if (lane == 31) totals[warp] = inc;
  __syncthreads();
  u64 before = 0;
#pragma unroll
  for (int k = 0; k < kSampleWarps; ++k) before += k < warp ? totals[k] : 0ull;
  return before + inc - v;
}

// A row, as one CTA of its cluster sees it.
template <typename T, int C>
struct Row {
  static constexpr int VEC = Pack16<T>::kElems;
  const uint4* packets;  // this CTA's part, in shared memory; past the row's end -inf
  int n;                 // packets
  int rank, chunk;
  SampleShared<C>* sh;
  float top;
  Weigh weigh;
  int tid, lane, warp;

  // f(value, index in the chunk) for every element of packets begin .. end - 1, each by one of `threads` threads
  template <typename F>
  __device__ __forceinline__ void each(int begin, int end, int first, int threads, F f) const {
    for (int i = begin + first; i < end; i += threads) {
      union { uint4 q; T v[VEC]; } u;
      u.q = ld_shared16(packets + i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f(u.v[e], i * VEC + e);
    }
  }

  __device__ __forceinline__ int bin_of(float x) const {  // bins of equal width below the maximum; monotone in x
    return static_cast<int>(fminf((top - x) * kSampleBinsPerUnit, static_cast<float>(kSampleBins - 1)));
  }

  __device__ __forceinline__ void clear_bins(bool weights) const {
    for (int i = tid; i < kSampleBins / 4; i += kSampleThreads) {
      reinterpret_cast<uint4*>(sh->lo)[i] = make_uint4(0, 0, 0, 0);
      if (weights) reinterpret_cast<uint4*>(sh->hi)[i] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
  }
  template <bool WEIGHT>
  __device__ __forceinline__ void add_to_bin(int b, float x) const {
    if constexpr (WEIGHT) {
      const u64 w = weigh(x);
      if (w == 0) return;
      // 64-bit addition in two native 32-bit ones: the low word's carry joins the high word
      const uint32_t wl = static_cast<uint32_t>(w);
      const uint32_t old = atomicAdd(&sh->lo[b], wl);
      const uint32_t wh = static_cast<uint32_t>(w >> 32) + (old + wl < old ? 1u : 0u);
      if (wh) atomicAdd(&sh->hi[b], wh);
    } else {
      atomicAdd(&sh->lo[b], 1u);
    }
  }
  // This thread's four bins, summed over the row's CTAs.  Behind it a row_sync is due before the bins change.
  template <bool WEIGHT>
  __device__ __forceinline__ void read_bins(u64 (&bin)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) bin[i] = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      uint4 l, h = make_uint4(0, 0, 0, 0);
      if constexpr (C == 1) {
        l = reinterpret_cast<const uint4*>(sh->lo)[tid];
        if (WEIGHT) h = reinterpret_cast<const uint4*>(sh->hi)[tid];
      } else {
        l = ld_cluster16(cluster_map(smem_addr(&sh->lo[4 * tid]), c));
        if (WEIGHT) h = ld_cluster16(cluster_map(smem_addr(&sh->hi[4 * tid]), c));
      }
      bin[0] += (static_cast<u64>(h.x) << 32) + l.x;
      bin[1] += (static_cast<u64>(h.y) << 32) + l.y;
      bin[2] += (static_cast<u64>(h.z) << 32) + l.z;
      bin[3] += (static_cast<u64>(h.w) << 32) + l.w;
    }
  }
  // The bin in which the running sum, `before` ahead of this thread's bins, reaches `need`: into found_bin, found_above.
  __device__ __forceinline__ void find_bin(const u64 (&bin)[4], u64 before, u64 need) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < need && before + bin[i] >= need) {
        sh->found_bin = 4 * tid + i;
        sh->found_above = before;
      }
      before += bin[i];
    }
  }

  // Lists the row's tokens that `pred` takes.  Returns how many there are; if they are at most kSampleList, the CTAs for
  // which `all` is set have them in sh->item, in any order.  A row_sync is due before the next listing.
  template <typename Pred>
  __device__ __forceinline__ int gather(bool all, Pred pred) const {
    if (tid == 0) sh->listed = 0;
    __syncthreads();
    each(0, n, tid, kSampleThreads, [&](T v, int i) {
      if (!pred(to_f32(v))) return;
      const int at = atomicAdd(&sh->listed, 1);
      if (at < kSampleList) sh->list[at] = (static_cast<u64>(token_key(v)) << 32) | static_cast<uint32_t>(rank * chunk + i);
    });
    row_sync<C>();
    int total = 0, from[C + 1];
#pragma unroll
    for (int c = 0; c < C; ++c) {
      from[c] = total;
      total += C == 1 ? sh->listed : ld_cluster_i32(cluster_map(smem_addr(&sh->listed), c));
    }
    from[C] = total;
    if (total <= kSampleList && all && tid < total) {
      u64 it = 0;
#pragma unroll
      for (int c = 0; c < C; ++c)
        if (tid >= from[c] && tid < from[c + 1])
          it = C == 1 ? sh->list[tid] : ld_cluster_u64(cluster_map(smem_addr(&sh->list[tid - from[c]]), c));
      sh->item[tid] = it;
    }
    return total;
  }
};

// A threshold in the order: the tokens whose key is above `key`, and `ties` of those at it.
struct Threshold {
  uint32_t key;
  u64 ties;
};

// The threshold within bin found_bin of the first histogram, found_above lying before it: by comparing the bin's tokens
// pairwise if `few` says that they are not too many, by finer histograms otherwise.  Amounts are weights, of the tokens
// above `floor`, or (WEIGHT false) counts of all.  Every CTA of the row gets the result.
template <typename T, int C, bool WEIGHT>
__device__ __forceinline__ Threshold refine(const Row<T, C>& row, u64 need, float floor, bool few) {
  SampleShared<C>* sh = row.sh;
  const int tid = row.tid, b = sh->found_bin;
  u64 above = sh->found_above;
  Threshold th;
  if (few) {
    const int n = row.gather(true, [&](float x) { return (!WEIGHT || x > floor) && row.bin_of(x) == b; });
    if (n <= kSampleList) {
      __syncthreads();
      const uint32_t key = tid < n ? static_cast<uint32_t>(sh->item[tid] >> 32) : 0u;
      if (tid < n) sh->amount[tid] = WEIGHT ? row.weigh(key_logit<T>(key)) : 1ull;
      __syncthreads();
      if (tid < n) {
        u64 more = above, same = 0;
        for (int j = 0; j < n; ++j) {
          const uint32_t k = static_cast<uint32_t>(sh->item[j] >> 32);
          const u64 a = sh->amount[j];
          if (k > key) more += a;
          if (k == key) same += a;
        }
        if (more < need && need <= more + same) {  // the same result in all tokens of that key
          sh->found_key = key;
          sh->found_above = more;
        }
      }
      row_sync<C>();
      th.key = sh->found_key;
      const u64 one = WEIGHT ? row.weigh(key_logit<T>(th.key)) : 1ull;
      th.ties = (need - sh->found_above + one - 1) / one;
      return th;
    }
    row_sync<C>();
  }
  // The keys of bin b, by bisection over the monotone bin_of: hi_key is the first key above it, lo_key its lowest.
  const uint32_t top_key = token_key(from_f32<T>(row.top));
  auto first_key = [&](int want) {  // the lowest key whose bin is at most `want`
    uint32_t a = 0, z = top_key;
    while (a < z) {
      const uint32_t m = a + (z - a) / 2;
      const float x = key_logit<T>(m);
      if (x == x && row.bin_of(x) <= want) z = m;  // the keys of negative NaNs lie below every number
      else a = m + 1;
    }
    return a;
  };
  uint32_t lo_key = first_key(b), hi_key = b == 0 ? top_key + 1 : first_key(b - 1);
  while (hi_key - lo_key > 1) {
    int shift = 0;
    while (((hi_key - 1 - lo_key) >> shift) >= static_cast<uint32_t>(kSampleBins)) ++shift;
    row.clear_bins(WEIGHT);
    row.each(0, row.n, tid, kSampleThreads, [&](T v, int) {
      const uint32_t k = token_key(v);
      if (k >= lo_key && k < hi_key && (!WEIGHT || to_f32(v) > floor))
        row.template add_to_bin<WEIGHT>(static_cast<int>((hi_key - 1 - k) >> shift), to_f32(v));
    });
    row_sync<C>();
    u64 bin[4];
    row.template read_bins<WEIGHT>(bin);
    row.find_bin(bin, above + block_scan64(bin[0] + bin[1] + bin[2] + bin[3], sh->warp_total, row.warp, row.lane), need);
    row_sync<C>();  // the result is in place, and every CTA has read this one's bins
    above = sh->found_above;
    const uint32_t width = 1u << shift;
    hi_key -= static_cast<uint32_t>(sh->found_bin) * width;
    lo_key = hi_key - lo_key > width ? hi_key - width : lo_key;
  }
  th.key = lo_key;
  const u64 one = WEIGHT ? row.weigh(key_logit<T>(lo_key)) : 1ull;
  th.ties = (need - above + one - 1) / one;
  return th;
}

// f * total for 0 < f < 1, rounded down or up; the product of a float's 24 bits and 64 is formed whole.
__device__ __forceinline__ u64 share_of(float f, u64 total, bool up) {
  const uint32_t bits = __float_as_uint(f), e = bits >> 23;
  const u64 m = e ? (bits & 0x7fffffu) | 0x800000u : bits;
  const int s = 150 - static_cast<int>(e ? e : 1u);  // f = m / 2^s, s >= 24
  const u64 lo = total * m, hi = __umul64hi(total, m);
  u64 q, rest;
  if (s < 64) {
    q = (hi << (64 - s)) | (lo >> s);
    rest = lo & ((1ull << s) - 1);
  } else {
    const int t = s - 64;
    q = t < 64 ? hi >> t : 0ull;
    rest = lo | (t < 64 ? hi & ((1ull << t) - 1) : hi);
  }
  return q + (up && rest ? 1ull : 0ull);
}
// The weight that a prefix has to reach for top-p < 1, of `total`.
__device__ __forceinline__ u64 prefix_weight(float top_p, u64 total) {
  return top_p > 0.f ? max(1ull, share_of(top_p, total, true)) : 1ull;
}
__device__ __forceinline__ u64 draw_target(float u, u64 total) {
  return u > 0.f ? (u < 1.f ? share_of(u, total, false) : total - 1) : 0ull;
}

// Finishes a row on the n listed tokens sh->item, which hold all that can be drawn: top-k (0: none), top-p (by `need`, the
// weight that the prefix has to reach, or where that is 0 by top_p of the list's total), min-p, the draw.  One thread a
// token; every sum runs over the whole list.
template <typename T, int C>
__device__ __forceinline__ void finish_list(const Row<T, C>& row, int n, int top_k, float top_p, u64 need, u64 least, float u,
                                            int64_t* token) {
  SampleShared<C>* sh = row.sh;
  const int tid = row.tid;
  __syncthreads();
  const u64 mine = tid < n ? sh->item[tid] : 0ull;
  const uint32_t key = static_cast<uint32_t>(mine >> 32), index = static_cast<uint32_t>(mine);
  const u64 full = tid < n ? row.weigh(key_logit<T>(key)) : 0ull;
  u64 w = full;
  auto ahead = [&](u64 other) {  // `other` comes first in the order
    const uint32_t k = static_cast<uint32_t>(other >> 32);
    return k > key || (k == key && static_cast<uint32_t>(other) < index);
  };
  if (top_k > 0 && tid < n) {
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += ahead(sh->item[j]) ? 1 : 0;
    if (rank >= top_k) w = 0;
  }
  if (top_p < 1.f) {
    if (tid < n) sh->amount[tid] = w;
    __syncthreads();
    if (tid < n) {
      u64 total = 0, before = 0;
      for (int j = 0; j < n; ++j) {
        const u64 a = sh->amount[j];
        total += a;
        if (ahead(sh->item[j])) before += a;
      }
      if (before >= (need ? need : prefix_weight(top_p, total))) w = 0;
    }
    __syncthreads();
  }
  if (full < least) w = 0;
  if (tid < n) sh->amount[tid] = w;
  __syncthreads();
  if (tid < n) {
    u64 total = 0, before = 0;
    for (int j = 0; j < n; ++j) {
      const u64 a = sh->amount[j];
      total += a;
      if (static_cast<uint32_t>(sh->item[j]) < index) before += a;
    }
    const u64 target = draw_target(u, total);
    if (before <= target && target < before + w) *token = static_cast<int64_t>(index);
  }
}

template <typename T, int C>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleParams p) {
  constexpr int VEC = Pack16<T>::kElems;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ SampleShared<C> shared;
  SampleShared<C>* sh = &shared;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = C > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  const int64_t row_index = blockIdx.x / C;
  if (tid < 16) sh->table[tid] = exp2(tid / 16.);
  grid_dependency_sync();
  trigger_dependents();
  if constexpr (C > 1) cluster_sync_all();  // every CTA of the row runs: its shared memory may be written

  float temperature = p.temperature_v ? p.temperature_v[row_index] : p.temperature;
  const float top_p = p.top_p_v ? p.top_p_v[row_index] : p.top_p;
  const float min_p = p.min_p_v ? p.min_p_v[row_index] : p.min_p;
  const int top_k = p.top_k_v ? p.top_k_v[row_index] : p.top_k;
  const float u = p.uniform[row_index];

  // The row's part into shared memory, and its maximum on the way (which a NaN takes over).
  const T* src = static_cast<const T*>(p.logits) + row_index * p.stride + (int64_t)rank * p.chunk;
  const int here = max(0, min(p.chunk, p.V - rank * p.chunk));
  const int n = p.chunk / VEC;
  const bool packed = (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
  float best = -INFINITY;
  for (int i = tid; i < n; i += kSampleThreads) {
    union { uint4 q; T v[VEC]; } pk;
    if (packed && (i + 1) * VEC <= here) {
      pk.q = ld_stream(reinterpret_cast<const uint4*>(src) + i);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) pk.v[e] = i * VEC + e < here ? src[i * VEC + e] : from_f32<T>(-INFINITY);
    }
    reinterpret_cast<uint4*>(dyn)[i] = pk.q;
#pragma unroll
    for (int e = 0; e < VEC; e += 2) {
      const float a = to_f32(pk.v[e]), b = to_f32(pk.v[e + 1]);
      asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(best) : "f"(best), "f"(a), "f"(b));
    }
  }
  asm volatile("redux.sync.max.NaN.f32 %0, %0, 0xffffffff;" : "+f"(best));
  if (lane == 0) sh->pending[0][warp] = best;
  __syncthreads();
  if (tid < C) {  // thread c tells CTA c
    float m = -INFINITY;
    for (int k = 0; k < kSampleWarps; ++k) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(sh->pending[0][k]));
    if constexpr (C == 1) sh->top[0] = m;
    else st_cluster_f32(cluster_map(smem_addr(&sh->top[rank]), tid), m);
  }
  row_sync<C>();
  float top = -INFINITY;
#pragma unroll
  for (int c = 0; c < C; ++c) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(sh->top[c]));
  if (!(top > -INFINITY)) {  // a NaN, or nothing to choose from
    if (rank == 0 && tid == 0) p.tokens[row_index] = -1;
    return;  // the same in every CTA of the row, and none reads another's memory after this
  }
  top += 0.f;  // -0 is +0
  const bool greedy = !(temperature > 0.f);
  temperature = greedy ? 1.f : fminf(temperature, 1e30f);  // at 1e30 every finite logit a model gives weighs the same
  // Rounded down: what is cut off weighs less than 2^-60 for certain, the maximum never is, and what is left has y > -976.
  float cut = __fsub_rd(top, 42.f * temperature);
  if (top == INFINITY || cut == -INFINITY) {
    // The limit of a maximum of +inf: the infinite ones share everything.  A maximum next to the lowest number: all finite
    // logits lie within a factor of two of it, so that their differences from it are exact.
    for (int i = tid; i < n * VEC; i += kSampleThreads) {
      T* v = reinterpret_cast<T*>(dyn) + i;
      const float x = to_f32(*v);
      *v = from_f32<T>(top == INFINITY ? (x == INFINITY ? 0.f : -INFINITY) : x - top);
    }
    top = 0.f;
    cut = -42.f * temperature;
    __syncthreads();
  }

  Row<T, C> row;
  row.packets = reinterpret_cast<const uint4*>(dyn);
  row.n = n; row.rank = rank; row.chunk = p.chunk; row.sh = sh; row.top = top;
  row.tid = tid; row.lane = lane; row.warp = warp;
  row.weigh.top = static_cast<double>(top);
  row.weigh.scale = 16. * 1.4426950408889634074 / static_cast<double>(temperature);
  row.weigh.least = cut;
  row.weigh.table = sh->table;

  // min-p as a lowest weight; the likeliest token always stays
  const float least_share = greedy || !(min_p > 0.f) ? 0.f : fminf(min_p, 1.f);
  const u64 least = static_cast<u64>(ceil(static_cast<double>(least_share) * static_cast<double>(row.weigh(top))));
  const bool use_k = !greedy && top_k > 0 && top_k < p.V, use_p = !greedy && top_p < 1.f;
  int64_t* token = p.tokens + row_index;

  Threshold th{0u, 0ull};
  if (greedy) th = Threshold{token_key(from_f32<T>(top)), 1ull};
  float floor = -INFINITY;
  u64 floor_weight = 0;
  if (use_k) {
    const u64 need = static_cast<u64>(top_k);
    row.clear_bins(false);
    row.each(0, n, tid, kSampleThreads, [&](T v, int) { row.template add_to_bin<false>(row.bin_of(to_f32(v)), 0.f); });
    row_sync<C>();
    u64 bin[4];
    row.template read_bins<false>(bin);
    u64 before = block_scan64(bin[0] + bin[1] + bin[2] + bin[3], sh->warp_total, warp, lane);
    row.find_bin(bin, before, need);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // how many tokens the bins down to the threshold's hold, and that one alone
      if (before < need && before + bin[i] >= need) {
        sh->down_to = static_cast<int>(before + bin[i]);
        sh->inside = static_cast<int>(bin[i]);
      }
      before += bin[i];
    }
    row_sync<C>();
    const int last = sh->found_bin, inside = sh->inside;
    if (sh->down_to <= kSampleFinish) {
      const int got = row.gather(rank == 0, [&](float x) { return row.bin_of(x) <= last; });
      if (rank == 0) finish_list<T, C>(row, got, top_k, top_p, 0ull, least, u, token);
      if constexpr (C > 1) cluster_sync_all();  // rank 0 has read the other lists
      return;
    }
    th = refine<T, C, false>(row, need, -INFINITY, inside <= kSampleList);
    floor = key_logit<T>(th.key);
    floor_weight = row.weigh(floor);
  }
  if (use_p) {
    // The weights above top-k's threshold; at it, `ties` tokens more.
    row.clear_bins(true);
    row.each(0, n, tid, kSampleThreads, [&](T v, int) {
      const float x = to_f32(v);
      if (x > floor) row.template add_to_bin<true>(row.bin_of(x), x);
    });
    row_sync<C>();
    u64 bin[4];
    row.template read_bins<true>(bin);
    const u64 before = block_scan64(bin[0] + bin[1] + bin[2] + bin[3], sh->warp_total, warp, lane);
    u64 total = 0;
#pragma unroll
    for (int k = 0; k < kSampleWarps; ++k) total += sh->warp_total[k];
    const u64 need = prefix_weight(top_p, total + th.ties * floor_weight);
    if (need > total) {  // the prefix ends among the ties at top-k's threshold
      th.ties = (need - total + floor_weight - 1) / floor_weight;
      row_sync<C>();
    } else {
      row.find_bin(bin, before, need);
      row_sync<C>();
      // How many tokens the bins down to the threshold's hold, from above: a bin's weight over the least that one of its
      // tokens weighs.  Weights of a few units say nothing.
      const int last = sh->found_bin;
      const float per_bin = 1.f / (kSampleBinsPerUnit * temperature);
      float count = 0.f, inside = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int b = 4 * tid + i;
        const float unit = expf(-static_cast<float>(b + 1) * per_bin) * 17592186044416.f * 0.999f;
        const float c = b > last || bin[i] == 0 ? 0.f : unit < 4096.f ? 1e9f : static_cast<float>(bin[i]) / unit;
        count += c;
        if (b == last) inside = c;
      }
      count = warp_sum(count);
      inside = warp_sum(inside);
      if (lane == 0) {
        sh->pending[warp][0] = count;
        sh->pending[warp][1] = inside;
      }
      __syncthreads();
      count = inside = 0.f;
#pragma unroll
      for (int k = 0; k < kSampleWarps; ++k) {
        count += sh->pending[k][0];
        inside += sh->pending[k][1];
      }
      if (count <= static_cast<float>(kSampleFinish)) {
        const int got = row.gather(rank == 0, [&](float x) { return x > floor && row.bin_of(x) <= last; });
        if (got <= kSampleList) {
          if (rank == 0) finish_list<T, C>(row, got, 0, top_p, need, least, u, token);
          if constexpr (C > 1) cluster_sync_all();  // rank 0 has read the other lists
          return;
        }
        row_sync<C>();
      }
      th = refine<T, C, true>(row, need, floor, inside <= static_cast<float>(kSampleList));
    }
  }

  // What is left, per warp segment of the row: the weight above the threshold and the tokens at it.
  const bool bounded = th.key != 0u;
  const float edge = bounded ? key_logit<T>(th.key) : -INFINITY;
  const u64 edge_weight = bounded ? row.weigh(edge) : 0ull;
  const bool use_ties = bounded && edge_weight >= least;
  // A logit below which min-p leaves nothing for certain (fp32 errs by far less than the margin).
  float skip = edge;
  if (least_share > 0.f) skip = fmaxf(skip, top + temperature * (logf(least_share) - 1e-3f) - fabsf(top) * 1e-5f);
  const int seg = (n + kSampleWarps - 1) / kSampleWarps;  // packets
  {
    u64 sum = 0;
    uint32_t ties = 0;
    const int begin = min(warp * seg, n), end = min(begin + seg, n);
    if (!(skip > -INFINITY)) {
      row.each(begin, end, lane, 32, [&](T v, int) { sum += row.weigh(to_f32(v)); });
    } else {
      // The kept ones are put side by side first, 32 at a time, since often a warp would weigh a few at a time.
      float* mine = sh->pending[warp];
      int waiting = 0;
      auto add = [&](float x, bool there) {
        const u64 w = there ? row.weigh(x) : 0ull;
        sum += w >= least ? w : 0ull;
      };
      __syncthreads();  // the counts above have been read
      for (int i0 = begin; i0 < end; i0 += 32) {
        union { uint4 q; T v[VEC]; } pk;
        const bool there = i0 + lane < end;
        if (there) pk.q = ld_shared16(row.packets + i0 + lane);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float x = there ? to_f32(pk.v[e]) : -INFINITY;
          ties += bounded && x == edge ? 1u : 0u;
          const uint32_t kept = __ballot_sync(0xffffffffu, x > skip);
          if (kept == 0) continue;
          if (x > skip) mine[waiting + __popc(kept & ((1u << lane) - 1u))] = x;
          waiting += __popc(kept);
          if (waiting >= 32) {
            __syncwarp();
            const float now = mine[lane], rest = mine[lane + 32];
            __syncwarp();
            mine[lane] = rest;
            waiting -= 32;
            add(now, true);
            __syncwarp();
          }
        }
      }
      __syncwarp();
      add(lane < waiting ? mine[lane] : 0.f, lane < waiting);
    }
    sum = warp_sum64(sum);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if (lane < C) {
      const int at = rank * kSampleWarps + warp;
      if constexpr (C == 1) {
        sh->weight[at] = sum;
        sh->ties[at] = use_ties ? ties : 0u;
      } else {
        st_cluster_u64(cluster_map(smem_addr(&sh->weight[at]), lane), sum);
        st_cluster_u32(cluster_map(smem_addr(&sh->ties[at]), lane), use_ties ? ties : 0u);
      }
    }
  }
  row_sync<C>();
  // No CTA touches another's memory from here on.  The segment in which the drawn token lies: one warp.
  if (warp == 0) {
    constexpr int PER = (C * kSampleWarps + 31) / 32;
    u64 ties = 0;
    uint32_t here_n[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = lane * PER + i;
      here_n[i] = s < C * kSampleWarps ? sh->ties[s] : 0u;
      ties += here_n[i];
    }
    u64 tie_before = warp_scan64(ties, lane) - ties;
    u64 w[PER], allowed[PER], own = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = lane * PER + i;
      allowed[i] = th.ties > tie_before ? min(th.ties - tie_before, static_cast<u64>(here_n[i])) : 0ull;
      tie_before += here_n[i];
      w[i] = (s < C * kSampleWarps ? sh->weight[s] : 0ull) + allowed[i] * edge_weight;
      own += w[i];
    }
    const u64 inc = warp_scan64(own, lane);
    const u64 target = draw_target(u, __shfl_sync(0xffffffffu, inc, 31));
    u64 before = inc - own;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (before <= target && target < before + w[i]) {
        sh->segment = lane * PER + i;
        sh->rest = target - before;
        sh->budget = static_cast<int>(allowed[i]);
      }
      before += w[i];
    }
  }
  __syncthreads();
  if (sh->segment / kSampleWarps != rank) return;
  // The token within the segment: consecutive tokens per thread, a scan of the ties, a scan of the weights.
  const int begin = (sh->segment % kSampleWarps) * seg * VEC, end = min(begin + seg * VEC, p.chunk);
  const u64 rest = sh->rest, budget = static_cast<u64>(sh->budget);
  const int share = (end - begin + kSampleThreads - 1) / kSampleThreads;
  const int b0 = min(begin + tid * share, end), b1 = min(b0 + share, end);
  const T* values = reinterpret_cast<const T*>(dyn);
  u64 ties = 0;
  if (use_ties) {
    for (int i = b0; i < b1; ++i) ties += to_f32(values[i]) == edge ? 1u : 0u;
    ties = block_scan64(ties, sh->warp_total, warp, lane);
  }
  auto weight_at = [&](int i, u64& tie) -> u64 {
    const float x = to_f32(values[i]);
    if (use_ties && x == edge) return tie++ < budget ? edge_weight : 0ull;
    const u64 w = x > edge || !bounded ? row.weigh(x) : 0ull;
    return w >= least ? w : 0ull;
  };
  u64 sum = 0, tie = ties;
  for (int i = b0; i < b1; ++i) sum += weight_at(i, tie);
  u64 before = block_scan64(sum, sh->warp_total, warp, lane);
  if (before <= rest && rest < before + sum) {
    tie = ties;
    for (int i = b0; i < b1; ++i) {
      const u64 w = weight_at(i, tie);
      if (rest < before + w) {
        *token = (int64_t)rank * p.chunk + i;
        break;
      }
      before += w;
    }
  }
}

}  // namespace b200norm
