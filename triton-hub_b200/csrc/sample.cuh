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
// bits can tell apart, and 2^18 weights of up to 2^44 stay within 64 bits.  The exponentials are fp64 for the same reason: with
// 10^5 tokens in play an fp32 running sum puts the border between two tokens off by more than a rare token's width.
//
// The first k and the shortest prefix are both thresholds in the order: a key and, among tokens of that very
// key, a number of them.  Both are found without sorting, by histograms: bins of 1/64 below the maximum first,
// then, inside the bin that holds the threshold, ever finer ranges of the order-preserving key down to one key.
//
// A cluster of C CTAs holds a row in its shared memory, so the logits are read from memory once.  What
// bounds the kernel: the fp64 exponentials (17 instructions a token on 64 lanes per SM and cycle) and, for a
// few rows, the chain of passes and barriers.
#pragma once

#include "norm_common.cuh"
#include "norm_stage.cuh"

namespace b200norm {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2048;
constexpr int kSampleMaxVocab = 1 << 18;
constexpr int kSampleMaxCluster = 8;
constexpr float kSampleBinsPerUnit = 64.f;

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
constexpr u64 kSampleOne = 1ull << 44;

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

// round(2^44 exp((x - top) / temperature)), with scale = log2(e) / temperature.  2^y is 2^n * 2^f with |f| <= 1/2 and
// 2^f = exp(f ln 2) by its Taylor series to the 11th power: a remainder of (ln 2 / 2)^12 / 12! = 6e-15.
__device__ __forceinline__ u64 token_weight(float x, float top, double scale) {
  if (x == top) return kSampleOne;  // also a maximum of +inf
  const double y = (static_cast<double>(x) - static_cast<double>(top)) * scale;
  if (!(y > -46.)) return 0ull;
  constexpr double kMagic = 6755399441055744.;  // 1.5 * 2^52: adding it rounds to an integer
  const double t = y + kMagic;
  const int n = __double2loint(t);
  const double f = (y - (t - kMagic)) * 0.693147180559945309417;
  double e = 1. / 39916800.;
  e = fma(e, f, 1. / 3628800.);
  e = fma(e, f, 1. / 362880.);
  e = fma(e, f, 1. / 40320.);
  e = fma(e, f, 1. / 5040.);
  e = fma(e, f, 1. / 720.);
  e = fma(e, f, 1. / 120.);
  e = fma(e, f, 1. / 24.);
  e = fma(e, f, 1. / 6.);
  e = fma(e, f, 0.5);
  e = fma(e, f, 1.);
  e = fma(e, f, 1.);
  const double w = __hiloint2double(__double2hiint(e) + (n << 20), __double2loint(e));
  // 256 has an ulp of 2^-44: the sum's fraction field is the rounded weight
  return static_cast<u64>(__double_as_longlong(w + 256.)) & ((1ull << 52) - 1);
}

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
  u64 warp_total[kSampleWarps];
  u64 top[C];                              // per CTA: the largest key, and above it whether a NaN was seen
  u64 weight[C * kSampleWarps];            // per warp segment of the row: weight above the threshold ...
  uint32_t ties[C * kSampleWarps];         // ... and number of tokens at it
  u64 found_above, rest;
  int found_bin, segment, budget;
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
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
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

// A CTA's part of a row in shared memory, visited packet by packet.
template <typename T>
struct Chunk {
  const uint4* packets;
  int n;  // packets

  // f(value, index in the chunk), every element of packets begin .. end - 1, each by one of `threads` threads
  template <typename F>
  __device__ __forceinline__ void each(int begin, int end, int first, int threads, F f) const {
    constexpr int VEC = Pack16<T>::kElems;
    for (int i = begin + first; i < end; i += threads) {
      union { uint4 q; T v[VEC]; } u;
      u.q = ld_shared16(packets + i);
#pragma unroll
      for (int e = 0; e < VEC; ++e) f(u.v[e], i * VEC + e);
    }
  }
};

// The threshold of a row: tokens whose key is above `key`, and `ties` of those at it.
struct Threshold {
  uint32_t key;
  u64 ties;
};

// Finds the key at which the amount of the tokens in descending order of key reaches `need`: the amount above the
// key is below `need`, that down to it is not.  Amounts are weights (WEIGHT) or counts.  Tokens below `floor` do not
// take part.  need is at least 1 and at most the amount of all that take part.
template <typename T, int C, bool WEIGHT>
__device__ __forceinline__ Threshold find_threshold(const Chunk<T>& chunk, SampleShared<C>* sh, u64 need, uint32_t floor, float top,
                                    double scale, int warp, int lane) {
  const int tid = threadIdx.x;
  auto bin_of = [&](float x) {  // bins of equal width below the maximum; monotone in x
    const float d = (top - x) * kSampleBinsPerUnit;
    return x == top ? 0 : (d < static_cast<float>(kSampleBins - 1) ? static_cast<int>(d) : kSampleBins - 1);
  };
  uint32_t lo_key = 0, hi_key = 0;  // the threshold lies in [lo_key, hi_key), once the first level has found its bin
  int shift = 0;
  u64 above = 0;
  for (int level = 0;; ++level) {
    for (int i = tid; i < kSampleBins / 4; i += kSampleThreads) {
      reinterpret_cast<uint4*>(sh->lo)[i] = make_uint4(0, 0, 0, 0);
      if (WEIGHT) reinterpret_cast<uint4*>(sh->hi)[i] = make_uint4(0, 0, 0, 0);
    }
    __syncthreads();
    chunk.each(0, chunk.n, tid, kSampleThreads, [&](T v, int) {
      const uint32_t k = token_key(v);
      if (k < floor) return;
      int b;
      const float x = to_f32(v);
      if (level == 0) {
        b = bin_of(x);
      } else {
        if (k < lo_key || k >= hi_key) return;
        b = static_cast<int>((hi_key - 1 - k) >> shift);
      }
      if constexpr (WEIGHT) {
        const u64 w = token_weight(x, top, scale);
        if (w == 0) return;
        // 64-bit addition in two native 32-bit ones: the low word's carry joins the high word
        const uint32_t wl = static_cast<uint32_t>(w);
        const uint32_t old = atomicAdd(&sh->lo[b], wl);
        const uint32_t wh = static_cast<uint32_t>(w >> 32) + (old + wl < old ? 1u : 0u);
        if (wh) atomicAdd(&sh->hi[b], wh);
      } else {
        atomicAdd(&sh->lo[b], 1u);
      }
    });
    row_sync<C>();
    // four bins a thread, over all CTAs of the row
    u64 bin[4] = {0, 0, 0, 0};
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
    u64 before = above + block_scan64(bin[0] + bin[1] + bin[2] + bin[3], sh->warp_total, warp, lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (before < need && before + bin[i] >= need) {
        sh->found_bin = 4 * tid + i;
        sh->found_above = before;
      }
      before += bin[i];
    }
    row_sync<C>();  // the result is in place, and every CTA has read this one's bins
    const int b = sh->found_bin;
    above = sh->found_above;
    if (level == 0) {
      // The keys of bin b, by bisection over the monotone bin_of: hi_key is the first key above it, lo_key its lowest.
      const uint32_t top_key = token_key(from_f32<T>(top));
      auto first_key = [&](int want) {  // the lowest key whose bin is at most `want`
        uint32_t a = 0, z = top_key;
        while (a < z) {
          const uint32_t m = a + (z - a) / 2;
          const float x = key_logit<T>(m);
          if (x == x && bin_of(x) <= want) z = m;  // the keys of negative NaNs lie below every number
          else a = m + 1;
        }
        return a;
      };
      lo_key = first_key(b);
      hi_key = b == 0 ? top_key + 1 : first_key(b - 1);
    } else {
      const uint32_t width = 1u << shift;
      hi_key = hi_key - static_cast<uint32_t>(b) * width;
      lo_key = hi_key - lo_key > width ? hi_key - width : lo_key;
    }
    if (hi_key - lo_key <= 1) break;
    shift = 0;
    while (((hi_key - 1 - lo_key) >> shift) >= static_cast<uint32_t>(kSampleBins)) ++shift;
  }
  Threshold th;
  th.key = lo_key;
  const u64 one = WEIGHT ? token_weight(key_logit<T>(lo_key), top, scale) : 1ull;
  th.ties = (need - above + one - 1) / one;
  return th;
}

template <typename T, int C>
__global__ void __launch_bounds__(kSampleThreads) sample_kernel(const SampleParams p) {
  constexpr int VEC = Pack16<T>::kElems;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ SampleShared<C> shared;
  SampleShared<C>* sh = &shared;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = C > 1 ? static_cast<int>(cluster_cta_rank()) : 0;
  const int64_t row = blockIdx.x / C;
  grid_dependency_sync();
  trigger_dependents();
  if constexpr (C > 1) cluster_sync_all();  // every CTA of the row runs: its shared memory may be written

  const float temperature = p.temperature_v ? p.temperature_v[row] : p.temperature;
  const float top_p = p.top_p_v ? p.top_p_v[row] : p.top_p;
  const float min_p = p.min_p_v ? p.min_p_v[row] : p.min_p;
  const int top_k = p.top_k_v ? p.top_k_v[row] : p.top_k;
  const float u = p.uniform[row];

  // The row's part into shared memory, and its largest key on the way; past the row's end -inf.
  const T* src = static_cast<const T*>(p.logits) + row * p.stride + (int64_t)rank * p.chunk;
  const int here = max(0, min(p.chunk, p.V - rank * p.chunk));
  const Chunk<T> chunk{reinterpret_cast<const uint4*>(dyn), p.chunk / VEC};
  const bool packed = (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
  uint32_t best = 0;
  bool nan = false;
  for (int i = tid; i < chunk.n; i += kSampleThreads) {
    union { uint4 q; T v[VEC]; } pk;
    if (packed && (i + 1) * VEC <= here) {
      pk.q = ld_stream(reinterpret_cast<const uint4*>(src) + i);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) pk.v[e] = i * VEC + e < here ? src[i * VEC + e] : from_f32<T>(-INFINITY);
    }
    reinterpret_cast<uint4*>(dyn)[i] = pk.q;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float x = to_f32(pk.v[e]);
      nan = nan || x != x;
      best = max(best, token_key(pk.v[e]));
    }
  }
  best = __reduce_max_sync(0xffffffffu, best);
  nan = __any_sync(0xffffffffu, nan);
  if (lane == 0) sh->warp_total[warp] = (static_cast<u64>(nan) << 32) | best;
  __syncthreads();
  if (tid < C) {  // thread c tells CTA c
    u64 m = 0;
    for (int k = 0; k < kSampleWarps; ++k) {
      const u64 v = sh->warp_total[k];
      m = max(m, v);  // a NaN's bit outweighs every key
    }
    if constexpr (C == 1) sh->top[0] = m;
    else st_cluster_u64(cluster_map(smem_addr(&sh->top[rank]), tid), m);
  }
  row_sync<C>();
  u64 most = 0;
#pragma unroll
  for (int c = 0; c < C; ++c) most = max(most, sh->top[c]);
  const float top = key_logit<T>(static_cast<uint32_t>(most));
  if ((most >> 32) != 0 || top == -INFINITY) {  // a NaN, or nothing to choose from
    if (rank == 0 && tid == 0) p.tokens[row] = -1;
    return;  // the same in every CTA of the row, and none reads another's memory after this
  }

  const double scale = 1.4426950408889634074 / static_cast<double>(temperature);
  Threshold th{0u, 0ull};
  float least = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;  // the likeliest token always stays
  if (!(temperature > 0.f)) {  // greedy
    th = Threshold{static_cast<uint32_t>(most), 1ull};
    least = 0.f;
  } else {
    if (top_k > 0 && top_k < p.V)
      th = find_threshold<T, C, false>(chunk, sh, static_cast<u64>(top_k), 0u, top, scale, warp, lane);
    if (top_p < 1.f) {
      // total weight of what top-k left
      u64 sum = 0;
      chunk.each(0, chunk.n, tid, kSampleThreads, [&](T v, int) {
        const uint32_t k = token_key(v);
        if (k > th.key) sum += token_weight(to_f32(v), top, scale);
      });
      sum = warp_sum64(sum);
      __syncthreads();
      if (lane == 0) sh->warp_total[warp] = sum;
      __syncthreads();
      if (tid < C) {
        u64 s = 0;
        for (int k = 0; k < kSampleWarps; ++k) s += sh->warp_total[k];
        if constexpr (C == 1) sh->weight[0] = s;
        else st_cluster_u64(cluster_map(smem_addr(&sh->weight[rank]), tid), s);
      }
      row_sync<C>();
      u64 total = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) total += sh->weight[c];
      if (th.key != 0u) total += th.ties * token_weight(key_logit<T>(th.key), top, scale);
      const double want = ceil(static_cast<double>(top_p) * static_cast<double>(total));
      const u64 need = want < 1. ? 1ull : min(static_cast<u64>(want), total);
      const Threshold tp = find_threshold<T, C, true>(chunk, sh, need, th.key, top, scale, warp, lane);
      th = Threshold{tp.key, tp.key == th.key ? min(th.ties, tp.ties) : tp.ties};
    }
  }
  // min-p as a lowest weight
  const double least_w = static_cast<double>(least) * static_cast<double>(kSampleOne);
  const u64 tie_weight = th.key != 0u ? token_weight(key_logit<T>(th.key), top, temperature > 0.f ? scale : 1.) : 0ull;
  const double draw_scale = temperature > 0.f ? scale : 1.;
  auto weight_above = [&](T v) -> u64 {
    if (token_key(v) <= th.key) return 0ull;
    const u64 w = token_weight(to_f32(v), top, draw_scale);
    return static_cast<double>(w) >= least_w ? w : 0ull;
  };
  const bool use_ties = th.key != 0u && static_cast<double>(tie_weight) >= least_w;

  // What is left, per warp segment of the row.
  const int seg = (chunk.n + kSampleWarps - 1) / kSampleWarps;  // packets
  {
    u64 sum = 0;
    uint32_t ties = 0;
    chunk.each(min(warp * seg, chunk.n), min((warp + 1) * seg, chunk.n), lane, 32, [&](T v, int) {
      sum += weight_above(v);
      ties += token_key(v) == th.key ? 1u : 0u;
    });
    sum = warp_sum64(sum);
    ties = __reduce_add_sync(0xffffffffu, ties);
    if constexpr (C > 1) cluster_sync_all();  // sh->weight's earlier values have been read
    else __syncthreads();
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
    uint32_t n[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = lane * PER + i;
      n[i] = s < C * kSampleWarps ? sh->ties[s] : 0u;
      ties += n[i];
    }
    u64 tie_before = warp_scan64(ties, lane) - ties;
    u64 w[PER], own = 0;
    u64 allowed[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int s = lane * PER + i;
      allowed[i] = th.ties > tie_before ? min(th.ties - tie_before, static_cast<u64>(n[i])) : 0ull;
      tie_before += n[i];
      w[i] = (s < C * kSampleWarps ? sh->weight[s] : 0ull) + allowed[i] * tie_weight;
      own += w[i];
    }
    const u64 inc = warp_scan64(own, lane);
    const u64 total = __shfl_sync(0xffffffffu, inc, 31);
    const double t = static_cast<double>(u) * static_cast<double>(total);
    u64 target = t > 0. ? static_cast<u64>(t) : 0ull;
    if (target >= total) target = total - 1;
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
  const int each = (end - begin + kSampleThreads - 1) / kSampleThreads;
  const int b0 = min(begin + tid * each, end), b1 = min(b0 + each, end);
  const T* values = reinterpret_cast<const T*>(dyn);
  u64 ties = 0;
  if (use_ties)
    for (int i = b0; i < b1; ++i) ties += token_key(values[i]) == th.key ? 1u : 0u;
  const u64 tie_before = block_scan64(ties, sh->warp_total, warp, lane);
  auto weight_at = [&](int i, u64& tie) -> u64 {
    if (use_ties && token_key(values[i]) == th.key) return tie++ < budget ? tie_weight : 0ull;
    return weight_above(values[i]);
  };
  u64 sum = 0, tie = tie_before;
  for (int i = b0; i < b1; ++i) sum += weight_at(i, tie);
  u64 before = block_scan64(sum, sh->warp_total, warp, lane);
  if (before <= rest && rest < before + sum) {
    tie = tie_before;
    for (int i = b0; i < b1; ++i) {
      const u64 w = weight_at(i, tie);
      if (rest < before + w) {
        p.tokens[row] = (int64_t)rank * p.chunk + i;
        break;
      }
      before += w;
    }
  }
}

}  // namespace b200norm
