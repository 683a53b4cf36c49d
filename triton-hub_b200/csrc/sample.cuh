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
// tokens of that very logit, a number of them -- and a histogram tells in which bin a threshold lies and how much lies
// before it: of counts over bins of 1/32 in the logit, of weights over bins in which the weight falls by 2^(1/32).
//   - When the bins down to it hold few tokens (the usual case of a peaked distribution or a small k), these are
//     listed, and one CTA finishes on the list by comparing its tokens pairwise.
//   - Otherwise the threshold is found within its bin: by comparing the bin's tokens pairwise, or, where they are too
//     many, by histograms over ever finer ranges of the order-preserving key.  A last pass sums what is kept, per
//     warp segment of the row; the segment that holds u * total is scanned for the token.
//
// A cluster of C CTAs holds a row in its shared memory, so the logits are read from memory once; cut at 16-byte boundaries
// of memory, a row of any alignment arrives in whole packets.  Memory is not what bounds it: 64 x 131072 bf16 are 2.6 us
// of bandwidth, but the greedy choice takes 14 us (load, maximum, barriers), top-k 50 22 us, the whole distribution 20 (some
// 16 fp64 instructions a token) and top-p 0.9 of a wide distribution 62 (the weight, and three shared-memory atomics a
// token).  One row of 32768 takes 6, 10, 6 and 16 us, chains of latencies.
#pragma once

#include "norm_common.cuh"
#include "norm_stage.cuh"

namespace b200norm {

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kSampleBins = 2 * kSampleThreads;  // two a thread
constexpr int kSampleMaxVocab = 1 << 18;
constexpr int kSampleMaxCluster = 8;
constexpr float kSampleBinsPerUnit = 32.f;
// A CTA with so many tokens bounds top-k's threshold by its threads' maxima before it counts: of 512 x 50257 bf16, k = 50,
// 69 -> 67 us; with 8192 tokens a CTA the bound costs more than it saves (1024 x 8192: 33 -> 35 us).
constexpr int kSampleBound = 16384;
constexpr int kSampleList = 256;  // tokens that are compared pairwise: all that may be drawn, or those of a threshold's bin

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
  int chunk;  // tokens of a row that a CTA holds: whole 16-byte packets
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
  float least;          // 42 to 64 temperatures below the maximum; lower logits count as this one
  const double* table;  // 2^(i / 16)

  // 256 + the weight, in units of 2^-44: 256 has just that ulp, so the addition rounds the weight, and the fraction field
  // of the sum is the integer wanted.
  static constexpr u64 kBias = 0x4070000000000000ull;
  static constexpr double kMagic = 6755399441055744.;  // 1.5 * 2^52: adding it rounds to an integer
  __device__ __forceinline__ u64 biased(float x, int& bin) const {
    const double y = (static_cast<double>(fmaxf(x, least)) - top) * scale;
    const double t = y + kMagic;
    const int n = __double2loint(t);
    const double g = y - (t - kMagic);
    bin = -2 * n - (g > 0. ? 1 : 0);
    double e = 1.2716085030349987e-09;
    e = fma(e, g, 1.467644462189871e-07);
    e = fma(e, g, 1.355080777749983e-05);
    e = fma(e, g, 0.000938384792486206);
    e = fma(e, g, 0.04332169878499661);
    e = fma(e, g, 1.0000000000000044);
    e *= table[n & 15];
    const double w = __hiloint2double(__double2hiint(e) + ((n >> 4) << 20), __double2loint(e));
    return static_cast<u64>(__double_as_longlong(w + 256.));
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    int n;
    return biased(x, n) - kBias;
  }
  // The number, 0 at the maximum, of the token's bin: floor(-2 y), bins in which weights differ by at most 2^(1/32).
  __device__ __forceinline__ int bin_of(float x) const {
    int bin;
    biased(x, bin);
    return bin;
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
  union {
    uint32_t bin[3][kSampleBins];  // a bin's weight or count: lo + (mid << 16) + (hi << 32)
    struct {
      u64 list[kSampleList];                       // this CTA's listed tokens: key, index
      u64 item[kSampleList], amount[kSampleList];  // the row's listed tokens
      u64 weight[C * kSampleWarps];     // per warp segment of the row: weight above the threshold ...
      uint32_t ties[C * kSampleWarps];  // ... and number of tokens at it
    };
  };
  float pending[kSampleWarps][32];  // logits that a warp has put side by side
  double table[16];
  u64 warp_total[kSampleWarps];
  float top[C];                     // per CTA: the largest logit
  u64 slice[2][C];  // per CTA: the sum of its share of the bins, and the tokens in them
  u64 found_above, found_here, found_tokens, rest;
  uint32_t found_key;
  int found_bin, segment, budget, listed;
  float warp_float[kSampleWarps];
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
  const uint4* packets;  // this CTA's part, in shared memory; -inf outside the row
  int n;                 // packets
  int seg;               // packets of a warp segment: warp w takes packets w * seg ... of the part
  int rank;
  int first;             // token index of this part's first element
  SampleShared<C>* sh;
  float top, temperature;
  Weigh weigh;
  int tid, lane, warp;

  // The part's i-th four values; -inf past its end.
  __device__ __forceinline__ void four(int i, float (&x)[4]) const {
    if (i >= n * (VEC / 4)) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = -INFINITY;
    } else if constexpr (VEC == 4) {
      Pack16<T>::unpack(ld_shared16(packets + i), x);
    } else {
      union { uint2 q; T v[4]; } u;
      u.q = reinterpret_cast<const uint2*>(packets)[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = to_f32(u.v[e]);
    }
  }
  // f(four values) for every four of packets begin .. end - 1, each by one of `threads` threads
  template <typename F>
  __device__ __forceinline__ void each_four(int begin, int end, int first, int threads, F f) const {
    constexpr int PARTS = VEC / 4;
    for (int i = begin * PARTS + first; i < end * PARTS; i += threads) {
      float x[4];
      four(i, x);
      f(x);
    }
  }
  // f(value, index in the part) for every element.  One element a turn: the passes that use it rarely do more than compare,
  // run once, and would spend longer fetching unrolled instructions than executing them.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    const T* values = reinterpret_cast<const T*>(packets);
#pragma unroll 1
    for (int i = tid; i < n * VEC; i += kSampleThreads) f(values[i], i);
  }

  // Tokens that few lanes of a warp have are put side by side and handed on 32 at a time: push(x, keep) by the whole warp,
  // then drain().  f(x, valid) is called by the whole warp.
  template <typename F>
  struct Side {
    float* slots;
    int lane, waiting;
    F f;
    __device__ __forceinline__ void push(float x, bool keep) {
      const uint32_t kept = __ballot_sync(0xffffffffu, keep);
      if (kept == 0) return;
      const int at = waiting + __popc(kept & ((1u << lane) - 1u));
      if (keep && at < 32) slots[at] = x;
      waiting += __popc(kept);
      if (waiting < 32) return;
      __syncwarp();
      const float full = slots[lane];
      __syncwarp();
      if (keep && at >= 32) slots[at - 32] = x;
      waiting -= 32;
      f(full, true);
    }
    __device__ __forceinline__ void drain() {
      __syncwarp();
      f(slots[lane], lane < waiting);
      __syncwarp();
    }
  };
  template <typename F>
  __device__ __forceinline__ Side<F> side(F f) const {
    return Side<F>{sh->pending[warp], lane, 0, f};
  }

  // The bin of a token, monotone in its logit: of counts by the distance from the maximum, of weights by the weight.  The
  // last one takes all that follows.
  template <bool WEIGHT>
  __device__ __forceinline__ int bin_of(float x) const {
    if constexpr (WEIGHT) return min(weigh.bin_of(x), kSampleBins - 1);
    else return static_cast<int>(fminf((top - x) * kSampleBinsPerUnit, static_cast<float>(kSampleBins - 1)));
  }
  // A logit below which no token of bins 0 .. b lies (fp32 errs by far less than half a bin).
  template <bool WEIGHT>
  __device__ __forceinline__ float bin_end(int b) const {
    if (b >= kSampleBins - 1) return -INFINITY;
    const float width = WEIGHT ? temperature * (0.69314718f / 32.f) : 1.f / kSampleBinsPerUnit;
    return top - width * static_cast<float>(b + 2) - 1e-5f * fabsf(top);
  }

  __device__ __forceinline__ void clear_bins() const {
    #pragma unroll
    for (int k = 0; k < 3; ++k) reinterpret_cast<u64*>(sh->bin[k])[tid] = 0ull;
    __syncthreads();
  }
  // 16 bits of a weight at a time, so that 2^16 tokens leave no carry and no addition has to return what it found: that is
  // several times as fast as a 64-bit addition, or a 32-bit one whose carry is looked for.
  __device__ __forceinline__ void add_to_bin(int b, u64 w) const {
    const uint32_t l = static_cast<uint32_t>(w), h = static_cast<uint32_t>(w >> 32);
    atomicAdd(&sh->bin[0][b], l & 0xffffu);
    atomicAdd(&sh->bin[1][b], l >> 16);
    if (h) atomicAdd(&sh->bin[2][b], h);
  }
  // The weights of the tokens above `floor`, or the counts of all, into bins 0 .. last; what lies beyond goes to the last bin
  // of all as one sum.
  template <bool WEIGHT>
  __device__ __forceinline__ void fill_bins(float floor, int last) const {
    clear_bins();
    u64 beyond = 0;
    if constexpr (WEIGHT) {
      each_four(0, n, tid, kSampleThreads, [&](const float (&x)[4]) {
        // all weights first, without a branch between: their chains of fp64 instructions overlap
        u64 w[4];
        int b[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] = weigh.biased(x[e], b[e]) - Weigh::kBias;
          w[e] = x[e] > floor ? w[e] : 0ull;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (b[e] <= last) add_to_bin(b[e], w[e]);
          else beyond += w[e];
        }
      });
    } else {
      const float end = static_cast<float>(last + 1) * (1.f / kSampleBinsPerUnit);
      each_four(0, n, tid, kSampleThreads, [&](const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          // the scale of the bins is a power of two: the comparison is that of the bin numbers
          if (top - x[e] < end) atomicAdd(&sh->bin[0][bin_of<false>(x[e])], 1u);
          else ++beyond;
        }
      });
    }
    beyond = warp_sum64(beyond);
    if (lane == 0) add_to_bin(kSampleBins - 1, beyond);
  }
  __device__ __forceinline__ static u64 bin_sum(u64 lo, u64 mid, u64 hi) { return lo + (mid << 16) + (hi << 32); }
  // An upper bound for the number of tokens with a weight in a bin: its sum over the least that one of them weighs.  Where that
  // is a few units it says nothing.
  __device__ __forceinline__ static u64 most_tokens(int b, u64 sum) {
    const float unit = exp2f(44.f - static_cast<float>(b + 1) / 32.f) * 0.999f;
    return sum == 0 ? 0ull : unit < 4096.f ? 1ull << 20 : static_cast<u64>(static_cast<float>(sum) / unit);
  }
  // The bin in which the running sum over the bins, `above` ahead of them, reaches what need_of(their total) says: into
  // found_bin, found_above (what lies before it), found_here and (TOKENS) found_tokens, an upper bound for the tokens down to
  // it.  It synchronises the row before and after: all CTAs' tokens are in the bins, and the bins may change again.  Each
  // CTA sums its share of the bins over the row.  MINE: this CTA's bins alone.
  template <bool TOKENS, bool MINE = C == 1, typename Need>
  __device__ __forceinline__ void locate(u64 above, Need need_of) const {
    constexpr int PER = MINE ? 2 : 1, SHARE = MINE ? kSampleBins : kSampleBins / C;  // bins a thread, a CTA
    u64 sum[PER], tokens[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) sum[i] = tokens[i] = 0;
    if constexpr (MINE) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int b = PER * tid + i;
        sum[i] = bin_sum(sh->bin[0][b], sh->bin[1][b], sh->bin[2][b]);
      }
    } else {
      row_sync<C>();
      if (tid < SHARE) {
        u64 part[3] = {0, 0, 0};
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int k = 0; k < 3; ++k)
            part[k] += static_cast<uint32_t>(ld_cluster_i32(cluster_map(smem_addr(&sh->bin[k][rank * SHARE + tid]), c)));
        sum[0] = bin_sum(part[0], part[1], part[2]);
      }
    }
    const int first_bin = MINE ? PER * tid : rank * SHARE + tid;
    u64 own = 0, own_tokens = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      own += sum[i];
      if (TOKENS) tokens[i] = most_tokens(first_bin + i, sum[i]);
      own_tokens += tokens[i];
    }
    auto scan = [&](u64 v, u64& total) {
      const u64 before = block_scan64(v, sh->warp_total, warp, lane);
      total = 0;
#pragma unroll
      for (int k = 0; k < kSampleWarps; ++k) total += sh->warp_total[k];
      return before;
    };
    u64 total, all_tokens = 0;
    u64 before = scan(own, total), tokens_before = TOKENS ? scan(own_tokens, all_tokens) : 0ull;
    if constexpr (!MINE) {
      if (tid < C) {  // thread c tells CTA c
        st_cluster_u64(cluster_map(smem_addr(&sh->slice[0][rank]), tid), total);
        st_cluster_u64(cluster_map(smem_addr(&sh->slice[1][rank]), tid), all_tokens);
      }
      row_sync<C>();
      total = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const u64 v = sh->slice[0][c];
        total += v;
        if (c < rank) {
          before += v;
          tokens_before += sh->slice[1][c];
        }
      }
    }
    const u64 need = need_of(total);
    before += above;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (before < need && before + sum[i] >= need) {
        const int b = first_bin + i;
        if constexpr (MINE) {
          sh->found_bin = b;
          sh->found_above = before;
          sh->found_here = sum[i];
          sh->found_tokens = tokens_before + tokens[i];
        } else {
#pragma unroll 1
          for (int c = 0; c < C; ++c) {
            st_cluster_u32(cluster_map(smem_addr(&sh->found_bin), c), static_cast<uint32_t>(b));
            st_cluster_u64(cluster_map(smem_addr(&sh->found_above), c), before);
            st_cluster_u64(cluster_map(smem_addr(&sh->found_here), c), sum[i]);
            st_cluster_u64(cluster_map(smem_addr(&sh->found_tokens), c), tokens_before + tokens[i]);
          }
        }
      }
      before += sum[i];
      tokens_before += tokens[i];
    }
    if constexpr (MINE) __syncthreads();
    else row_sync<C>();
  }

  // Lists the row's tokens that `pred` takes.  Returns how many there are; if they are at most kSampleList, the CTAs for
  // which `all` is set have them in sh->item, in any order.  A row_sync is due before the next listing.
  template <typename Pred>
  __device__ __forceinline__ int gather(bool all, Pred pred) const {
    if (tid == 0) sh->listed = 0;
    __syncthreads();
    each([&](T v, int i) {
      if (!pred(v, to_f32(v))) return;
      const int at = atomicAdd(&sh->listed, 1);
      if (at < kSampleList) sh->list[at] = (static_cast<u64>(token_key(v)) << 32) | static_cast<uint32_t>(first + i);
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

// Threads that share a token of a list of n in pairwise comparisons: a power of two, 2 to 16.
__device__ __forceinline__ int list_share(int n) { return n <= 32 ? 16 : n <= 64 ? 8 : n <= 128 ? 4 : 2; }
template <typename V>
__device__ __forceinline__ V share_sum(V v, int share) {
  for (int o = 1; o < share; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The threshold within bin found_bin of the first histogram, found_above lying before it: by finer histograms, over ranges of
// the order-preserving key, until one key or few enough tokens for a comparison by pairs are left.  Amounts are weights, of
// the tokens above `floor`, or (WEIGHT false) counts of all.  Every CTA of the row gets the result.
template <typename T, int C, bool WEIGHT>
__device__ __forceinline__ Threshold refine(const Row<T, C>& row, u64 need, float floor) {
  SampleShared<C>* sh = row.sh;
  const int tid = row.tid, b = sh->found_bin;
  u64 above = sh->found_above, here = sh->found_here;
  // A range of keys that holds the bin's: its ends in fp32, and 1e-5 of the maximum, by which they err less, to either side.
  const float margin = 1e-5f * fabsf(row.top);
  const float width = WEIGHT ? row.temperature * (0.69314718f / 32.f) : 1.f / kSampleBinsPerUnit;
  const float x1 = fminf(row.top - width * (static_cast<float>(b) - 0.5f) + margin, row.top);
  const float x0 = b == kSampleBins - 1 ? -INFINITY : row.top - width * (static_cast<float>(b) + 1.5f) - margin;
  uint32_t lo_key = token_key(from_f32<T>(x0)), hi_key = token_key(from_f32<T>(x1)) + 2;
  lo_key = lo_key > 1 ? lo_key - 2 : 0;
  auto inside = [&](float x, uint32_t k) {
    return k >= lo_key && k < hi_key && (!WEIGHT || x > floor) && row.template bin_of<WEIGHT>(x) == b;
  };
  const float unit = WEIGHT ? exp2f(44.f - static_cast<float>(b + 1) / 32.f) * 0.999f : 1.f;  // the least a token of the bin weighs
  Threshold th;
  while (hi_key - lo_key > 1) {
    if (unit >= 1.f && static_cast<float>(here) <= unit * kSampleList) {
      const int n = row.gather(true, [&](T v, float x) { return x >= x0 && x <= x1 && inside(x, token_key(v)); });
      if (n <= kSampleList) {
        __syncthreads();
        if (tid < n) sh->amount[tid] = WEIGHT ? row.weigh(key_logit<T>(static_cast<uint32_t>(sh->item[tid] >> 32))) : 1ull;
        __syncthreads();
        const int share = list_share(n), i = tid / share;
        const uint32_t key = i < n ? static_cast<uint32_t>(sh->item[i] >> 32) : 0u;
        u64 more = 0, same = 0;
        if (i < n) {
#pragma unroll 2
          for (int j = tid & (share - 1); j < n; j += share) {
            const uint32_t k = static_cast<uint32_t>(sh->item[j] >> 32);
            const u64 a = sh->amount[j];
            more += k > key ? a : 0ull;
            same += k == key ? a : 0ull;
          }
        }
        more = share_sum(more, share) + above;
        same = share_sum(same, share);
        if (i < n && more < need && need <= more + same) {  // the same result in all tokens of that key
          sh->found_key = key;
          sh->found_above = more;
        }
        row_sync<C>();
        lo_key = sh->found_key;
        above = sh->found_above;
        break;
      }
      row_sync<C>();
    }
    int shift = 0;
    while (((hi_key - 1 - lo_key) >> shift) >= static_cast<uint32_t>(kSampleBins)) ++shift;
    row.clear_bins();
    row.each([&](T v, int) {
      const float x = to_f32(v);
      if (!(x >= x0 && x <= x1)) return;
      const uint32_t k = token_key(v);
      if (inside(x, k)) row.add_to_bin(static_cast<int>((hi_key - 1 - k) >> shift), WEIGHT ? row.weigh(x) : 1ull);
    });
    row.template locate<false>(above, [&](u64) { return need; });
    above = sh->found_above;
    here = sh->found_here;
    const uint32_t span = 1u << shift;
    hi_key -= static_cast<uint32_t>(sh->found_bin) * span;
    lo_key = hi_key - lo_key > span ? hi_key - span : lo_key;
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
// weight that the prefix has to reach, or where that is 0 by top_p of the list's total), min-p, the draw.  Several threads
// a token; every sum runs over the whole list.
template <typename T, int C>
__device__ __forceinline__ void finish_list(const Row<T, C>& row, int n, int top_k, float top_p, u64 need, u64 least, float u,
                                            int64_t* token) {
  SampleShared<C>* sh = row.sh;
  const int tid = row.tid;
  const int share = list_share(n), i = tid / share, part = tid & (share - 1);
  __syncthreads();
  const u64 mine = i < n ? sh->item[i] : 0ull;
  const uint32_t key = static_cast<uint32_t>(mine >> 32), index = static_cast<uint32_t>(mine);
  const u64 full = i < n ? row.weigh(key_logit<T>(key)) : 0ull;
  u64 w = full;
  auto ahead = [&](u64 other) {  // `other` comes first in the order
    const uint32_t k = static_cast<uint32_t>(other >> 32);
    return k > key || (k == key && static_cast<uint32_t>(other) < index);
  };
  auto whole = [&](auto v) { return share_sum(v, share); };
  if (top_k > 0) {
    int rank = 0;
    if (i < n) {
#pragma unroll 2
      for (int j = part; j < n; j += share) rank += ahead(sh->item[j]) ? 1 : 0;
    }
    if (whole(rank) >= top_k) w = 0;
  }
  if (top_p < 1.f) {
    if (i < n && part == 0) sh->amount[i] = w;
    __syncthreads();
    u64 total = 0, before = 0;
    if (i < n) {
#pragma unroll 2
      for (int j = part; j < n; j += share) {
        const u64 a = sh->amount[j];
        total += a;
        before += ahead(sh->item[j]) ? a : 0ull;
      }
    }
    total = whole(total);
    before = whole(before);
    if (i < n && before >= (need ? need : prefix_weight(top_p, total))) w = 0;
    __syncthreads();
  }
  if (full < least) w = 0;
  if (i < n && part == 0) sh->amount[i] = w;
  __syncthreads();
  u64 total = 0, before = 0;
  if (i < n) {
#pragma unroll 2
    for (int j = part; j < n; j += share) {
      const u64 a = sh->amount[j];
      total += a;
      before += static_cast<uint32_t>(sh->item[j]) < index ? a : 0ull;
    }
  }
  total = whole(total);
  before = whole(before);
  if (i < n && part == 0) {
    const u64 target = draw_target(u, total);
    if (before <= target && target < before + w) *token = static_cast<int64_t>(index);
  }
}

template <typename T, int C>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const SampleParams p) {
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

  // The row's part into shared memory, and its maximum on the way (which a NaN takes over).  The parts are cut at
  // 16-byte boundaries of memory, so that a row of any alignment is loaded in whole packets but for its two ends.
  const T* logits = static_cast<const T*>(p.logits) + row_index * p.stride;
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(logits) & 15u) / sizeof(T));
  const int first = rank * p.chunk - lead;
  const int n = p.chunk / VEC;
  float best = -INFINITY;
  auto take = [&](int i, const uint4& q) {
    union { uint4 q; T v[VEC]; } pk;
    pk.q = q;
    reinterpret_cast<uint4*>(dyn)[i] = q;
#pragma unroll
    for (int e = 0; e < VEC; e += 2)
      asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(best) : "f"(to_f32(pk.v[e])), "f"(to_f32(pk.v[e + 1])));
  };
  const int i0 = first < 0 ? 1 : 0;                             // whole packets: i0 ...
  const int i1 = max(i0, min(n, (p.V - first) / VEC));  // ... to i1
  constexpr int kAhead = 4;
  for (int i = i0 + tid; i < i1; i += kAhead * kSampleThreads) {
    uint4 q[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k * kSampleThreads < i1) q[k] = ld_stream(reinterpret_cast<const uint4*>(logits + first) + i + k * kSampleThreads);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (i + k * kSampleThreads < i1) take(i + k * kSampleThreads, q[k]);
  }
  for (int i = tid; i < n - (i1 - i0); i += kSampleThreads) {  // the ends, and what lies outside the row
    const int at = i < i0 ? i : i + (i1 - i0);
    union { uint4 q; T v[VEC]; } pk;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const int t = first + at * VEC + e;
      pk.v[e] = t >= 0 && t < p.V ? logits[t] : from_f32<T>(-INFINITY);
    }
    take(at, pk.q);
  }
  const float mine = best;
  asm volatile("redux.sync.max.NaN.f32 %0, %0, 0xffffffff;" : "+f"(best));
  if (lane == 0) sh->warp_float[warp] = best;
  __syncthreads();
  if (tid < C) {  // thread c tells CTA c
    float m = -INFINITY;
    for (int k = 0; k < kSampleWarps; ++k) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(sh->warp_float[k]));
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
  // Rounded down: what is cut off weighs less than 2^-60 for certain, and the maximum never is.
  float cut = __fsub_rd(top, 42.f * temperature);
  const bool replaced = !(top - cut <= 64.f * temperature);
  if (replaced) {
    // A maximum of +inf: in the limit the infinite ones share everything.  A maximum so large that fp32 has no number
    // between 42 and 64 temperatures below it: logits are replaced by their differences from it, exact within a factor of
    // two of it, and of no weight beyond.
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
  row.n = n; row.seg = (n + kSampleWarps - 1) / kSampleWarps; row.rank = rank; row.first = first; row.sh = sh; row.top = top; row.temperature = temperature;
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
    int beyond = kSampleBins - 2;
    if (top_k <= kSampleThreads && n * VEC >= kSampleBound && !replaced) {
      // Of the largest logits that this CTA's threads have seen the k-th: k tokens are at or above it.
      row.clear_bins();
      atomicAdd(&sh->bin[0][row.template bin_of<false>(mine)], 1u);
      row.template locate<false, true>(0, [&](u64) { return need; });
      beyond = min(sh->found_bin, beyond);
    }
    row.template fill_bins<false>(floor, beyond);
    row.template locate<false>(0, [&](u64) { return need; });
    const int last = sh->found_bin;
    if (sh->found_above + sh->found_here <= kSampleList) {
      const int got = row.gather(rank == 0, [&](T, float x) { return x > -INFINITY && row.template bin_of<false>(x) <= last; });
      if (rank == 0) finish_list<T, C>(row, got, top_k, top_p, 0ull, least, u, token);
      if constexpr (C > 1) cluster_sync_all();  // rank 0 has read the other lists
      return;
    }
    th = refine<T, C, false>(row, need, floor);
    floor = key_logit<T>(th.key);
    floor_weight = row.weigh(floor);
  }
  if (use_p) {
    // The weights above top-k's threshold; at it, `ties` tokens more.
    // Tokens too light for min-p need no bins of their own, only their sum: when the prefix ends among them, it keeps all that
    // min-p does.  (A bin is floor(-32 log2 w); one more for the rounding of min-p's.)  64 x 131072 bf16, p = 0.95 and
    // min-p up to 0.02 a row: 50 -> 41 us.
    const int heavy = least_share > 0.f ? static_cast<int>(fminf(-32.f * log2f(least_share), 2.f * kSampleBins)) + 2 : kSampleBins;
    const bool light = heavy < kSampleBins - 2;
    row.template fill_bins<true>(floor, min(heavy, kSampleBins - 2));
    u64 total, need;
    row.template locate<true>(0, [&](u64 sum) {
      total = sum;
      return need = prefix_weight(top_p, total + th.ties * floor_weight);
    });
    if (need > total) {  // the prefix ends among the ties at top-k's threshold
      th.ties = (need - total + floor_weight - 1) / floor_weight;
    } else if (!light || sh->found_bin < kSampleBins - 1) {
      const int last = sh->found_bin;
      if (sh->found_tokens <= kSampleList / 2) {  // room for some of the bins beyond, which the test may take along
        const float end = row.template bin_end<true>(last);
        const int got = row.gather(rank == 0, [&](T, float x) { return x > floor && x >= end; });
        if (got <= kSampleList) {
          if (rank == 0) finish_list<T, C>(row, got, 0, top_p, need, least, u, token);
          if constexpr (C > 1) cluster_sync_all();  // rank 0 has read the other lists
          return;
        }
        row_sync<C>();
      }
      th = refine<T, C, true>(row, need, floor);
    }
  }

  // What is left, per warp segment of the row: the weight above the threshold and the tokens at it.
  const bool bounded = th.key != 0u;
  const float edge = bounded ? key_logit<T>(th.key) : -INFINITY;
  const u64 edge_weight = bounded ? row.weigh(edge) : 0ull;
  const bool use_ties = bounded && edge_weight >= least;
  // A logit below which min-p leaves nothing for certain (fp32 errs by far less than the margin).
  float skip = edge;
  if (least_share > 0.f) skip = fmaxf(skip, top + temperature * (logf(least_share) - 1e-3f) - 1e-5f * fabsf(top));
  const int seg = row.seg;
  {
    u64 sum = 0;
    uint32_t ties = 0;
    const int begin = min(warp * seg, n), end = min(begin + seg, n);
    if (!(skip > -INFINITY)) {
      uint32_t count = 0;
      row.each_four(begin, end, lane, 32, [&](const float (&x)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          int bin;
          sum += row.weigh.biased(x[e], bin);
        }
        count += 4;
      });
      sum -= count * Weigh::kBias;
    } else {
      auto queue = row.side([&](float x, bool valid) {
        const u64 w = valid ? row.weigh(x) : 0ull;
        sum += w >= least ? w : 0ull;
      });
      for (int i0 = begin * (VEC / 4); i0 < end * (VEC / 4); i0 += 32) {
        float x[4];
        row.four(i0 + lane < end * (VEC / 4) ? i0 + lane : INT_MAX, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          ties += bounded && x[e] == edge ? 1u : 0u;
          queue.push(x[e], x[e] > skip);
        }
      }
      queue.drain();
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
        *token = first + i;
        break;
      }
      before += w;
    }
  }
}

}  // namespace b200norm
