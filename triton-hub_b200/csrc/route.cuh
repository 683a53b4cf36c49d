// Choice of experts from router logits, with per-expert counts and a balance loss, forward and backward.
//
//   p = softmax(l) over E experts;  the k largest logits are chosen, ties to the lower index;
//   gate = p of the chosen, or (normalize) p / sum of the chosen p
//   over the n live tokens:  f_e = counts_e / (n k),  P_e = sum p_e / n,  loss = E sum_e f_e P_e
//   backward, f held constant:  c_e = dloss E f_e / n
//     plain gates       dl = p (c + dgate - (sum p c + sum_chosen gate dgate)),  dgate 0 outside the choice
//     normalized gates  dl = p (c - sum p c) + gate (dgate - sum_chosen gate dgate)
//
// A token is not live when its mask is 0 or when all its logits are -inf: it chooses nothing (experts -1,
// gates 0), is not counted, and its gradient is 0.  An expert whose logit is -inf is never chosen; when
// fewer than k others exist, the slots left over hold -1 and gate 0.
//
// A warp takes a token; lane i holds the EPL neighbouring experts from i * EPL on, so the lowest of several
// lanes with one maximum also has the lowest index.  Reading the logits once is all that memory asks for (65536 x 128
// fp32: 6 us); what bounds the forward is the instructions of the choice, the exponentials and the sums, 475 a token
// (44 us, 37 of them in route_fwd_kernel), and the backward (17 us for 11 us of traffic; 183 a token) their share of it.  Column sums of p
// stay in registers over all of a warp's tokens and meet once per CTA, in shared memory; counts are shared-memory integer
// atomics, whose order cannot show; the CTAs' partial rows are added in one fixed order.
#pragma once

#include "norm_common.cuh"
#include "norm_stage.cuh"

namespace b200norm {

constexpr int kRouteThreads = 512;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteBwdThreads = 256;
constexpr int kRouteBwdWarps = kRouteBwdThreads / 32;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 32;
constexpr int kRouteMaxCluster = 8;

struct RouteParams {
  const void* logits;
  int64_t stride;       // elements
  const uint8_t* mask;  // (T,) or null
  float* gates;         // (T, k)
  int* experts;         // (T, k)
  float* lse;           // (T,) log of the softmax's denominator; -inf marks a token that is not live
  int* counts;          // (E + 1): per expert, then the number of live tokens
  int* kept;            // the same once more, for a backward whose caller gives `counts` away; may be null
  float* loss;
  float* part_p;  // (gridDim.x, columns) partial sums of p
  int* part_n;    // (gridDim.x, columns) partial counts
  int* part_live; // (gridDim.x,) partial numbers of live tokens
  int columns;    // E rounded up to whole 16-byte packets
  // backward
  const float* dgates;  // (T, k) or null
  int64_t dgates_stride;
  const float* dloss;  // scalar or null
  void* dlogits;       // (T, E) contiguous
  int64_t T;
  int E, k, normalize, parts;
  int cluster;  // CTAs of the forward's one cluster, which finishes by itself; 0: route_finish_kernel does
};

// exp(d) of a difference d <= 0 from the maximum, in two instructions: good to 2 ulp, and to |d| ulp more for the product with log2 e
// and its rounding, which expf does without (at d = -10, where a gate is below 5e-5, 7e-7 of it).  Below 2^-126 it is 0.
__device__ __forceinline__ float exp_below(float d) { return ex2_fast(d * kLog2e); }

// Order-preserving integer of a float; -0 counts as +0.  -inf maps to kKeyNegInf, 0 is below every number.
constexpr uint32_t kKeyNegInf = 0x007fffffu;
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}

// Lane's EPL logits of one token; experts past E read as -inf.  `packed`: EPL divides E and the rows are
// aligned, so a lane's experts are whole vectors.
template <typename T, int EPL>
__device__ __forceinline__ void load_logits(const T* row, int E, int lane, bool packed, float* x) {
  const int e0 = lane * EPL;
  constexpr int BYTES = EPL * static_cast<int>(sizeof(T));
  if (packed) {
    if (e0 >= E) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) x[i] = -INFINITY;
      return;
    }
    if constexpr (BYTES >= 16) {
      constexpr int VEC = Pack16<T>::kElems;
#pragma unroll
      for (int i = 0; i < EPL / VEC; ++i) Pack16<T>::unpack(ld_stream(reinterpret_cast<const uint4*>(row + e0) + i), x + i * VEC);
    } else {
      union { uint32_t w[BYTES >= 4 ? BYTES / 4 : 1]; T v[EPL]; } u;
      if constexpr (BYTES == 8) *reinterpret_cast<uint2*>(u.w) = __ldg(reinterpret_cast<const uint2*>(row + e0));
      else if constexpr (BYTES == 4) u.w[0] = __ldg(reinterpret_cast<const uint32_t*>(row + e0));
      else *reinterpret_cast<uint16_t*>(u.v) = __ldg(reinterpret_cast<const uint16_t*>(row + e0));
#pragma unroll
      for (int i = 0; i < EPL; ++i) x[i] = to_f32(u.v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = e0 + i < E ? to_f32(row[e0 + i]) : -INFINITY;
  }
}

// The k rounds of "maximum over the warp".  After it lane r < c holds the r-th choice (its expert in `chosen`, its
// logit in `chosen_x`), c = the number of choices returned: fewer than k when only -inf is left.
//
// Two to 8 experts a lane are sorted once, descending, by exchanges of neighbours, which keep equal ones in their order;
// a round then looks at the lanes' first keys only, and the lane that held the maximum moves its list up.  Which
// expert it was is worked out once, after the rounds: the owner's list of indices and how often it was chosen before.
// A round is a dozen instructions, most of them on the half-rate integer pipe.  Scanning all of a lane's keys in every
// round instead made the forward of 65536 x 128 fp32, k = 8, 55.6 us instead of 48.5 and of 32768 x 256 44.5 instead of
// 39.7; of one expert a lane (65536 x 32, k = 2) 26.4 instead of 29.5, and 16 a lane (16384 x 512) take 39.2 scanned, 44.2
// sorted.
template <int EPL>
__device__ __forceinline__ int route_choose(const float (&x)[EPL], int k, int lane, float& top, int& chosen, float& chosen_x) {
  uint32_t key[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) key[i] = order_key(x[i]);
  uint32_t mine = 0;
  int r = 0;
  if constexpr (EPL > 1 && EPL <= 8) {
    uint32_t id[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) id[i] = i;
#pragma unroll
    for (int n = EPL - 1; n > 0; --n)
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const bool swap = key[i + 1] > key[i];
        const uint32_t a = key[i], b = key[i + 1], c = id[i], d = id[i + 1];
        key[i] = swap ? b : a;
        key[i + 1] = swap ? a : b;
        id[i] = swap ? d : c;
        id[i + 1] = swap ? c : d;
      }
    uint32_t order = 0;
#pragma unroll
    for (int i = 0; i < EPL; ++i) order |= id[i] << (4 * i);
    int owner_of_mine = 64 + lane;  // lanes without a choice match nobody
    for (; r < k; ++r) {
      const uint32_t most = __reduce_max_sync(0xffffffffu, key[0]);
      if (r == 0) top = key_value(most);
      if (most <= kKeyNegInf) break;
      const int owner = __ffs(__ballot_sync(0xffffffffu, key[0] == most)) - 1;
      if (lane == r) {
        mine = most;
        owner_of_mine = owner;
      }
      if (lane == owner) {
#pragma unroll
        for (int i = 0; i + 1 < EPL; ++i) key[i] = key[i + 1];
        key[EPL - 1] = 0u;
      }
    }
    const int before = __popc(__match_any_sync(0xffffffffu, owner_of_mine) & ((1u << lane) - 1u));
    const uint32_t list = __shfl_sync(0xffffffffu, order, owner_of_mine & 31);
    if (lane < r) chosen = owner_of_mine * EPL + static_cast<int>((list >> (4 * before)) & 15u);
  } else {
    for (; r < k; ++r) {
      uint32_t best = key[0];
      int at = 0;
#pragma unroll
      for (int i = 1; i < EPL; ++i)
        if (key[i] > best) {
          best = key[i];
          at = i;
        }
      const uint32_t most = __reduce_max_sync(0xffffffffu, best);
      if (r == 0) top = key_value(most);
      if (most <= kKeyNegInf) break;
      const int owner = __ffs(__ballot_sync(0xffffffffu, best == most)) - 1;
      const int e = EPL == 1 ? owner : __shfl_sync(0xffffffffu, lane * EPL + at, owner);
      if (lane == r) {
        chosen = e;
        mine = most;
      }
      if (lane == owner) {
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (i == at) key[i] = 0u;
      }
    }
  }
  if (lane < r) chosen_x = key_value(mine);
  return r;
}

// A word of the same variable in CTA c of the cluster.
template <typename V>
__device__ __forceinline__ V ld_cluster(const V* own, int c) {
  static_assert(sizeof(V) == 4, "32-bit words");
  uint32_t v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(cluster_map(smem_addr(own), c)) : "memory");
  return reinterpret_cast<const V&>(v);
}

__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) {
  asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory");
}

// The counts of experts e0 .. e1 - 1, from `count(e)`, and in thread 0 the sum over them of count(e) * sum(e), which is the sum
// of p over the tokens.
template <int THREADS, typename Sum, typename Count>
__device__ __forceinline__ double route_share(const RouteParams& p, int e0, int e1, Sum sum, Count count) {
  __shared__ double red[THREADS / 32];
  double share = 0.;
  for (int e = e0 + threadIdx.x; e < e1; e += THREADS) {
    const int c = count(e);
    p.counts[e] = c;
    if (p.kept != nullptr) p.kept[e] = c;
    share += static_cast<double>(sum(e)) * c;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) share += __shfl_xor_sync(0xffffffffu, share, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = share;
  __syncthreads();
  double total = 0.;
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) total += red[w];
  }
  return total;
}
// One thread: the number of live tokens and the loss.
__device__ __forceinline__ void route_loss(const RouteParams& p, int n, double share) {
  p.counts[p.E] = n;
  if (p.kept != nullptr) p.kept[p.E] = n;
  *p.loss = n > 0 ? static_cast<float>(share * p.E / (static_cast<double>(n) * n * p.k)) : 0.f;
}

template <typename T, int EPL>
__global__ void __launch_bounds__(kRouteThreads, EPL <= 8 ? 2 : 1) route_fwd_kernel(const RouteParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];  // float sums[warps][columns]; int counts[columns + 1]
  float* sums = reinterpret_cast<float*>(dyn);
  int* counts = reinterpret_cast<int*>(sums + (size_t)kRouteWarps * p.columns);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e <= p.columns; e += kRouteThreads) counts[e] = 0;
  __syncthreads();
  grid_dependency_sync();
  trigger_dependents();

  const T* logits = static_cast<const T*>(p.logits);
  const bool packed = p.E % EPL == 0 && (reinterpret_cast<uintptr_t>(logits) & 15u) == 0 && (p.stride * sizeof(T)) % 16 == 0;
  int group = 1;  // lanes over which the gates are summed: a power of two, at least k
  while (group < p.k) group *= 2;
  float acc[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) acc[i] = 0.f;
  int live_tokens = 0;
  const int64_t step = (int64_t)gridDim.x * kRouteWarps;
  int64_t tok = (int64_t)blockIdx.x * kRouteWarps + warp;
  float nx[EPL];
  uint8_t next_on = 1;
  auto fetch = [&](int64_t at) {
    load_logits<T, EPL>(logits + at * p.stride, p.E, lane, packed, nx);
    if (p.mask != nullptr) next_on = p.mask[at];
  };
  if (tok < p.T) fetch(tok);
  for (; tok < p.T; tok += step) {
    float x[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = nx[i];
    const bool masked = next_on == 0;
    if (tok + step < p.T) fetch(tok + step);

    float top = 0.f, chosen_x = 0.f;
    int chosen = -1;
    const bool live = route_choose<EPL>(x, p.k, lane, top, chosen, chosen_x) > 0 && !masked;

    float s = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      x[i] = exp_below(x[i] - top);
      s += x[i];
    }
    s = warp_sum(s);
    float gate = chosen >= 0 ? exp_below(chosen_x - top) : 0.f;
    float total = s;
    if (p.normalize) {
      total = gate;
      for (int o = 1; o < group; o <<= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    if (lane < p.k) {
      const bool choice = live && chosen >= 0;
      p.gates[tok * p.k + lane] = choice ? gate * rcp_fast(total) : 0.f;
      p.experts[tok * p.k + lane] = choice ? chosen : -1;
      if (choice) atomicAdd(&counts[chosen], 1);
    }
    if (p.lse != nullptr && lane == 0) p.lse[tok] = live ? top + logf(s) : -INFINITY;
    if (live) {
      ++live_tokens;
      const float inv = rcp_fast(s);  // s >= 1
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[i] = fmaf(x[i], inv, acc[i]);
    }
  }
  if (lane == 0) atomicAdd(&counts[p.columns], live_tokens);
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (lane * EPL + i < p.columns) sums[(size_t)warp * p.columns + lane * EPL + i] = acc[i];
  __syncthreads();
  auto cta_sum = [&](int e) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kRouteWarps; ++w) s += sums[(size_t)w * p.columns + e];
    return s;
  };
  if (p.cluster > 0) {  // the grid is one cluster: its first CTA adds up the others' rows
    for (int e = threadIdx.x; e < p.E; e += kRouteThreads) sums[e] = cta_sum(e);  // column e is this thread's alone
    if (p.cluster > 1) cluster_sync_all();
    else __syncthreads();
    if (blockIdx.x == 0) {
      auto over_ctas = [&](auto* at, auto zero) {
        for (int c = 0; c < p.cluster; ++c) zero += ld_cluster(at, c);
        return zero;
      };
      const double share = route_share<kRouteThreads>(p, 0, p.E, [&](int e) { return over_ctas(sums + e, 0.f); },
                                                      [&](int e) { return over_ctas(counts + e, 0); });
      if (threadIdx.x == 0) route_loss(p, over_ctas(counts + p.columns, 0), share);
    }
    if (p.cluster > 1) cluster_sync_all();  // the others' shared memory has been read
    return;
  }
  for (int e = threadIdx.x; e < p.columns; e += kRouteThreads) {
    p.part_p[(size_t)blockIdx.x * p.columns + e] = e < p.E ? cta_sum(e) : 0.f;
    p.part_n[(size_t)blockIdx.x * p.columns + e] = counts[e];
  }
  if (threadIdx.x == 0) p.part_live[blockIdx.x] = counts[p.columns];
}

// Adds the CTAs' partial rows: a cluster, each of whose CTAs takes its share of the columns, 16 bytes a thread and as many rows
// side by side as there are threads, then a warp a column; every column in one fixed order.  It is a chain of latencies: one
// CTA for all columns took 6 us for 128 experts and 15 us for 1024, of 45 and 71 us in all.
constexpr int kRouteFinishThreads = 1024;
__global__ void __launch_bounds__(kRouteFinishThreads) route_finish_kernel(const RouteParams p) {
  constexpr int MOST = kRouteMaxExperts / kRouteMaxCluster;  // columns of a CTA
  constexpr int ROWS = 128;                                  // side by side, at most
  constexpr int SLOTS = kRouteFinishThreads + ROWS;
  __shared__ float4 sum_s[SLOTS];
  __shared__ int4 count_s[SLOTS];
  __shared__ float column_sum[MOST];
  __shared__ int column_count[MOST];
  __shared__ double shares[kRouteMaxCluster];  // of the first CTA: every CTA's part of the loss
  const int tid = threadIdx.x, lane = tid & 31, rank = static_cast<int>(cluster_cta_rank());
  const int quads = (p.columns / 4 + kRouteMaxCluster - 1) / kRouteMaxCluster;  // of a CTA, 16 bytes each
  const int groups = min(min(ROWS, kRouteFinishThreads / quads), p.parts);
  const int pitch = quads | 1;  // odd: a warp that reads down a column meets a bank four times, not 32
  const int q = tid % quads, g = tid / quads, column = 4 * (rank * quads + q);
  grid_dependency_sync();
  trigger_dependents();
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  int4 n = make_int4(0, 0, 0, 0);
  if (g < groups && column < p.columns) {
#pragma unroll 2
    for (int r = g; r < p.parts; r += groups) {
      const float4 a = *reinterpret_cast<const float4*>(p.part_p + (size_t)r * p.columns + column);
      const int4 b = *reinterpret_cast<const int4*>(p.part_n + (size_t)r * p.columns + column);
      s.x += a.x; s.y += a.y; s.z += a.z; s.w += a.w;
      n.x += b.x; n.y += b.y; n.z += b.z; n.w += b.w;
    }
  }
  if (g < groups) {
    sum_s[g * pitch + q] = s;
    count_s[g * pitch + q] = n;
  }
  int live = 0;
  if (rank == 0 && tid < 32) {
    for (int r = tid; r < p.parts; r += 32) live += p.part_live[r];
    live = __reduce_add_sync(0xffffffffu, live);
  }
  cluster_sync_all();
  for (int c = tid >> 5; c < 4 * quads; c += kRouteFinishThreads / 32) {
    float cs = 0.f;
    int cn = 0;
    for (int r = lane; r < groups; r += 32) {
      cs += reinterpret_cast<const float*>(sum_s)[r * pitch * 4 + c];
      cn += reinterpret_cast<const int*>(count_s)[r * pitch * 4 + c];
    }
    cs = warp_sum(cs);
    cn = __reduce_add_sync(0xffffffffu, cn);
    if (lane == 0) {
      column_sum[c] = cs;
      column_count[c] = cn;
    }
  }
  __syncthreads();
  const int first = min(rank * quads * 4, p.E), last = min(first + quads * 4, p.E);
  const double share = route_share<kRouteFinishThreads>(p, first, last, [&](int e) { return column_sum[e - first]; },
                                                        [&](int e) { return column_count[e - first]; });
  if (tid == 0) st_cluster_f64(cluster_map(smem_addr(&shares[rank]), 0), share);
  cluster_sync_all();
  if (rank == 0 && tid == 0) {
    double total = 0.;
#pragma unroll
    for (int c = 0; c < kRouteMaxCluster; ++c) total += shares[c];
    route_loss(p, live, total);
  }
}

// Backward: p comes from the logits and the saved log-sum, the chosen experts' part is put in its place
// through a row of shared memory per warp.  The log-sum, one fp32 number, has lost of the sum what lies below half an ulp of a
// large maximum (logits around 1e4: 3e-4 of p; whole rows at the type's lowest value: all of it), so it only shifts the
// exponentials, and p are their shares of their own sum.
template <typename T, int EPL>
__global__ void __launch_bounds__(kRouteBwdThreads) route_bwd_kernel(const RouteParams p) {
  __shared__ __align__(16) float place[kRouteBwdWarps][32 * EPL];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* mine = place[warp];
#pragma unroll
  for (int i = 0; i < EPL; ++i) mine[lane * EPL + i] = 0.f;
  __syncwarp();
  grid_dependency_sync();
  trigger_dependents();

  const T* logits = static_cast<const T*>(p.logits);
  const bool packed = p.E % EPL == 0 && (reinterpret_cast<uintptr_t>(logits) & 15u) == 0 && (p.stride * sizeof(T)) % 16 == 0;
  float c[EPL];
  {
    const float n = static_cast<float>(p.counts[p.E]);
    const float f = p.dloss != nullptr && n > 0.f ? *p.dloss * static_cast<float>(p.E) / (n * n * static_cast<float>(p.k)) : 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) c[i] = lane * EPL + i < p.E ? f * static_cast<float>(p.counts[lane * EPL + i]) : 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * kRouteBwdWarps;
  int64_t tok = (int64_t)blockIdx.x * kRouteBwdWarps + warp;
  float nx[EPL];
  if (tok < p.T) load_logits<T, EPL>(logits + tok * p.stride, p.E, lane, packed, nx);
  for (; tok < p.T; tok += step) {
    float x[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = nx[i];
    if (tok + step < p.T) load_logits<T, EPL>(logits + (tok + step) * p.stride, p.E, lane, packed, nx);
    const float lse = p.lse[tok];
    const bool live = lse != -INFINITY;
    int e = -1;
    float dg = 0.f, gate = 0.f;
    if (live && lane < p.k) {
      e = p.experts[tok * p.k + lane];
      gate = p.gates[tok * p.k + lane];
      if (p.dgates != nullptr) dg = p.dgates[tok * p.dgates_stride + lane];
    }
    float s = 0.f, total = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      x[i] = live ? exp_below(x[i] - lse) : 0.f;
      total += x[i];
      s = fmaf(x[i], c[i], s);
    }
    const bool any = static_cast<unsigned>(e) < static_cast<unsigned>(p.E);  // -1: none; and no other place is written to
    float g = any ? gate * dg : 0.f;
    const float inv = rcp_fast(warp_sum(total)), sum_g = warp_sum(g);
    s = warp_sum(s) * inv;
    if (p.normalize) g -= gate * sum_g;
    else s += sum_g;
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] *= inv;
    if (any) mine[e] = g;
    __syncwarp();
    T* out = static_cast<T*>(p.dlogits) + tok * p.E;
    const int e0 = lane * EPL;
    float d[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] = mine[e0 + i];
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] = live ? fmaf(x[i], c[i] - s, d[i]) : 0.f;  // c may be infinite
    __syncwarp();
    if (any) mine[e] = 0.f;
    if (packed && EPL * sizeof(T) >= 16 && p.E * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.dlogits) & 15u) == 0) {
      if constexpr (EPL * sizeof(T) >= 16) {
        constexpr int VEC = Pack16<T>::kElems;
        if (e0 < p.E) {
#pragma unroll
          for (int i = 0; i < EPL / VEC; ++i) st_stream(reinterpret_cast<uint4*>(out + e0) + i, Pack16<T>::pack(d + i * VEC));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i)
        if (e0 + i < p.E) out[e0 + i] = from_f32<T>(d[i]);
    }
    __syncwarp();
  }
}

}  // namespace b200norm
