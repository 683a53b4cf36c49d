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
// lanes with one maximum also has the lowest index.  Reading the logits is 6 us at 65536 x 128 fp32; the k
// rounds of "maximum over the warp" are what the instructions go to.
#pragma once

#include "norm_common.cuh"

namespace b200norm {

constexpr int kRouteThreads = 512;
constexpr int kRouteWarps = kRouteThreads / 32;
constexpr int kRouteBwdThreads = 256;
constexpr int kRouteBwdWarps = kRouteBwdThreads / 32;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 32;

struct RouteParams {
  const void* logits;
  int64_t stride;       // elements
  const uint8_t* mask;  // (T,) or null
  float* gates;         // (T, k)
  int* experts;         // (T, k)
  float* lse;           // (T,) log of the softmax's denominator; -inf marks a token that is not live
  int* counts;          // (E + 1): per expert, then the number of live tokens
  float* loss;
  float* part_p;  // (gridDim.x, E) partial sums of p
  int* part_n;    // (gridDim.x, E + 1) partial counts
  // backward
  const float* dgates;  // (T, k) or null
  int64_t dgates_stride;
  const float* dloss;  // scalar or null
  void* dlogits;       // (T, E) contiguous
  int64_t T;
  int E, k, normalize, parts;
};

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

// Sums the partial rows of all CTAs and forms counts, the number of live tokens and the loss.  Runs in one CTA of
// `threads` threads; every column is added in CTA order.
__device__ __forceinline__ void route_finish(const RouteParams& p, int parts, const float* part_p, const int* part_n,
                                             double* red, int threads) {
  const int tid = threadIdx.x;
  __shared__ int live_s;
  if (tid < 32) {
    int n = 0;
    for (int g = tid; g < parts; g += 32) n += part_n[(size_t)g * (p.E + 1) + p.E];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if (tid == 0) live_s = n;
  }
  double share = 0.;
  for (int e = tid; e < p.E; e += threads) {
    float s = 0.f;
    int n = 0;
    for (int g = 0; g < parts; ++g) {
      s += part_p[(size_t)g * p.E + e];
      n += part_n[(size_t)g * (p.E + 1) + e];
    }
    p.counts[e] = n;
    share += static_cast<double>(s) * n;
  }
  red[tid] = share;
  __syncthreads();
  if (tid >= 32) return;
  double total = 0.;
  for (int i = tid; i < threads; i += 32) total += red[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (tid == 0) {
    const int n = live_s;
    p.counts[p.E] = n;
    *p.loss = n > 0 ? static_cast<float>(total * p.E / (static_cast<double>(n) * n * p.k)) : 0.f;
  }
}

template <typename T, int EPL>
__global__ void __launch_bounds__(kRouteThreads) route_fwd_kernel(const RouteParams p) {
  extern __shared__ __align__(16) unsigned char dyn[];  // float sums[warps][E]; the counts of the CTA: int [E + 1]
  float* sums = reinterpret_cast<float*>(dyn);
  int* counts = reinterpret_cast<int*>(sums + (size_t)kRouteWarps * p.E);
  __shared__ double red[kRouteThreads];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e <= p.E; e += kRouteThreads) counts[e] = 0;
  __syncthreads();
  grid_dependency_sync();
  trigger_dependents();

  const T* logits = static_cast<const T*>(p.logits);
  const bool packed = p.E % EPL == 0 && (reinterpret_cast<uintptr_t>(logits) & 15u) == 0 && (p.stride * sizeof(T)) % 16 == 0;
  float acc[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) acc[i] = 0.f;
  int live_tokens = 0;
  const int64_t step = (int64_t)gridDim.x * kRouteWarps;
  int64_t tok = (int64_t)blockIdx.x * kRouteWarps + warp;
  float nx[EPL];
  if (tok < p.T) load_logits<T, EPL>(logits + tok * p.stride, p.E, lane, packed, nx);
  for (; tok < p.T; tok += step) {
    float x[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) x[i] = nx[i];
    if (tok + step < p.T) load_logits<T, EPL>(logits + (tok + step) * p.stride, p.E, lane, packed, nx);
    const bool masked = p.mask != nullptr && p.mask[tok] == 0;

    uint32_t key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) key[i] = order_key(x[i]);
    float top = 0.f;
    int chosen = -1;
    float chosen_x = 0.f;
    bool live = !masked;
    for (int r = 0; r < p.k; ++r) {
      uint32_t best = key[0];
      int at = 0;
#pragma unroll
      for (int i = 1; i < EPL; ++i)
        if (key[i] > best) {
          best = key[i];
          at = i;
        }
      const uint32_t most = __reduce_max_sync(0xffffffffu, best);
      if (r == 0) {
        top = key_value(most);
        live = live && most > kKeyNegInf;
      }
      if (most <= kKeyNegInf) break;  // only -inf is left
      const int owner = __ffs(__ballot_sync(0xffffffffu, best == most)) - 1;
      const int e = __shfl_sync(0xffffffffu, lane * EPL + at, owner);
      if (lane == r) {
        chosen = e;
        chosen_x = key_value(most);
      }
      if (lane == owner) {
#pragma unroll
        for (int i = 0; i < EPL; ++i)
          if (i == at) key[i] = 0u;
      }
    }

    float s = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      x[i] = expf(x[i] - top);
      s += x[i];
    }
    s = warp_sum(s);
    float gate = chosen >= 0 ? expf(chosen_x - top) : 0.f;
    const float total = p.normalize ? warp_sum(gate) : s;
    gate = live && chosen >= 0 ? gate / total : 0.f;
    if (lane < p.k) {
      p.gates[tok * p.k + lane] = gate;
      p.experts[tok * p.k + lane] = live ? chosen : -1;
      if (live && chosen >= 0) atomicAdd(&counts[chosen], 1);
    }
    if (p.lse != nullptr && lane == 0) p.lse[tok] = live ? top + logf(s) : -INFINITY;
    if (live) {
      ++live_tokens;
      const float inv = 1.f / s;
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[i] = fmaf(x[i], inv, acc[i]);
    }
  }
  if (lane == 0) atomicAdd(&counts[p.E], live_tokens);
#pragma unroll
  for (int i = 0; i < EPL; ++i)
    if (lane * EPL + i < p.E) sums[(size_t)warp * p.E + lane * EPL + i] = acc[i];
  __syncthreads();
  float* out_p = p.part_p + (size_t)blockIdx.x * p.E;
  int* out_n = p.part_n + (size_t)blockIdx.x * (p.E + 1);
  const bool alone = gridDim.x == 1;  // a single CTA finishes by itself: no second launch
  for (int e = threadIdx.x; e < p.E; e += kRouteThreads) {
    float s = 0.f;
    for (int w = 0; w < kRouteWarps; ++w) s += sums[(size_t)w * p.E + e];
    if (alone) sums[e] = s;  // row 0 of a column is read and written by one thread only
    else out_p[e] = s;
  }
  if (alone) {
    __syncthreads();
    route_finish(p, 1, sums, counts, red, kRouteThreads);
  } else {
    for (int e = threadIdx.x; e <= p.E; e += kRouteThreads) out_n[e] = counts[e];
  }
}

__global__ void __launch_bounds__(kRouteThreads) route_finish_kernel(const RouteParams p) {
  __shared__ double red[kRouteThreads];
  grid_dependency_sync();
  trigger_dependents();
  route_finish(p, p.parts, p.part_p, p.part_n, red, kRouteThreads);
}

// Backward: p comes from the logits and the saved log-sum, the chosen experts' part is put in its place
// through a row of shared memory per warp.
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
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      x[i] = live ? expf(x[i] - lse) : 0.f;
      s = fmaf(x[i], c[i], s);
    }
    const bool any = e >= 0;
    float g = any ? gate * dg : 0.f;
    if (p.normalize) {
      g -= gate * warp_sum(g);
      s = warp_sum(s);
    } else {
      s = warp_sum(s + g);
    }
    if (any) mine[e] = g;
    __syncwarp();
    T* out = static_cast<T*>(p.dlogits) + tok * p.E;
    const int e0 = lane * EPL;
    float d[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) d[i] = x[i] * (c[i] - s) + mine[e0 + i];
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
