// Entry points of the expert choice (route.cuh): argument checks, launch planning, launches.
#include <algorithm>

#include "host.h"
#include "route.cuh"

namespace b200norm {
namespace {

// Up to this many tokens, two a warp, the grid is one cluster, which finishes in one launch and without a workspace: 128 x 64
// takes 5 us, with two launches 7; 256 x 64 6.6 and 7.1.
constexpr int64_t kRouteClusterTokens = 2 * kRouteMaxCluster * kRouteWarps;

const void* route_fn(int dtype, int E, bool bwd) {
#define B200NORM_ROUTE(EPL)                                                                                    \
  if (E <= 32 * EPL) {                                                                                         \
    if (dtype == B200NORM_F32)                                                                                 \
      return bwd ? reinterpret_cast<const void*>(&route_bwd_kernel<float, EPL>)                                \
                 : reinterpret_cast<const void*>(&route_fwd_kernel<float, EPL>);                               \
    if (dtype == B200NORM_F16)                                                                                 \
      return bwd ? reinterpret_cast<const void*>(&route_bwd_kernel<__half, EPL>)                               \
                 : reinterpret_cast<const void*>(&route_fwd_kernel<__half, EPL>);                              \
    return bwd ? reinterpret_cast<const void*>(&route_bwd_kernel<__nv_bfloat16, EPL>)                          \
               : reinterpret_cast<const void*>(&route_fwd_kernel<__nv_bfloat16, EPL>);                         \
  }
  B200NORM_ROUTE(1)
  B200NORM_ROUTE(2)
  B200NORM_ROUTE(4)
  B200NORM_ROUTE(8)
  B200NORM_ROUTE(16)
  B200NORM_ROUTE(32)
#undef B200NORM_ROUTE
  return nullptr;
}

int check(int64_t T, int E, int k, int dtype) {
  if (dtype != B200NORM_F32 && dtype != B200NORM_F16 && dtype != B200NORM_BF16)
    return fail(B200NORM_ERR_ARG, "router logits are fp32, fp16 or bf16 (dtype code %d)", dtype);
  if (T < 0 || E < 1 || E > kRouteMaxExperts) return fail(B200NORM_ERR_ARG, "1 to %d experts, got %d", kRouteMaxExperts, E);
  if (k < 1 || k > E || k > kRouteMaxK) return fail(B200NORM_ERR_ARG, "top_k is 1 to min(%d, experts), got %d of %d", kRouteMaxK, k, E);
  if (T * k > INT32_MAX) return fail(B200NORM_ERR_ARG, "%lld tokens x %d choices do not fit 32-bit counts", (long long)T, k);
  return B200NORM_OK;
}

int columns_of(int E) { return (E + 3) / 4 * 4; }

size_t fwd_smem(int E) { return (static_cast<size_t>(kRouteWarps + 1) * columns_of(E) + 1) * 4; }

// Partial rows of the sums and of the counts, and the live tokens, of every CTA; 1 for a cluster.
size_t workspace_need(int grid, int cluster, int E) {
  return cluster > 0 ? 1 : static_cast<size_t>(grid) * (2 * columns_of(E) + 1) * 4;
}

int fwd_grid(DeviceState& dev, const void* fn, int64_t T, int E, int* grid, int* cluster) {
  int occ;  // also raises the kernel's shared-memory allowance
  if (int rc = occupancy(dev, fn, kRouteThreads, fwd_smem(E), &occ)) return rc;
  const int64_t want = std::max<int64_t>(1, (T + kRouteWarps - 1) / kRouteWarps);
  *cluster = 0;
  if (T <= kRouteClusterTokens) {
    *cluster = 1;
    while (*cluster < std::min<int64_t>(want, kRouteMaxCluster)) *cluster *= 2;
  }
  *grid = *cluster > 0 ? *cluster : static_cast<int>(std::min<int64_t>(want, (int64_t)dev.sm_count * occ));
  return B200NORM_OK;
}

}  // namespace
}  // namespace b200norm

using namespace b200norm;

extern "C" {

size_t b200norm_route_workspace_bytes(int64_t T, int E, int k, int dtype) {
  if (check(T, E, k, dtype)) return 0;
  DeviceState* dev = nullptr;
  if (device_caches(&dev)) return 0;
  int grid, cluster;
  if (fwd_grid(*dev, route_fn(dtype, E, false), T, E, &grid, &cluster)) return 0;
  return workspace_need(grid, cluster, E);
}

int b200norm_route_fwd(const void* logits, int64_t row_stride, const uint8_t* mask, float* gates, int* experts, float* lse,
                       int* counts, float* loss, void* workspace, size_t workspace_bytes, int64_t T, int E, int k,
                       int normalize, int dtype, void* stream) {
  return b200norm_route_fwd_kept(logits, row_stride, mask, gates, experts, lse, counts, nullptr, loss, workspace, workspace_bytes,
                                 T, E, k, normalize, dtype, stream);
}

int b200norm_route_fwd_kept(const void* logits, int64_t row_stride, const uint8_t* mask, float* gates, int* experts, float* lse,
                            int* counts, int* kept, float* loss, void* workspace, size_t workspace_bytes, int64_t T, int E,
                            int k, int normalize, int dtype, void* stream_v) {
  if (int rc = check(T, E, k, dtype)) return rc;
  if (!counts || !loss || (T > 0 && (!logits || !gates || !experts))) return fail(B200NORM_ERR_ARG, "null buffer");
  if (row_stride < E) return fail(B200NORM_ERR_ARG, "row stride smaller than the number of experts");
  if (!on_element(logits, dtype_size(dtype)) || !on_element(gates, 4) || !on_element(experts, 4) || !on_element(lse, 4) ||
      !on_element(counts, 4) || !on_element(kept, 4) || !on_element(loss, 4))
    return fail_off_element();
  DeviceState* dev = nullptr;
  if (int rc = device_caches(&dev)) return rc;
  const void* fn = route_fn(dtype, E, false);
  int grid, cluster;
  if (int rc = fwd_grid(*dev, fn, T, E, &grid, &cluster)) return rc;
  const size_t need = workspace_need(grid, cluster, E);
  if (cluster == 0 && (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 15u)))
    return fail(B200NORM_ERR_ARG, "workspace needs %zu bytes, 16-byte aligned (got %zu)", need, workspace_bytes);
  RouteParams p = {};
  p.logits = logits; p.stride = row_stride; p.mask = mask; p.gates = gates; p.experts = experts; p.lse = lse;
  p.counts = counts; p.kept = kept; p.loss = loss;
  p.part_p = static_cast<float*>(workspace);
  p.columns = columns_of(E);
  p.part_n = reinterpret_cast<int*>(p.part_p + static_cast<size_t>(grid) * p.columns);
  p.part_live = p.part_n + static_cast<size_t>(grid) * p.columns;
  p.T = T; p.E = E; p.k = k; p.normalize = normalize != 0; p.parts = grid;
  p.cluster = cluster;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (int rc = launch(fn, dim3(grid), dim3(kRouteThreads), fwd_smem(E), &p, stream, true, std::max(cluster, 1))) return rc;
  if (cluster > 0) return B200NORM_OK;
  return launch(reinterpret_cast<const void*>(&route_finish_kernel), dim3(kRouteMaxCluster), dim3(kRouteFinishThreads),
                0, &p, stream, true, kRouteMaxCluster);
}

int b200norm_route_bwd(const void* logits, int64_t row_stride, const float* gates, const int* experts, const float* lse,
                       const int* counts, const float* dgates, int64_t dgates_row_stride, const float* dloss, void* dlogits,
                       int64_t T, int E, int k, int normalize, int dtype, void* stream) {
  if (int rc = check(T, E, k, dtype)) return rc;
  if (T == 0) return B200NORM_OK;
  if (!logits || !gates || !experts || !lse || !counts || !dlogits) return fail(B200NORM_ERR_ARG, "null buffer");
  if (row_stride < E || (dgates && dgates_row_stride < k)) return fail(B200NORM_ERR_ARG, "row stride smaller than the row");
  if (!on_element(logits, dtype_size(dtype)) || !on_element(gates, 4) || !on_element(experts, 4) || !on_element(lse, 4) ||
      !on_element(counts, 4) || !on_element(dgates, 4) || !on_element(dloss, 4) || !on_element(dlogits, dtype_size(dtype)))
    return fail_off_element();
  DeviceState* dev = nullptr;
  if (int rc = device_caches(&dev)) return rc;
  const void* fn = route_fn(dtype, E, true);
  int occ;
  if (int rc = occupancy(*dev, fn, kRouteBwdThreads, 0, &occ)) return rc;
  RouteParams p = {};
  p.logits = logits; p.stride = row_stride; p.gates = const_cast<float*>(gates); p.experts = const_cast<int*>(experts);
  p.lse = const_cast<float*>(lse); p.counts = const_cast<int*>(counts);
  p.dgates = dgates; p.dgates_stride = dgates_row_stride; p.dloss = dloss; p.dlogits = dlogits;
  p.T = T; p.E = E; p.k = k; p.normalize = normalize != 0;
  const int64_t want = (T + kRouteBwdWarps - 1) / kRouteBwdWarps;
  const int grid = static_cast<int>(std::min<int64_t>(want, (int64_t)dev->sm_count * occ));
  return launch(fn, dim3(grid), dim3(kRouteBwdThreads), 0, &p, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
