// Entry point of the token choice (sample.cuh): argument checks, launch planning, launch.
#include <algorithm>

#include "host.h"
#include "sample.cuh"

namespace b200norm {
namespace {

template <typename T>
const void* sample_fn(int cluster) {
  switch (cluster) {
    case 1: return reinterpret_cast<const void*>(&sample_kernel<T, 1>);
    case 2: return reinterpret_cast<const void*>(&sample_kernel<T, 2>);
    case 4: return reinterpret_cast<const void*>(&sample_kernel<T, 4>);
    default: return reinterpret_cast<const void*>(&sample_kernel<T, 8>);
  }
}

}  // namespace
}  // namespace b200norm

using namespace b200norm;

extern "C" int b200norm_sample(const void* logits, int64_t row_stride, const float* uniform, const float* temperature_v,
                               float temperature, const int* top_k_v, int top_k, const float* top_p_v, float top_p,
                               const float* min_p_v, float min_p, int64_t* tokens, int64_t M, int64_t V, int dtype,
                               void* stream) {
  if (dtype != B200NORM_F32 && dtype != B200NORM_F16 && dtype != B200NORM_BF16)
    return fail(B200NORM_ERR_ARG, "logits are fp32, fp16 or bf16 (dtype code %d)", dtype);
  if (M < 0 || V < 1) return fail(B200NORM_ERR_ARG, "bad shape M=%lld V=%lld", (long long)M, (long long)V);
  if (V > kSampleMaxVocab)
    return fail(B200NORM_ERR_UNSUPPORTED, "a vocabulary of up to %d tokens, got %lld", kSampleMaxVocab, (long long)V);
  if (M == 0) return B200NORM_OK;
  if (M > INT32_MAX / kSampleMaxCluster) return fail(B200NORM_ERR_ARG, "too many rows: %lld", (long long)M);
  if (!logits || !uniform || !tokens) return fail(B200NORM_ERR_ARG, "null logits / uniform / tokens");
  if (row_stride < V) return fail(B200NORM_ERR_ARG, "row stride smaller than the vocabulary");
  const int es = static_cast<int>(dtype_size(dtype)), vec = 16 / es;
  if (!on_element(logits, es) || !on_element(uniform, 4) || !on_element(temperature_v, 4) || !on_element(top_k_v, 4) ||
      !on_element(top_p_v, 4) || !on_element(min_p_v, 4) || !on_element(tokens, 8))
    return fail_off_element();
  DeviceState* dev = nullptr;
  if (int rc = device_caches(&dev)) return rc;
  // CTAs per row: as few as have parts of up to 112 KB.  Parts of up to 98 KB let two CTAs share an SM (228 KB, 16 of it
  // static or reserved per CTA), so that one's barriers hide behind the other's arithmetic, but each CTA has its fixed
  // costs: top-p 0.9 of 512 x 65536 bf16 takes 238 us with 1 CTA a row, 189 with 2, 266 with 4; 512 x 50257 fp32 157 with 2
  // parts of 98 KB and more, 214 with 4; 512 x 50257 bf16 144 with 1, 160 with 2.
  // With few rows as many as there are SMs, while a part keeps 4096 tokens: one row of 32768 bf16 takes 34 us with 1 CTA,
  // 25, 19 and 17 with 2, 4 and 8; one of 8192 is as quick with 1.
  constexpr int64_t kPart = 112 * 1024;
  constexpr int64_t kSplit = 16384;
  int cluster = 1;
  while (cluster < kSampleMaxCluster && V * es > cluster * kPart) cluster *= 2;
  while (cluster < kSampleMaxCluster && M * cluster * 2 <= dev->sm_count && V >= std::max<int64_t>(kSplit, cluster * 2 * 4096))
    cluster *= 2;
  SampleParams p = {};
  p.logits = logits; p.stride = row_stride; p.uniform = uniform;
  p.temperature_v = temperature_v; p.temperature = temperature;
  p.top_k_v = top_k_v; p.top_k = top_k;
  p.top_p_v = top_p_v; p.top_p = top_p;
  p.min_p_v = min_p_v; p.min_p = min_p;
  p.tokens = tokens; p.M = M; p.V = static_cast<int>(V);
  // whole packets, of a row that may start and end inside one
  const int64_t packets = (V + 2 * vec - 2) / vec;
  p.chunk = static_cast<int>((packets + cluster - 1) / cluster * vec);
  const size_t smem = static_cast<size_t>(p.chunk) * es;
  const void* fn = dtype == B200NORM_F32 ? sample_fn<float>(cluster)
                   : dtype == B200NORM_F16 ? sample_fn<__half>(cluster) : sample_fn<__nv_bfloat16>(cluster);
  int occ;  // also raises the kernel's shared-memory allowance
  if (int rc = occupancy(*dev, fn, kSampleThreads, smem, &occ, cluster)) return rc;
  return launch(fn, dim3(static_cast<unsigned>(M * cluster)), dim3(kSampleThreads), smem, &p,
                static_cast<cudaStream_t>(stream), true, cluster);
}
