// Entry points of the residual + RMSNorm operators: argument checks, launch planning, launches.
#include <algorithm>
#include <numeric>

#include "addnorm.cuh"
#include "host.h"

namespace b200norm {
namespace {

// How the rows of a call's buffers lie: on packet boundaries, at one common offset from them, or neither.
enum Layout { kAligned = 0, kOffset = 1, kAny = 2 };
enum Which { kFwd, kFp8, kBwd };

struct Buffer {
  const void* p;
  int64_t stride;
  int size;  // bytes per element
};

const AddNormTable* table_for(int io, int res) {
  if (io == B200NORM_F32 && res == B200NORM_F32) return addnorm_table_f32();
  if (io == B200NORM_F16 && res == B200NORM_F16) return addnorm_table_f16();
  if (io == B200NORM_BF16 && res == B200NORM_BF16) return addnorm_table_bf16();
  if (io == B200NORM_F16 && res == B200NORM_F32) return addnorm_table_f16_f32();
  if (io == B200NORM_BF16 && res == B200NORM_F32) return addnorm_table_bf16_f32();
  return nullptr;
}

int check(int64_t M, int64_t N, int io, int res, int w_dtype) {
  if (table_for(io, res) == nullptr)
    return fail(B200NORM_ERR_ARG, "residual + RMSNorm runs on fp32, fp16 and bf16 rows with a residual of the same type or "
                "fp32 (io code %d, residual code %d)", io, res);
  if (w_dtype < B200NORM_F32 || w_dtype > B200NORM_F64) return fail(B200NORM_ERR_ARG, "unknown weight dtype code %d", w_dtype);
  if (M < 0 || N < 1) return fail(B200NORM_ERR_ARG, "bad shape M=%lld N=%lld", (long long)M, (long long)N);
  if (N * table_for(io, res)->size_t_ > kMaxRowBytes)
    return fail(B200NORM_ERR_UNSUPPORTED, "This layer norm doesn't support feature dim >= 64KB.");
  return B200NORM_OK;
}

// The common layout of the buffers (null ones are skipped) in packets of `vec` elements; *period: after how
// many rows the offset repeats.
Layout layout_of(const Buffer* b, int n, int64_t N, int vec, const void* w, int* period) {
  *period = 1;
  int64_t phase = -1, stride = -1;
  for (int i = 0; i < n; ++i) {
    if (b[i].p == nullptr) continue;
    const uintptr_t a = reinterpret_cast<uintptr_t>(b[i].p);
    const int64_t ph = static_cast<int64_t>((a / b[i].size) % vec), st = b[i].stride % vec;
    if (phase >= 0 && (ph != phase || st != stride)) return kAny;
    phase = ph;
    stride = st;
  }
  if (phase == 0 && stride == 0 && N % vec == 0 && (reinterpret_cast<uintptr_t>(w) & 15u) == 0) return kAligned;
  if (stride > 0) *period = static_cast<int>(vec / std::gcd<int64_t>(vec, stride));
  return kOffset;
}

struct Plan {
  const void* fn;
  int threads, grid, stages, ring_at;
  size_t smem;
};

// Dynamic shared memory of a CTA, at most: the rest is its static part.
constexpr size_t kMostSmem = kMaxSmemPerCta - 4096;

// Slots of a ring: as many, up to `most`, as leave room for three, two or one CTA per SM (228 KB, 1 KB of it
// reserved per CTA, and a little static shared memory), at least two; 0 when two do not fit.  Four slots always, with fewer
// CTAs, is the same within 2 % (backward of 16384 x 4096 bf16 84.3 instead of 83.5 us, of 16384 x 1024 29.3 instead of 28.6).
int ring_stages(size_t slot, int most, size_t fixed, int groups, size_t* smem) {
  for (size_t cap : {size_t{74 * 1024}, size_t{112 * 1024}, kMostSmem})
    for (int stages = most; stages >= 2; --stages)
      if (fixed + slot * stages * groups <= cap) {
        *smem = fixed + slot * stages * groups;
        return stages;
      }
  return 0;
}

int scale_kind(Layout layout, int group) { return layout == kOffset ? 4 : group == 0 ? 0 : group == 32 ? 1 : group == 64 ? 2 : 3; }

int plan(DeviceState& dev, const AddNormTable* t, Which which, Layout layout, int period, int64_t M, int64_t N,
         bool has_residual, int group, Plan* out) {
  const int vec = 16 / t->size_t_;
  const int64_t need = N / vec;  // whole packets, at most
  const AddNormShape* s = nullptr;
  out->stages = out->ring_at = 0;
  const int kind = layout == kAny ? 0 : scale_kind(layout, group);
  if (layout != kAny)
    for (int i = 0; i < t->n && s == nullptr; ++i) {
      const AddNormShape& c = t->shapes[i];
      const bool has = which == kFwd ? c.fwd[layout] != nullptr : which == kFp8 ? c.fp8[kind] != nullptr
                       : c.bwd[layout] != nullptr || c.bwd_ring[layout] != nullptr;
      if (has && c.capacity() >= need) s = &c;
    }
  int groups = 1;
  out->smem = 0;
  if (s != nullptr) {
    groups = s->groups();
    out->fn = which == kFwd ? s->fwd[layout] : which == kBwd ? s->bwd[layout] : s->fp8[kind];
    out->threads = s->threads();
    // off the packet boundaries, weights that are not in registers
    const size_t weights = layout == kOffset && s->ld * vec > 16 ? sizeof(float) * w_slots(static_cast<int>(N)) : 0;
    out->smem = weights;
    if (which == kFp8) {
      size_t fixed = 0;
      if (layout == kOffset)  // the maxima, two halves per row group
        fixed = weights + (sizeof(uint32_t) * 2 * groups * (group ? (N + group - 1) / group : 1) + 127) / 128 * 128;
      out->smem = fixed;
      const void* ring_fn = s->fp8_ring[kind];
      // two slots: four make 20480 x 4096 bf16 with a scale per 32 columns 56.4 instead of 54.8 us
      if (ring_fn != nullptr && !has_residual) {
        size_t ring = 0;
        out->stages = ring_stages(static_cast<size_t>(need) * vec * t->size_t_, 2, fixed, groups, &ring);
        if (out->stages > 0) {
          out->fn = ring_fn;
          out->smem = ring;
          out->ring_at = static_cast<int>(fixed);
        }
      }
    }
    if (which == kBwd) {
      const size_t fixed = weights + (addnorm_wide(s->ld, vec, s->tpr) ? sizeof(float) * s->ld * vec * s->tpr : 0);
      const size_t sums = groups > 1 ? sizeof(float) * groups * N : 0;
      const size_t slot = static_cast<size_t>(need) * vec * (t->size_t_ + t->size_r * (has_residual ? 2 : 1));
      size_t ring = 0;
      if (s->bwd_ring[layout] != nullptr) out->stages = ring_stages(slot, kAddNormStages, fixed, groups, &ring);
      if (out->stages > 0) out->fn = s->bwd_ring[layout];
      out->smem = std::max(ring, fixed + sums);
    }
    // a row without a kernel that fits
    if (out->fn == nullptr || out->smem > kMostSmem) s = nullptr;
  }
  if (s == nullptr) {
    out->fn = which == kFwd ? t->fwd_any : which == kFp8 ? t->fp8_any : t->bwd_any;
    out->threads = 512;
    out->smem = static_cast<size_t>(N) * sizeof(float);
    groups = 1;
  }
  int occ;
  if (int rc = occupancy(dev, out->fn, out->threads, out->smem, &occ)) return rc;
  const int64_t want = std::max<int64_t>(1, (M + groups - 1) / groups), resident = (int64_t)dev.sm_count * occ;
  int64_t grid = std::min(want, resident);
  // a row group's rows have to share one offset (see the kernels): a step that is a multiple of the period
  if (s != nullptr && layout == kOffset && grid < want) {
    const int64_t unit = period / std::gcd<int64_t>(period, groups);
    grid = std::max<int64_t>(unit, grid / unit * unit);
  }
  out->grid = static_cast<int>(grid);
  return B200NORM_OK;
}

int forward(bool fp8, const void* x, int64_t xs, const void* r, int64_t rs, const void* w, void* y, int64_t ys, void* scale,
            void* h, int64_t hs, float* rstd, int64_t M, int64_t N, float eps, int group, int e8m0, int io, int res,
            int w_dtype, void* stream) {
  if (int rc = check(M, N, io, res, w_dtype)) return rc;
  if (group != 0 && group != 32 && group != 64 && group != 128)
    return fail(B200NORM_ERR_ARG, "a scale covers 32, 64 or 128 columns, or (0) a row; got %d", group);
  if (M == 0) return B200NORM_OK;
  if (!x || !y || (fp8 && !scale) || (!fp8 && (!r || !h))) return fail(B200NORM_ERR_ARG, "null buffer");
  if (r == nullptr && h != nullptr) return fail(B200NORM_ERR_ARG, "h is the sum with a residual: there is none");
  if (xs < N || ys < N || (r && rs < N) || (h && hs < N)) return fail(B200NORM_ERR_ARG, "row stride smaller than N");
  const AddNormTable* t = table_for(io, res);
  if (!on_element(x, t->size_t_) || !on_element(r, t->size_r) || !on_element(w, dtype_size(w_dtype)) ||
      !on_element(y, fp8 ? 1 : t->size_t_) || !on_element(h, t->size_r) || !on_element(rstd, 4) || !on_element(scale, e8m0 ? 1 : 4))
    return fail_off_element();
  DeviceState* dev = nullptr;
  if (int rc = fp8 ? device_state(&dev) : device_caches(&dev)) return rc;
  const Buffer bufs[4] = {{x, xs, t->size_t_}, {r, rs, t->size_r}, {y, ys, fp8 ? 1 : t->size_t_}, {h, hs, t->size_r}};
  int period;
  const Layout layout = layout_of(bufs, 4, N, 16 / t->size_t_, w, &period);
  Plan pl;
  if (int rc = plan(*dev, t, fp8 ? kFp8 : kFwd, layout, period, M, N, r != nullptr, group, &pl)) return rc;
  AddNormParams p = {};
  p.x = x; p.r = r; p.w = w; p.y = y; p.h = h; p.rstd = rstd; p.scale = scale;
  p.x_stride = xs; p.r_stride = rs; p.y_stride = ys; p.h_stride = hs;
  p.stages = pl.stages; p.ring_at = pl.ring_at; p.status = dev->status_dev;
  p.M = M; p.N = static_cast<int>(N); p.w_dtype = w_dtype; p.eps = eps;
  p.group = group; p.groups_per_row = group ? static_cast<int>((N + group - 1) / group) : 1; p.e8m0 = e8m0 != 0;
  return launch(pl.fn, dim3(pl.grid), dim3(pl.threads), pl.smem, &p, static_cast<cudaStream_t>(stream));
}

}  // namespace
}  // namespace b200norm

using namespace b200norm;

extern "C" {

int b200norm_add_rms_fwd(const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride, const void* w,
                         void* y, int64_t y_row_stride, void* h, int64_t h_row_stride, float* rstd, int64_t M, int64_t N,
                         float eps, int io_dtype, int res_dtype, int w_dtype, void* stream) {
  return forward(false, x, x_row_stride, residual, residual_row_stride, w, y, y_row_stride, nullptr, h, h_row_stride, rstd, M,
                 N, eps, 0, 0, io_dtype, res_dtype, w_dtype, stream);
}

int b200norm_rms_fp8(const void* x, int64_t x_row_stride, const void* residual, int64_t residual_row_stride, const void* w,
                     void* q, int64_t q_row_stride, void* scale, void* h, int64_t h_row_stride, int64_t M, int64_t N,
                     float eps, int group, int e8m0, int io_dtype, int res_dtype, int w_dtype, void* stream) {
  return forward(true, x, x_row_stride, residual, residual_row_stride, w, q, q_row_stride, scale, h, h_row_stride, nullptr, M,
                 N, eps, group, e8m0, io_dtype, res_dtype, w_dtype, stream);
}

size_t b200norm_add_rms_bwd_workspace_bytes(int64_t M, int64_t N, int io_dtype, int res_dtype) {
  if (check(M, N, io_dtype, res_dtype, B200NORM_F32)) return 0;
  DeviceState* dev = nullptr;
  if (device_caches(&dev)) return 0;
  const AddNormTable* t = table_for(io_dtype, res_dtype);
  int64_t rows = 0;
  for (Layout layout : {kAligned, kOffset, kAny})  // whichever the buffers turn out to have
    for (bool has_dh : {false, true}) {
      Plan pl;
      if (plan(*dev, t, kBwd, layout, 1, M, N, has_dh, 0, &pl)) return 0;
      rows = std::max<int64_t>(rows, pl.grid);
    }
  return (static_cast<size_t>(rows) * N * sizeof(float) + 255) & ~static_cast<size_t>(255);
}

int b200norm_add_rms_bwd(const void* h, int64_t h_row_stride, const void* dy, int64_t dy_row_stride, const void* dh,
                         int64_t dh_row_stride, const void* w, const float* rstd, void* dx, int64_t dx_row_stride, void* dres,
                         int64_t dres_row_stride, void* dw, void* workspace, size_t workspace_bytes, int64_t M, int64_t N,
                         int io_dtype, int res_dtype, int w_dtype, void* stream_v) {
  if (int rc = check(M, N, io_dtype, res_dtype, w_dtype)) return rc;
  if (M == 0 && dw == nullptr) return B200NORM_OK;
  const bool split = io_dtype != res_dtype;
  if (M > 0 && (!h || !dy || !rstd || !dx || (split && !dres))) return fail(B200NORM_ERR_ARG, "null h / dy / rstd / dx / dres");
  if (!split && dres != nullptr)
    return fail(B200NORM_ERR_ARG, "dres is written only when the residual's type is not that of the rows: it equals dx");
  if (h_row_stride < N || dy_row_stride < N || dx_row_stride < N || (dh && dh_row_stride < N) || (dres && dres_row_stride < N))
    return fail(B200NORM_ERR_ARG, "row stride smaller than N");
  const AddNormTable* t = table_for(io_dtype, res_dtype);
  if (!on_element(h, t->size_r) || !on_element(dy, t->size_t_) || !on_element(dh, t->size_r) || !on_element(w, dtype_size(w_dtype)) ||
      !on_element(rstd, 4) || !on_element(dx, t->size_t_) || !on_element(dres, t->size_r) || !on_element(dw, dtype_size(w_dtype)))
    return fail_off_element();
  DeviceState* dev = nullptr;
  if (int rc = device_state(&dev)) return rc;
  const Buffer bufs[5] = {{dy, dy_row_stride, t->size_t_}, {h, h_row_stride, t->size_r}, {dh, dh_row_stride, t->size_r},
                          {dx, dx_row_stride, t->size_t_}, {dres, dres_row_stride, t->size_r}};
  int period;
  const Layout layout = layout_of(bufs, 5, N, 16 / t->size_t_, w, &period);
  Plan pl;
  if (int rc = plan(*dev, t, kBwd, layout, period, M, N, dh != nullptr, 0, &pl)) return rc;
  AddNormParams p = {};
  p.x = dy; p.r = dh; p.w = w; p.y = dx; p.h = const_cast<void*>(h); p.rstd = const_cast<float*>(rstd); p.dr = dres;
  p.x_stride = dy_row_stride; p.r_stride = dh_row_stride; p.y_stride = dx_row_stride; p.h_stride = h_row_stride;
  p.dr_stride = dres_row_stride;
  p.M = M; p.N = static_cast<int>(N); p.w_dtype = w_dtype;
  p.stages = pl.stages; p.status = dev->status_dev;
  if (dw != nullptr) {
    const size_t need = static_cast<size_t>(pl.grid) * N * sizeof(float);
    if (workspace == nullptr || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u))
      return fail(B200NORM_ERR_ARG, "workspace needs %zu bytes, 256-byte aligned (got %zu)", need, workspace_bytes);
    p.part = static_cast<float*>(workspace);
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  if (int rc = launch(pl.fn, dim3(pl.grid), dim3(pl.threads), pl.smem, &p, stream)) return rc;
  if (dw == nullptr) return B200NORM_OK;
  AddNormReduceParams c = {p.part, dw, pl.grid, static_cast<int>(N), w_dtype};
  return launch(reinterpret_cast<const void*>(&addnorm_reduce_kernel), dim3(static_cast<unsigned>((N + 31) / 32)), dim3(1024), 0,
                &c, stream);
}

}  // extern "C"
