// Residual addition + RMSNorm, forward and backward, and RMSNorm (with or without the residual
// addition) with an 8-bit output and scales.
//
//   forward    h = round_R(x + r);  rstd = 1 / sqrt(sum(h^2)/N + eps);  y = h * rstd * w
//   backward   xhat = h * rstd;  wdy = w * dy;  c1 = sum(xhat * wdy) / N
//              d = (wdy - xhat * c1) * rstd + dh;  dx = round_T(d), dr = round_R(d);  dw = sum_rows(dy * xhat)
//   8 bits     a_g = max |y| over a group of columns;  s_g = max(a_g, 2^-64) / 448 (or the next power of two
//              up);  q = e4m3(y / s_g), from the unrounded y; of a whole row a_g = rstd max |h w|
//
// T is the storage type of x, y, dy and dx; R that of the residual stream (r, h, dh, dr): T or fp32.  h is
// rounded to R before the statistics are taken, so that y is the norm of the h that is returned and that
// the backward reads; everything else stays fp32 until its one rounding on store.
//
// Most of it is bound by memory: the forward reads x, r and writes h, y, the backward reads h, dy, dh and
// writes one gradient (two when R is not T), so the aim is only to touch each byte once and to keep
// enough of them in flight.  A row lives in the registers of TPR threads, LD 16-byte packets each.
//   16384 x 4096 bf16           forward 84 us, backward 83: 0.98 of the copy bandwidth
//   6001 x 5120 bf16, fp32 h    forward 63 us (0.90), backward 76 (0.99)
//   16384 x 5120 bf16 to 8 bits, a scale a row, with residual  96 us (0.94)
//   8191 x 4104 fp16 to 8 bits, a scale per 32 columns  28 us (0.55): 20 instructions an element, the issue slots 67 % busy, the
//     rest of the time mostly in shared memory's latency and the row's barrier
//   8182 x 4101 bf16 (rows off the packet boundaries)  forward 45 us (0.91), backward 52 (0.79), to 8 bits per 128 columns 47
//     (0.33); 3001 x 1001 fp16 7 and 11 us, of which the launches, the first loads and the column reduce are half
//   229824 x 146 bf16  forward 66 us (0.62), backward 73 (0.56): 18 packets cost the instructions of 32
// The backward's ring makes 8192 x 8192 bf16 113 -> 86 us and 6001 x 5120 with fp32 h 100 -> 76; 16384 x 1024 is as quick
// without one.  The forward needs none (it writes as much as it reads), but for the 8-bit form without a residual: 20480 x 4096
// bf16, a scale per 32 columns, 63 -> 51 us.  (This pair and those at the choices of shapes were measured with quotients of one
// product; those of two, see Fp8Scale, add 2 to 8 % to 8-bit forms with fp32 scales: 51 -> 53 here.)
#pragma once

#include "norm_common.cuh"
#include "norm_stage.cuh"

namespace b200norm {

struct AddNormParams {
  // forward: x, r (null without a residual), w -> y (or q), h, rstd, scale
  // backward: h, dy (as x), dh (as r; null for none), w, rstd -> dx (as y), dr, part
  const void* x;
  const void* r;
  const void* w;  // may be null
  void* y;
  void* h;      // forward: may be null in the 8-bit form
  float* rstd;  // forward: may be null in the 8-bit form
  void* scale;  // 8-bit form
  float* part;  // backward: (gridDim.x, N) partial rows of dw, or null
  void* dr;     // backward: the gradient in R, null when R is T (it is dx then)
  int64_t x_stride, r_stride, y_stride, h_stride, dr_stride;  // elements
  int64_t M;
  int N;
  int w_dtype;
  float eps;
  int group;  // 8-bit form, element by element: columns per scale, 0 for one scale a row
  int groups_per_row;
  int e8m0;  // 8-bit form: scales are powers of two, stored as their biased exponent
  int stages;   // with a ring: slots per row group ...
  int ring_at;  // ... and, 8-bit form, where in the dynamic shared memory they begin
  int* status;  // device status word for bounded waits that ran out
};
constexpr int kAddNormStages = 4;  // slots of a ring, at most

constexpr float kE4m3Max = 448.f;
constexpr float kAmaxFloor = 5.421010862427522e-20f;  // 2^-64: a group of zeros still gets a finite scale

// VEC consecutive elements of E as raw registers.  The streams are read once, hence past L1.
template <typename E, int VEC>
struct RawVec {
  static constexpr int kWords = VEC * static_cast<int>(sizeof(E)) / 4;
  static_assert(kWords == 4 || kWords == 8, "16 or 32 bytes");
  uint32_t w[kWords];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void load(const E* p) {
    if constexpr (kWords == 4) {
      const uint4 v = ld_stream(reinterpret_cast<const uint4*>(p));
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    } else {
      asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p));
    }
  }
  __device__ __forceinline__ void load_shared(const void* p) {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) {
      const uint4 v = ld_shared16(static_cast<const unsigned char*>(p) + 16 * i);
      w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
  }
  __device__ __forceinline__ void store(E* p) const {
    if constexpr (kWords == 4) {
      st_stream(reinterpret_cast<uint4*>(p), make_uint4(w[0], w[1], w[2], w[3]));
    } else {
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                   "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
    }
  }
  __device__ __forceinline__ void unpack(float2* f) const {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < kWords / 2; ++i) f[i] = make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    } else {
      Pack16<E>::unpack2(make_uint4(w[0], w[1], w[2], w[3]), f);
    }
  }
  __device__ __forceinline__ void pack(const float2* f) {
    if constexpr (sizeof(E) == 4) {
#pragma unroll
      for (int i = 0; i < kWords / 2; ++i) {
        w[2 * i] = __float_as_uint(f[i].x);
        w[2 * i + 1] = __float_as_uint(f[i].y);
      }
    } else {
      const uint4 v = Pack16<E>::pack2(f);
      w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
  }
};

// Rows of one buffer.
template <typename E, int VEC>
struct Rows {
  E* base;
  int64_t stride;

  __device__ __forceinline__ Rows(const void* p, int64_t stride) : base(static_cast<E*>(const_cast<void*>(p))), stride(stride) {}
  __device__ __forceinline__ E* at(int64_t row, int c) const { return base + row * stride + c; }
  __device__ __forceinline__ RawVec<E, VEC> load(int64_t row, int c0) const {
    RawVec<E, VEC> r;
    r.load(at(row, c0));
    return r;
  }
  __device__ __forceinline__ void store(int64_t row, int c0, const RawVec<E, VEC>& r) const { r.store(at(row, c0)); }
};

// How a row of n columns lies on packet boundaries when it starts `off` elements behind one: a head of up to VEC - 1
// elements, whole packets, a tail of up to VEC - 1.  The packets are handled as those of an aligned row; the head's and the
// tail's elements are dealt out singly, EDGES a thread, and everything is done for them beside the packets, without a branch
// on their number.
template <int VEC, int TPR, bool OFF>
struct Span {
  static constexpr int EDGES = OFF ? (2 * VEC - 2 + TPR - 1) / TPR : 0;
  static constexpr int kSlots = OFF ? EDGES : 1;
  int head, packets, edges;

  __device__ __forceinline__ Span(int off, int n) {
    head = OFF ? min((VEC - off) % VEC, n) : 0;
    packets = (n - head) / VEC;
    edges = n - packets * VEC;
  }
  // Column of a thread's k-th single element, or -1.
  __device__ __forceinline__ int edge(int t, int k) const {
    const int i = t + k * TPR;
    return i >= edges ? -1 : i < head ? i : packets * VEC + i;
  }
};

// VEC parameter values from column c0, a multiple of VEC, of a 16-byte aligned vector.  The parameters are
// re-read by every row a CTA handles: L1 serves them.
template <int VEC>
__device__ __forceinline__ void load_w(const void* p, int dtype, int c0, float2* f) {
  float v[VEC];
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 1.f;
  } else if (dtype == kF32) {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(p) + c0) + i);
      v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w;
    }
  } else if (dtype == kF64) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = static_cast<float>(static_cast<const double*>(p)[c0 + e]);
  } else {
    uint32_t q[VEC / 2];
    const uint16_t* src = static_cast<const uint16_t*>(p) + c0;
    if constexpr (VEC == 8) {
      const uint4 t = __ldg(reinterpret_cast<const uint4*>(src));
      q[0] = t.x; q[1] = t.y; q[2] = t.z; q[3] = t.w;
    } else {
      const uint2 t = __ldg(reinterpret_cast<const uint2*>(src));
      q[0] = t.x; q[1] = t.y;
    }
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      if (dtype == kBF16) {
        v[2 * i] = __uint_as_float(q[i] << 16);
        v[2 * i + 1] = __uint_as_float(q[i] & 0xffff0000u);
      } else {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&q[i]));
        v[2 * i] = h.x;
        v[2 * i + 1] = h.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i) f[i] = make_float2(v[2 * i], v[2 * i + 1]);
}

// The same from any column, one by one.
template <int VEC>
__device__ __forceinline__ void load_w_any(const void* p, int dtype, int c0, float2* f) {
#pragma unroll
  for (int i = 0; i < VEC / 2; ++i)
    f[i] = p == nullptr ? splat2(1.f) : make_float2(load_param(p, dtype, c0 + 2 * i), load_param(p, dtype, c0 + 2 * i + 1));
}

// Rows off the packet boundaries, too wide for the weights to stay in registers: the packets' weights wait in shared memory
// as fp32, on packet boundaries like the rows' packets.
__host__ __device__ constexpr int w_slots(int n) { return (n + 31) / 32 * 32; }
template <int VEC>
__device__ __forceinline__ void staged_w(const float* ws, int pk, float2* f) {
#pragma unroll
  for (int i = 0; i < VEC / 4; ++i) {
    const float4 q = reinterpret_cast<const float4*>(ws + pk * VEC)[i];
    f[2 * i] = make_float2(q.x, q.y);
    f[2 * i + 1] = make_float2(q.z, q.w);
  }
}

// Maxima of magnitudes that keep a NaN, so that a poisoned group shows in its scale.
__device__ __forceinline__ float max_abs(float a, float b) {
  float r;
  asm("max.NaN.xorsign.abs.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return fabsf(r);
}
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float warp_max_abs(float v) {
  float r;
  asm volatile("redux.sync.max.abs.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// A group's scale from its largest magnitude, the byte that a power-of-two scale is stored as, and 1 / scale as a sum of two
// numbers.  An fp32 scale is the product with 1 / 448, within an ulp of the quotient.  With 48 bits of 1 / scale a quotient
// y / scale comes out correctly rounded (but for one within 2^-24 of an ulp of the middle between two fp32 numbers).  One that lies
// on a border between two e4m3 values has to: y * (1 / scale) alone, an ulp off now and then, put 6 % of those on the wrong side,
// and 16-bit rows and weights have such quotients (one in 10^4 of 16384 x 5120 bf16).
struct Fp8Scale {
  float scale, inv, inv_low;
  uint32_t code;
};
__device__ __forceinline__ Fp8Scale fp8_scale(float amax, bool e8m0) {
  Fp8Scale r;
  amax = max_abs(amax, kAmaxFloor);
  r.inv_low = 0.f;
  if (e8m0) {
    // The lowest 2^e with amax <= 448 * 2^e = 1.75 * 2^(e + 8): eight below amax's exponent, or seven where its fraction is
    // above .75.  The reciprocal of a power of two is one, too.
    const uint32_t bits = __float_as_uint(amax), e = (bits >> 23) - 8u + ((bits & 0x7fffffu) > 0x600000u ? 1u : 0u);
    const bool bad = bits >= 0x7f800000u;  // infinity and NaN have the NaN code
    r.code = bad ? 255u : e;
    r.scale = 0.f;
    r.inv = __uint_as_float(bad ? 0x7fffffffu : (254u - e) << 23);
  } else {
    r.code = 0;
    r.scale = amax * (1.f / kE4m3Max);
    r.inv = rcp_fast(r.scale);
    if (r.scale < INFINITY) r.inv_low = fmaf(-r.scale, r.inv, 1.f) * r.inv;  // of an infinite scale 0: 0 / inf is 0
  }
  return r;
}
__device__ __forceinline__ float2 fp8_quotient2(float2 y, float2 inv, float2 low) { return fma2(y, inv, mul2(y, low)); }
__device__ __forceinline__ float fp8_quotient(float y, const Fp8Scale& s) { return fmaf(y, s.inv, y * s.inv_low); }
__device__ __forceinline__ void store_scale(void* p, int64_t at, const Fp8Scale& s, bool e8m0) {
  if (e8m0) static_cast<uint8_t*>(p)[at] = static_cast<uint8_t>(s.code);
  else static_cast<float*>(p)[at] = s.scale;
}

__device__ __forceinline__ uint32_t fp8x2(float lo, float hi) {  // saturating, NaN stays NaN
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// Threads of a CTA: row groups of fewer than 160 threads share one.
__host__ __device__ constexpr int addnorm_threads(int tpr) { return tpr < 160 ? 256 / tpr * tpr : tpr; }

// Whether a backward thread's LD * VEC dweight sums go to shared memory: they would not fit in the
// registers beside the row.
__host__ __device__ constexpr bool addnorm_wide(int ld, int vec, int tpr) { return ld * vec > 24 || tpr > 768; }

// CTAs per SM that the register allocation leaves room for, as so many threads: forward 512 (128 registers) above 16 elements a
// thread, else 768 (80) or, `lean`, 1024 (64); backward 512 or, lean, 768.  Lean are all forwards but the one through a ring with a
// scale a row, and backwards of up to 8 elements without a ring.  It makes the forward of 8182 x 4101 bf16 50 -> 45 us, of 4091 x
// 4101 fp32 61 -> 45, the 8-bit form of 8192 x 8192 bf16 58 -> 48, the backward of 335544 x 100 bf16 85 -> 72, and costs
// 16384 x 2048 bf16 forward 2 us of 43.  Lean forwards spill a little: 4 to 76 bytes a thread in a dozen kernels of 16-bit rows on
// 8 to 128 threads, up to 192 in those with an fp32 residual, up to 52 in fp32 ones of four packets; the times are with that.  1024
// threads have no more than 64 registers: with two packets up to 24 bytes are spilled, with four 12 to 484.
__host__ __device__ constexpr int addnorm_fwd_ctas(int elements, int tpr, bool lean) {
  const int n = (elements > 16 ? 512 : lean ? 1024 : 768) / addnorm_threads(tpr);
  return n < 1 ? 1 : n;
}
__host__ __device__ constexpr int addnorm_bwd_ctas(int tpr, bool lean) {
  const int n = (lean ? 768 : 512) / addnorm_threads(tpr);
  return n < 1 ? 1 : n;
}

// After a wait that ran out: the copies that a row group has in flight get a bounded chance to land.
__device__ __forceinline__ void addnorm_drain(uint64_t* bars, int stages, int64_t rows) {
  const unsigned long long t0 = global_ns();
  for (int s = 0; s < stages && s < rows; ++s) {
    const int64_t fills = (rows - s + stages - 1) / stages;
    while (!mbar_try_wait(&bars[s], static_cast<uint32_t>((fills - 1) & 1)))
      if (global_ns() - t0 > 10000000ull) return;
  }
}

// Sum over the TPR threads that share a row.  `scratch`: two halves, used in turn, of one float per warp, padded with zeros to
// whole 16-byte words; every thread adds all warps' sums in one order.
__host__ __device__ constexpr int row_scratch(int tpr) { return tpr <= 32 ? 4 : (tpr / 32 + 3) / 4 * 4; }
template <int TPR, int FIRST>
__device__ __forceinline__ float row_sum(float v, float* scratch, int& phase, int group, int warp_n, int lane) {
  if constexpr (TPR <= 32) {
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  } else {
    v = warp_sum(v);
    float* buf = scratch + phase * row_scratch(TPR);
    if (lane == 0) buf[warp_n] = v;
    group_sync<TPR / 32, FIRST>(group);
    float2 s = splat2(0.f);
#pragma unroll
    for (int k = 0; k < row_scratch(TPR) / 4; ++k) {
      const float4 q = reinterpret_cast<const float4*>(buf)[k];
      s = add2(s, make_float2(q.x, q.y));
      s = add2(s, make_float2(q.z, q.w));
    }
    phase ^= 1;
    return s.x + s.y;
  }
}

// The same, and the largest magnitude, with one barrier for both.
template <int TPR>
__device__ __forceinline__ float row_sum_max(float v, float& amax, float* scratch, float* max_scratch, int& phase, int group,
                                             int warp_n, int lane) {
  if constexpr (TPR <= 32) {
#pragma unroll
    for (int o = TPR / 2; o > 0; o >>= 1) amax = max_abs(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  } else {
    amax = warp_max_abs(amax);
    float* buf = max_scratch + phase * row_scratch(TPR);
    if (lane == 0) buf[warp_n] = amax;
    v = row_sum<TPR, 0>(v, scratch, phase, group, warp_n, lane);
#pragma unroll
    for (int k = 0; k < row_scratch(TPR) / 4; ++k) {
      const float4 q = reinterpret_cast<const float4*>(buf)[k];
      amax = max_abs3(max_abs3(amax, q.x, q.y), q.z, q.w);
    }
    return v;
  }
  return row_sum<TPR, 0>(v, scratch, phase, group, warp_n, lane);
}

// Forward.  OFF: the rows of all buffers start at one common offset within a packet that need not be
// zero (contiguous tensors of an odd row length); see Span.  The launch gives every row group rows of one offset
// only (its step is a multiple of the offsets' period), so that a thread's columns stay the same.
// GROUP: the 8-bit form with a scale for so many columns, 0 for one a row; -1: the output is y.  Thread t of a
// row group holds packets t, t + TPR, ...: neighbouring lanes hold neighbouring columns, so a scale's 32, 64 or
// 128 columns are 4 to 32 adjacent lanes of one warp, or all lanes of a group of 8 or 16 and several of their packets.  OFF: a packet may belong to two scales' columns, so the
// maxima are found in shared memory, by one or two atomic maxima a packet; the columns per scale are those of p.group.
// RING: as in the backward below, the rows of x arrive through p.stages shared-memory slots per row group.  For the 8-bit form
// without a residual; with one, as for y, as much is written as read, and direct loads by more threads are quicker: 20480 x
// 4096 bf16, a scale a row 108 -> 90 us, per 128 columns 103 -> 95.
template <typename T, typename R, int LD, int TPR, bool OFF, int GROUP, bool RING>
__global__ void __launch_bounds__(addnorm_threads(TPR),
                                  addnorm_fwd_ctas(LD * Pack16<T>::kElems, TPR, OFF || GROUP != 0 || !RING))
    addnorm_fwd_kernel(const AddNormParams p) {
  constexpr bool FP8 = GROUP >= 0, PER_ROW = GROUP == 0 && !OFF;
  static_assert(!(OFF && GROUP > 0), "rows off the packets read p.group");
  static_assert(!RING || TPR > 32, "a ring belongs to a group with a barrier");
  constexpr int VEC = Pack16<T>::kElems, H = VEC / 2;
  constexpr int GROUPS = addnorm_threads(TPR) / TPR;
  constexpr int WARPS = TPR >= 32 ? TPR / 32 : 1;
  constexpr bool WREG = LD * VEC <= 16;  // the weights fit in registers next to the row
  static_assert(!OFF || WREG || GROUPS == 1, "staged weights have one offset");
  // OFF: the weights unless in registers, and of the 8-bit form the maxima, two halves in turn per row group; RING: the slots
  extern __shared__ __align__(128) unsigned char dyn[];
  float* ws = reinterpret_cast<float*>(dyn);
  __shared__ __align__(8) uint64_t bars[RING ? GROUPS : 1][kAddNormStages];
  __shared__ int cta_abort;
  __shared__ __align__(16) float scratch[GROUPS][2 * row_scratch(TPR)];
  __shared__ __align__(16) float max_scratch[FP8 ? GROUPS : 1][2 * row_scratch(TPR)];

  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int lane = threadIdx.x & 31, warp_n = TPR >= 32 ? t / 32 : 0;
  int phase = 0;
  // PAIR: the row comes out of shared memory, where neighbouring packets cost nothing: a thread takes them two by two, which
  // halves the work per scale.
  constexpr bool PAIR = RING && GROUP > 0 && LD % 2 == 0;
  auto packet = [&](int j) { return PAIR ? (j / 2 * TPR + t) * 2 + j % 2 : j * TPR + t; };
  if constexpr (TPR > 32) {
    for (int i = threadIdx.x; i < GROUPS * 2 * row_scratch(TPR); i += blockDim.x) {
      (&scratch[0][0])[i] = 0.f;
      if (FP8) (&max_scratch[0][0])[i] = 0.f;
    }
    if (RING && threadIdx.x == 0) {
      for (int g = 0; g < GROUPS; ++g)
        for (int i = 0; i < p.stages; ++i) mbar_init(&bars[g][i], 1);
      cta_abort = 0;
      mbar_init_fence();
    }
    __syncthreads();
  }
  grid_dependency_sync();
  trigger_dependents();

  const Rows<T, VEC> xs(p.x, p.x_stride), ys(p.y, p.y_stride);
  const Rows<R, VEC> rs(p.r, p.r_stride), hs(p.h, p.h_stride);
  const int64_t first = (int64_t)blockIdx.x * GROUPS + group;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const int off = OFF ? static_cast<int>((reinterpret_cast<uintptr_t>(p.x) / sizeof(T) + first * p.x_stride) % VEC) : 0;
  const Span<VEC, TPR, OFF> span(off, p.N);
  const int packets = span.packets, head = span.head;
  const float inv_n = 1.f / static_cast<float>(p.N);
  const bool has_r = !RING && p.r != nullptr;
  // a slot has room for as many packets as rows of any offset have; a row's own may be one fewer
  const uint32_t slot_bytes = p.N / VEC * VEC * sizeof(T);
  unsigned char* slots = dyn + p.ring_at + (size_t)group * p.stages * slot_bytes;
  auto fill = [&](int s, int64_t row) {  // the group's first thread: x of a row into slot s
    mbar_expect_tx(&bars[group][s], packets * VEC * sizeof(T));
    bulk_load(slots + (size_t)s * slot_bytes, xs.at(row, head), packets * VEC * sizeof(T), &bars[group][s]);
  };
  if constexpr (RING) {
    if (t == 0)
      for (int s = 0; s < p.stages; ++s)
        if (first + s * step < p.M) fill(s, first + s * step);
  }
  int slot = 0;
  uint32_t parity = 0;

  uint32_t* maxima = reinterpret_cast<uint32_t*>(ws + (WREG ? 0 : w_slots(p.N))) + (size_t)group * 2 * p.groups_per_row;
  int half = 0;
  const int group_bits = 31 - __clz(p.group | 1);  // the columns per scale are a power of two
  constexpr int EDGES = Span<VEC, TPR, OFF>::EDGES, SLOTS = Span<VEC, TPR, OFF>::kSlots;
  int ec[SLOTS];  // the single elements' columns and weights
  float ew[SLOTS];
  if constexpr (OFF) {
#pragma unroll
    for (int k = 0; k < EDGES; ++k) {
      ec[k] = span.edge(t, k);
      ew[k] = ec[k] >= 0 && p.w != nullptr ? load_param(p.w, p.w_dtype, ec[k]) : 1.f;
    }
    if constexpr (!WREG)
      for (int i = threadIdx.x; i < packets * VEC; i += blockDim.x) ws[i] = p.w != nullptr ? load_param(p.w, p.w_dtype, head + i) : 1.f;
    if (FP8)
      for (int i = t; i < 2 * p.groups_per_row; i += TPR) maxima[i] = 0u;
    if (!WREG || FP8) __syncthreads();
  }
  auto weights = [&](int pk, float2* f) {
    if constexpr (!OFF) load_w<VEC>(p.w, p.w_dtype, pk * VEC, f);
    else if constexpr (WREG) load_w_any<VEC>(p.w, p.w_dtype, head + pk * VEC, f);
    else staged_w<VEC>(ws, pk, f);
  };
  // Packets past a row's end are zeros, with weights of zero: what is done to them in registers needs no test.
  float2 wr[WREG ? LD : 1][H];
  if constexpr (WREG) {
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int pk = packet(j);
#pragma unroll
      for (int k = 0; k < H; ++k) wr[j][k] = splat2(0.f);
      if (pk < packets) weights(pk, wr[j]);
    }
  }

  // Rows of fewer than 32 threads share a warp: the loop runs while the warp's first row is a row.
  const int64_t lead = TPR < 32 ? (int64_t)blockIdx.x * GROUPS + (threadIdx.x & ~31) / TPR : first;
  for (int64_t i = 0; lead + i < p.M; i += step) {
    const int64_t row = first + i;
    const bool valid = TPR >= 32 || row < p.M;

    float2 hf[LD][H];
    float eh[SLOTS];
    {
      T xe[SLOTS];
      R re[SLOTS];
#pragma unroll
      for (int k = 0; k < EDGES; ++k) {  // ahead of the wait for the packets
        xe[k] = from_f32<T>(0.f);
        re[k] = from_f32<R>(0.f);
        if (!valid || ec[k] < 0) continue;
        xe[k] = *xs.at(row, ec[k]);
        if (has_r) re[k] = *rs.at(row, ec[k]);
      }
      RawVec<T, VEC> xv[LD];
      RawVec<R, VEC> rv[LD];
      const unsigned char* src = slots + (size_t)slot * slot_bytes;
      if constexpr (RING) mbar_wait(&bars[group][slot], parity, &cta_abort, p.status);
#pragma unroll
      for (int j = 0; j < LD; ++j) {
        const int pk = packet(j);
        xv[j].zero();
        rv[j].zero();
        if (!valid || pk >= packets) continue;
        if constexpr (RING) {
          xv[j].load_shared(src + (size_t)pk * VEC * sizeof(T));
        } else {
          xv[j] = xs.load(row, head + pk * VEC);
          if (has_r) rv[j] = rs.load(row, head + pk * VEC);
        }
      }
#pragma unroll
      for (int j = 0; j < LD; ++j) {
        const int pk = packet(j);
        xv[j].unpack(hf[j]);
        if (has_r) {
          float2 rf[H];
          rv[j].unpack(rf);
#pragma unroll
          for (int k = 0; k < H; ++k) hf[j][k] = add2(hf[j][k], rf[k]);
          rv[j].pack(hf[j]);
          if (sizeof(R) < 4) rv[j].unpack(hf[j]);  // the norm is that of h as stored
          if (p.h != nullptr && valid && pk < packets) hs.store(row, head + pk * VEC, rv[j]);
        }
      }
#pragma unroll
      for (int k = 0; k < EDGES; ++k) {
        eh[k] = to_f32(xe[k]);
        if (has_r) {
          const R v = from_f32<R>(eh[k] + to_f32(re[k]));
          eh[k] = to_f32(v);
          if (p.h != nullptr && valid && ec[k] >= 0) *hs.at(row, ec[k]) = v;
        }
      }
    }

    float2 q2 = splat2(0.f);
#pragma unroll
    for (int j = 0; j < LD; ++j)
#pragma unroll
      for (int k = 0; k < H; ++k) q2 = fma2(hf[j][k], hf[j][k], q2);
#pragma unroll
    for (int k = 0; k < EDGES; ++k) q2.x = fmaf(eh[k], eh[k], q2.x);
    auto w_of = [&](int j, float2* wf) {
      if constexpr (WREG) {
#pragma unroll
        for (int k = 0; k < H; ++k) wf[k] = wr[j][k];
      } else {
        weights(packet(j), wf);
      }
    };
    // One scale a row: max |y| is rstd * max |h w|, so the maximum is found along with the sum.
    float q, amax = 0.f;
    if constexpr (PER_ROW) {
#pragma unroll
      for (int j = 0; j < LD; ++j) {
        if (!WREG && packet(j) >= packets) continue;
        float2 wf[H];
        w_of(j, wf);
#pragma unroll
        for (int k = 0; k < H; ++k) {
          const float2 v = mul2(hf[j][k], wf[k]);
          amax = max_abs3(amax, v.x, v.y);
        }
      }
      q = row_sum_max<TPR>(q2.x + q2.y, amax, scratch[group], max_scratch[group], phase, group, warp_n, lane);
    } else {
      q = row_sum<TPR, 0>(q2.x + q2.y, scratch[group], phase, group, warp_n, lane);
    }
    if constexpr (RING) {  // behind a barrier that every thread passes with its packets read
      if (t == 0 && row + p.stages * step < p.M) fill(slot, row + p.stages * step);
      if (++slot == p.stages) {
        slot = 0;
        parity ^= 1u;
      }
    }
    const float rstd = rsqrtf(q * inv_n + p.eps);
    if (t == 0 && valid && p.rstd != nullptr) p.rstd[row] = rstd;
    const float2 r2 = splat2(rstd);

    float amax_j[FP8 ? LD : 1];
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int pk = packet(j);
      if constexpr (FP8) amax_j[j] = 0.f;
      if (!WREG && pk >= packets) continue;
      float2 wf[H];
      w_of(j, wf);
#pragma unroll
      for (int k = 0; k < H; ++k) hf[j][k] = mul2(mul2(hf[j][k], r2), wf[k]);
      if constexpr (!FP8) {
        RawVec<T, VEC> o;
        o.pack(hf[j]);
        if (valid && pk < packets) ys.store(row, head + pk * VEC, o);
      } else if constexpr (!PER_ROW && !OFF) {
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < H; ++k) a = max_abs3(a, hf[j][k].x, hf[j][k].y);
        amax_j[j] = a;
      }
    }

#pragma unroll
    for (int k = 0; k < EDGES; ++k) {
      eh[k] = eh[k] * rstd * ew[k];
      if (!FP8 && valid && ec[k] >= 0) *ys.at(row, ec[k]) = from_f32<T>(eh[k]);
    }

    if constexpr (FP8 && OFF) {
      // Bit patterns of magnitudes order like the magnitudes, NaN above all.
      uint32_t* mx = maxima + half * p.groups_per_row;
      auto group_of = [&](int c) { return p.group == 0 ? 0 : c >> group_bits; };
      auto parts = [&](int c0, int& g0, int& cut) {  // a packet's first scale, and its elements from which the next one holds
        g0 = group_of(c0);
        cut = p.group == 0 ? VEC : (g0 + 1) * p.group - c0;
      };
      float whole = 0.f;
#pragma unroll
      for (int j = 0; j < LD; ++j) {
        const int pk = packet(j), c0 = head + pk * VEC;
        if (!valid || pk >= packets) continue;
        int g0, cut;
        parts(c0, g0, cut);
        float lo = 0.f, hi = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const float v = (e & 1) ? hf[j][e / 2].y : hf[j][e / 2].x;
          if (e < cut) lo = max_abs(lo, v);
          else hi = max_abs(hi, v);
        }
        if (p.group == 0) {
          whole = max_abs(whole, lo);
        } else {
          atomicMax(&mx[g0], __float_as_uint(lo));
          if (cut < VEC) atomicMax(&mx[g0 + 1], __float_as_uint(hi));
        }
      }
#pragma unroll
      for (int k = 0; k < EDGES; ++k) {
        if (!valid || ec[k] < 0) continue;
        if (p.group == 0) whole = max_abs(whole, eh[k]);
        else atomicMax(&mx[group_of(ec[k])], __float_as_uint(max_abs(0.f, eh[k])));
      }
      if (p.group == 0 && valid) atomicMax(&mx[0], __float_as_uint(whole));
      if constexpr (TPR > 32) group_sync<WARPS, 0>(group);
      else __syncwarp();
      // the other half is free: every thread is past the row before
      uint32_t* other = maxima + (half ^ 1) * p.groups_per_row;
      for (int g = t; g < p.groups_per_row; g += TPR) {
        if (valid) store_scale(p.scale, row * p.groups_per_row + g, fp8_scale(__uint_as_float(mx[g]), p.e8m0 != 0), p.e8m0 != 0);
        other[g] = 0u;
      }
      if constexpr (TPR <= 32) __syncwarp();  // wider groups meet at the next row's first barrier
      half ^= 1;
      uint8_t* qrow = static_cast<uint8_t*>(p.y) + row * p.y_stride;
#pragma unroll
      for (int j = 0; j < LD; ++j) {
        const int pk = packet(j), c0 = head + pk * VEC;
        if (!valid || pk >= packets) continue;
        int g0, cut;
        parts(c0, g0, cut);
        const Fp8Scale lo = fp8_scale(__uint_as_float(mx[g0]), p.e8m0 != 0);
        const Fp8Scale hi = cut < VEC ? fp8_scale(__uint_as_float(mx[g0 + 1]), p.e8m0 != 0) : lo;
        auto pair = [&](int e) {  // elements e and e + 1
          const float2 inv = make_float2(e < cut ? lo.inv : hi.inv, e + 1 < cut ? lo.inv : hi.inv);
          const float2 low = make_float2(e < cut ? lo.inv_low : hi.inv_low, e + 1 < cut ? lo.inv_low : hi.inv_low);
          const float2 v = fp8_quotient2(hf[j][e / 2], inv, low);
          return fp8x2(v.x, v.y);
        };
        uint32_t word[VEC / 4];
#pragma unroll
        for (int k = 0; k < VEC / 4; ++k) word[k] = pair(4 * k) | (pair(4 * k + 2) << 16);
        if constexpr (VEC == 8) __stcs(reinterpret_cast<uint2*>(qrow + c0), make_uint2(word[0], word[1]));
        else __stcs(reinterpret_cast<uint32_t*>(qrow + c0), word[0]);
      }
#pragma unroll
      for (int k = 0; k < EDGES; ++k) {
        if (!valid || ec[k] < 0) continue;
        const Fp8Scale sc = fp8_scale(__uint_as_float(mx[group_of(ec[k])]), p.e8m0 != 0);
        qrow[ec[k]] = static_cast<uint8_t>(fp8x2(fp8_quotient(eh[k], sc), 0.f));
      }
    }
    if constexpr (FP8 && !OFF) {
      uint8_t* qrow = static_cast<uint8_t*>(p.y) + row * p.y_stride;
      Fp8Scale sc;
      if constexpr (PER_ROW) {
        // A sum of squares that overflows makes rstd 0 and y 0, or NaN where h is infinite; and a product h w may overflow,
        // along with it or for a large weight alone, where y does not.  The maximum is then taken again, of y itself.
        const bool over = rstd == 0.f || amax == INFINITY;
        amax *= rstd;
        const bool again = TPR <= 32 ? __any_sync(0xffffffffu, over) : over;
        if (again) {
          float a = 0.f;
#pragma unroll
          for (int j = 0; j < LD; ++j)
#pragma unroll
            for (int k = 0; k < H; ++k) a = max_abs3(a, hf[j][k].x, hf[j][k].y);
          row_sum_max<TPR>(0.f, a, scratch[group], max_scratch[group], phase, group, warp_n, lane);
          if (over) amax = a;
        }
        sc = fp8_scale(amax, p.e8m0 != 0);
        if (t == 0 && valid) store_scale(p.scale, row, sc, p.e8m0 != 0);
      }
      constexpr int SPAN = PAIR ? 2 * VEC : VEC;  // neighbouring columns of a thread
      constexpr int LANES = PER_ROW ? 1 : (GROUP / SPAN < TPR ? GROUP / SPAN : TPR);  // adjacent lanes that share a scale
      constexpr int JS = PER_ROW || GROUP <= TPR * SPAN ? 1 : GROUP / (TPR * SPAN) < LD ? GROUP / (TPR * SPAN) : LD;  // ... and packets of a lane
#pragma unroll
      for (int j = 0; j < LD; ++j) {
        const int pk = packet(j);
        if (!PER_ROW && !(PAIR && j % 2 == 1) && j % JS == 0) {
          float a = amax_j[j];
#pragma unroll
          for (int k = 1; k < JS; ++k) a = max_abs(a, amax_j[j + k < LD ? j + k : j]);
          if constexpr (PAIR) a = max_abs(a, amax_j[j + 1 < LD ? j + 1 : j]);
#pragma unroll
          for (int o = 1; o < LANES; o <<= 1) a = max_abs(a, __shfl_xor_sync(0xffffffffu, a, o));
          sc = fp8_scale(a, p.e8m0 != 0);
          if (valid && pk < packets && (t & (LANES - 1)) == 0)
            store_scale(p.scale, row * p.groups_per_row + pk * VEC / (PER_ROW ? 1 : GROUP), sc, p.e8m0 != 0);
        }
        if (valid && pk < packets) {
          const float2 inv2 = splat2(sc.inv), low2 = splat2(sc.inv_low);
          uint32_t word[VEC / 4];
          auto divide = [&](auto quotient) {
#pragma unroll
            for (int k = 0; k < VEC / 4; ++k) {
              const float2 lo = quotient(hf[j][2 * k]), hi = quotient(hf[j][2 * k + 1]);
              word[k] = fp8x2(lo.x, lo.y) | (fp8x2(hi.x, hi.y) << 16);
            }
          };
          if (p.e8m0) divide([&](float2 v) { return mul2(v, inv2); });
          else divide([&](float2 v) { return fp8_quotient2(v, inv2, low2); });
          if constexpr (VEC == 8) __stcs(reinterpret_cast<uint2*>(qrow + pk * VEC), make_uint2(word[0], word[1]));
          else __stcs(reinterpret_cast<uint32_t*>(qrow + pk * VEC), word[0]);
        }
      }
    }
  }
  if constexpr (RING) {
    if (t == 0 && cta_abort) addnorm_drain(bars[group], p.stages, first < p.M ? (p.M - first + step - 1) / step : 0);
  }
}

// Backward.  A thread owns fixed columns of every row its group visits and carries their dweight sums:
// in registers, or (WIDE) in shared memory, laid out so that lane t touches word t.  The row groups of a
// CTA are added in order at the end: one partial row per CTA.
//
// RING: the rows of h, dy and dh reach the registers through a ring of p.stages shared-memory slots per row
// group, filled by bulk asynchronous copies, so that whole rows stay in flight while others are reduced.
// A slot is refilled behind the row's reduction, a barrier that every thread passes with its packets read.
template <typename T, typename R, int LD, int TPR, bool OFF, bool RING>
__global__ void __launch_bounds__(addnorm_threads(TPR),
                                  addnorm_bwd_ctas(TPR, !RING && LD * Pack16<T>::kElems <= 8))
    addnorm_bwd_kernel(const AddNormParams p) {
  static_assert(!RING || TPR > 32, "a ring belongs to a group with a barrier");
  constexpr int VEC = Pack16<T>::kElems, H = VEC / 2;
  constexpr int GROUPS = addnorm_threads(TPR) / TPR;
  constexpr bool WREG = LD * VEC <= 16;
  constexpr bool WIDE = addnorm_wide(LD, VEC, TPR);
  static_assert(!OFF || WREG || GROUPS == 1, "staged weights have one offset");
  // OFF: the weights unless in registers; then the sums, WIDE [LD * VEC][TPR] or, of several groups, [GROUPS][N]; RING: the
  // slots, which the sums of several groups reuse
  extern __shared__ __align__(128) unsigned char dyn[];
  float* ws = reinterpret_cast<float*>(dyn);
  float* acc = ws + (OFF && !WREG ? w_slots(p.N) : 0);
  __shared__ __align__(16) float scratch[GROUPS][2 * row_scratch(TPR)];
  __shared__ __align__(8) uint64_t bars[RING ? GROUPS : 1][kAddNormStages];
  __shared__ int cta_abort;

  const int group = threadIdx.x / TPR, t = threadIdx.x % TPR;
  const int lane = threadIdx.x & 31, warp_n = TPR >= 32 ? t / 32 : 0;
  int phase = 0;
  for (int i = threadIdx.x; i < GROUPS * 2 * row_scratch(TPR); i += blockDim.x) (&scratch[0][0])[i] = 0.f;
  if constexpr (RING) {
    if (threadIdx.x == 0) {
      for (int g = 0; g < GROUPS; ++g)
        for (int i = 0; i < p.stages; ++i) mbar_init(&bars[g][i], 1);
      cta_abort = 0;
      mbar_init_fence();
    }
  }
  __syncthreads();
  grid_dependency_sync();
  trigger_dependents();

  const Rows<T, VEC> gs(p.x, p.x_stride), dxs(p.y, p.y_stride);
  const Rows<R, VEC> hs(p.h, p.h_stride), ds(p.r, p.r_stride), drs(p.dr, p.dr_stride);
  const int64_t first = (int64_t)blockIdx.x * GROUPS + group;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const int off = OFF ? static_cast<int>((reinterpret_cast<uintptr_t>(p.x) / sizeof(T) + first * p.x_stride) % VEC) : 0;
  const Span<VEC, TPR, OFF> span(off, p.N);
  const int packets = span.packets, head = span.head;
  const float inv_n = 1.f / static_cast<float>(p.N);

  // a slot has room for as many packets as rows of any offset have; a row's own may be one fewer
  const uint32_t t_bytes = p.N / VEC * VEC * sizeof(T), r_bytes = p.N / VEC * VEC * sizeof(R);
  const uint32_t slot_bytes = t_bytes + r_bytes * (p.r != nullptr ? 2 : 1);
  unsigned char* slots = reinterpret_cast<unsigned char*>(acc + (WIDE ? LD * VEC * TPR : 0)) + (size_t)group * p.stages * slot_bytes;
  auto fill = [&](int s, int64_t row) {  // the group's first thread: dy, h, dh of a row into slot s
    unsigned char* dst = slots + (size_t)s * slot_bytes;
    uint64_t* bar = &bars[group][s];
    const uint32_t tb = packets * VEC * sizeof(T), rb = packets * VEC * sizeof(R);
    mbar_expect_tx(bar, tb + rb * (p.r != nullptr ? 2 : 1));
    bulk_load(dst, gs.at(row, head), tb, bar);
    bulk_load(dst + t_bytes, hs.at(row, head), rb, bar);
    if (p.r != nullptr) bulk_load(dst + t_bytes + r_bytes, ds.at(row, head), rb, bar);
  };
  if constexpr (RING) {
    if (t == 0)
      for (int s = 0; s < p.stages; ++s)
        if (first + s * step < p.M) fill(s, first + s * step);
  }
  constexpr int EDGES = Span<VEC, TPR, OFF>::EDGES, SLOTS = Span<VEC, TPR, OFF>::kSlots;
  int ec[SLOTS];  // the single elements' columns, weights and dweight sums
  float ew[SLOTS], edw[SLOTS];
  if constexpr (OFF) {
#pragma unroll
    for (int k = 0; k < EDGES; ++k) {
      ec[k] = span.edge(t, k);
      ew[k] = ec[k] >= 0 && p.w != nullptr ? load_param(p.w, p.w_dtype, ec[k]) : 1.f;
      edw[k] = 0.f;
    }
    if constexpr (!WREG) {
      for (int i = threadIdx.x; i < packets * VEC; i += blockDim.x) ws[i] = p.w != nullptr ? load_param(p.w, p.w_dtype, head + i) : 1.f;
      __syncthreads();
    }
  }
  auto weights = [&](int pk, float2* f) {
    if constexpr (!OFF) load_w<VEC>(p.w, p.w_dtype, pk * VEC, f);
    else if constexpr (WREG) load_w_any<VEC>(p.w, p.w_dtype, head + pk * VEC, f);
    else staged_w<VEC>(ws, pk, f);
  };
  float2 wr[WREG ? LD : 1][H];
  float2 dw[WIDE ? 1 : LD][H];
  if constexpr (WREG) {
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int pk = j * TPR + t;
#pragma unroll
      for (int k = 0; k < H; ++k) wr[j][k] = splat2(0.f);  // packets past a row's end: zeros all the way
      if (pk < packets) weights(pk, wr[j]);
    }
  }
  if constexpr (WIDE) {
#pragma unroll
    for (int k = 0; k < LD * VEC; ++k) acc[k * TPR + t] = 0.f;
  } else {
#pragma unroll
    for (int j = 0; j < LD; ++j)
#pragma unroll
      for (int k = 0; k < H; ++k) dw[j][k] = splat2(0.f);
  }

  int slot = 0;
  uint32_t parity = 0;
  const int64_t lead = TPR < 32 ? (int64_t)blockIdx.x * GROUPS + (threadIdx.x & ~31) / TPR : first;
  for (int64_t i = 0; lead + i < p.M; i += step) {
    const int64_t row = first + i;
    const bool valid = TPR >= 32 || row < p.M;
    const float rstd = valid ? __ldg(p.rstd + row) : 0.f;

    T ge[SLOTS];
    R he[SLOTS], de[SLOTS];
#pragma unroll
    for (int k = 0; k < EDGES; ++k) {  // ahead of the wait for the packets
      ge[k] = from_f32<T>(0.f);
      he[k] = de[k] = from_f32<R>(0.f);
      if (!valid || ec[k] < 0) continue;
      ge[k] = *gs.at(row, ec[k]);
      he[k] = *hs.at(row, ec[k]);
      if (p.r != nullptr) de[k] = *ds.at(row, ec[k]);
    }
    RawVec<T, VEC> gv[LD];
    RawVec<R, VEC> hv[LD], dv[LD];
    const unsigned char* src = slots + (size_t)slot * slot_bytes;
    if constexpr (RING) mbar_wait(&bars[group][slot], parity, &cta_abort, p.status);
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int pk = j * TPR + t;
      gv[j].zero();
      hv[j].zero();
      dv[j].zero();
      if (!valid || pk >= packets) continue;
      if constexpr (RING) {
        gv[j].load_shared(src + (size_t)pk * VEC * sizeof(T));
        hv[j].load_shared(src + t_bytes + (size_t)pk * VEC * sizeof(R));
        if (p.r != nullptr) dv[j].load_shared(src + t_bytes + r_bytes + (size_t)pk * VEC * sizeof(R));
      } else {
        gv[j] = gs.load(row, head + pk * VEC);
        hv[j] = hs.load(row, head + pk * VEC);
        if (p.r != nullptr) dv[j] = ds.load(row, head + pk * VEC);
      }
    }
    float2 s2 = splat2(0.f);
    const float2 rs2 = splat2(rstd);
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int pk = j * TPR + t;
      // With 768 threads, hence 80 registers, the test keeps these from being spilled (5000 x 12288 bf16: 87 -> 79 us).
      if ((!WREG || TPR > 512) && pk >= packets) continue;
      float2 gf[H], hf[H], wf[H];
      gv[j].unpack(gf);
      hv[j].unpack(hf);
      if constexpr (WREG) {
#pragma unroll
        for (int k = 0; k < H; ++k) wf[k] = wr[j][k];
      } else {
        weights(pk, wf);
      }
#pragma unroll
      for (int k = 0; k < H; ++k) {
        const float2 a = mul2(gf[k], mul2(hf[k], rs2));  // dy * xhat
        s2 = fma2(wf[k], a, s2);
        if constexpr (WIDE) {
          acc[(j * VEC + 2 * k) * TPR + t] += a.x;
          acc[(j * VEC + 2 * k + 1) * TPR + t] += a.y;
        } else {
          dw[j][k] = add2(dw[j][k], a);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < EDGES; ++k) {
      const float a = to_f32(ge[k]) * (to_f32(he[k]) * rstd);
      s2.x = fmaf(ew[k], a, s2.x);
      edw[k] += a;
    }
    const float c1 = row_sum<TPR, (GROUPS == 1 ? 0 : 1)>(s2.x + s2.y, scratch[group], phase, group, warp_n, lane) * inv_n;
    if constexpr (RING) {
      if (t == 0 && row + p.stages * step < p.M) fill(slot, row + p.stages * step);
      if (++slot == p.stages) {
        slot = 0;
        parity ^= 1u;
      }
    }
    // d = w * dy * rstd - h * (c1 * rstd^2) + dh
    const float2 kh = splat2(-c1 * rstd * rstd);
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int pk = j * TPR + t;
      if (!valid || pk >= packets) continue;
      float2 gf[H], hf[H], wf[H], df[H];
      gv[j].unpack(gf);
      hv[j].unpack(hf);
      dv[j].unpack(df);
      if constexpr (WREG) {
#pragma unroll
        for (int k = 0; k < H; ++k) wf[k] = wr[j][k];
      } else {
        weights(pk, wf);
      }
#pragma unroll
      for (int k = 0; k < H; ++k) df[k] = fma2(mul2(wf[k], rs2), gf[k], fma2(hf[k], kh, df[k]));
      RawVec<T, VEC> o;
      o.pack(df);
      dxs.store(row, head + pk * VEC, o);
      if constexpr (sizeof(R) != sizeof(T)) {
        RawVec<R, VEC> od;
        od.pack(df);
        drs.store(row, head + pk * VEC, od);
      }
    }
#pragma unroll
    for (int k = 0; k < EDGES; ++k) {
      if (!valid || ec[k] < 0) continue;
      const float d = fmaf(ew[k] * rstd, to_f32(ge[k]), fmaf(to_f32(he[k]), kh.x, to_f32(de[k])));
      *dxs.at(row, ec[k]) = from_f32<T>(d);
      if constexpr (sizeof(R) != sizeof(T)) *drs.at(row, ec[k]) = from_f32<R>(d);
    }
  }
  if constexpr (RING) {
    if (t == 0 && cta_abort) addnorm_drain(bars[group], p.stages, first < p.M ? (p.M - first + step - 1) / step : 0);
  }

  if (p.part == nullptr) return;
  float* out = p.part + (size_t)blockIdx.x * p.N;
  if constexpr (GROUPS > 1) {
    static_assert(GROUPS == 1 || !WIDE, "several row groups keep their sums in registers");
    if constexpr (RING) __syncthreads();  // every group has read its slots: the sums go there
    float* mine = acc + (size_t)group * p.N;
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int pk = j * TPR + t, c0 = head + pk * VEC;
      if (pk >= packets) continue;
#pragma unroll
      for (int k = 0; k < VEC; ++k) mine[c0 + k] = (k & 1) ? dw[j][k / 2].y : dw[j][k / 2].x;
    }
#pragma unroll
    for (int k = 0; k < EDGES; ++k)
      if (ec[k] >= 0) mine[ec[k]] = edw[k];
    __syncthreads();
    for (int c = threadIdx.x; c < p.N; c += GROUPS * TPR) {
      float s = 0.f;
      for (int g = 0; g < GROUPS; ++g) s += acc[(size_t)g * p.N + c];
      out[c] = s;
    }
  } else {
#pragma unroll
    for (int j = 0; j < LD; ++j) {
      const int pk = j * TPR + t, c0 = head + pk * VEC;
      if (pk >= packets) continue;
      float2 a[H];
#pragma unroll
      for (int k = 0; k < H; ++k) {
        if constexpr (WIDE) a[k] = make_float2(acc[(j * VEC + 2 * k) * TPR + t], acc[(j * VEC + 2 * k + 1) * TPR + t]);
        else a[k] = dw[j][k];
      }
      if constexpr (!OFF) {
        st_f32_pairs<H>(out + c0, a);
      } else {
#pragma unroll
        for (int k = 0; k < VEC; ++k) out[c0 + k] = (k & 1) ? a[k / 2].y : a[k / 2].x;
      }
    }
#pragma unroll
    for (int k = 0; k < EDGES; ++k)
      if (ec[k] >= 0) out[ec[k]] = edw[k];
  }
}

// dweight from the CTAs' partial rows: a CTA takes 32 columns, its warps every 32nd row each, eight loads in flight
// per thread; then a warp adds a column's 32 sums.  The order depends on the number of rows alone.
struct AddNormReduceParams {
  const float* part;
  void* dw;
  int rows, N, w_dtype;
};
static __global__ void __launch_bounds__(1024) addnorm_reduce_kernel(const AddNormReduceParams p) {
  __shared__ float tile[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int col = blockIdx.x * 32 + tx;
  grid_dependency_sync();
  trigger_dependents();
  float s = 0.f;
  if (col < p.N) {
    for (int r = ty; r < p.rows; r += 256) {
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = r + 32 * k < p.rows ? p.part[(size_t)(r + 32 * k) * p.N + col] : 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) s += v[k];
    }
  }
  tile[ty][tx] = s;
  __syncthreads();
  s = warp_sum(tile[tx][ty]);
  if (tx == 0 && blockIdx.x * 32 + ty < p.N) store_param(p.dw, p.w_dtype, blockIdx.x * 32 + ty, s);
}

// Buffers whose rows are aligned differently (views, odd strides): one CTA per row, element by element,
// the row kept in shared memory as fp32 between the two passes.  In the 8-bit form a warp takes a scale's
// columns at a time.
template <typename T, typename R, bool FP8>
__global__ void __launch_bounds__(512) addnorm_fwd_any_kernel(const AddNormParams p) {
  extern __shared__ float hs[];  // [N]
  __shared__ float scratch[2 * 16];
  __shared__ float max_scratch[16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int phase = 0;
  grid_dependency_sync();
  trigger_dependents();
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const T* xrow = static_cast<const T*>(p.x) + row * p.x_stride;
    const R* rrow = static_cast<const R*>(p.r) + row * p.r_stride;
    R* hrow = static_cast<R*>(p.h) + row * p.h_stride;
    float q = 0.f;
#pragma unroll 4
    for (int c = threadIdx.x; c < p.N; c += 512) {
      float v = to_f32(xrow[c]);
      if (p.r != nullptr) v = to_f32(from_f32<R>(v + to_f32(rrow[c])));
      if (p.h != nullptr) hrow[c] = from_f32<R>(v);
      hs[c] = v;
      q = fmaf(v, v, q);
    }
    float s[1] = {q};
    group_sum<16, 1, 0>(s, scratch, phase, 0, warp, lane);  // a barrier: the row is in shared memory after it
    const float rstd = 1.f / sqrtf(s[0] / static_cast<float>(p.N) + p.eps);
    if (threadIdx.x == 0 && p.rstd != nullptr) p.rstd[row] = rstd;
    if constexpr (!FP8) {
      T* yrow = static_cast<T*>(p.y) + row * p.y_stride;
      for (int c = threadIdx.x; c < p.N; c += 512) {
        const float w = p.w != nullptr ? load_param(p.w, p.w_dtype, c) : 1.f;
        yrow[c] = from_f32<T>(hs[c] * rstd * w);
      }
    } else {
      uint8_t* qrow = static_cast<uint8_t*>(p.y) + row * p.y_stride;
      const bool whole = p.group == 0;
      float amax = 0.f;
      for (int c = threadIdx.x; c < p.N; c += 512) {
        const float w = p.w != nullptr ? load_param(p.w, p.w_dtype, c) : 1.f;
        const float v = hs[c] * rstd * w;
        hs[c] = v;
        amax = max_abs(amax, v);
      }
      amax = warp_max_abs(amax);
      if (lane == 0) max_scratch[warp] = amax;
      __syncthreads();
      if (whole) {
        for (int k = 0; k < 16; ++k) amax = max_abs(amax, max_scratch[k]);
        const Fp8Scale sc = fp8_scale(amax, p.e8m0 != 0);
        if (threadIdx.x == 0) store_scale(p.scale, row, sc, p.e8m0 != 0);
        for (int c = threadIdx.x; c < p.N; c += 512) qrow[c] = static_cast<uint8_t>(fp8x2(fp8_quotient(hs[c], sc), 0.f));
      } else {
        for (int g = warp; g < p.groups_per_row; g += 16) {
          const int c0 = g * p.group;
          float v[4], a = 0.f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int c = c0 + k * 32 + lane;
            v[k] = (k * 32 < p.group && c < p.N) ? hs[c] : 0.f;
            a = max_abs(a, v[k]);
          }
          const Fp8Scale sc = fp8_scale(warp_max_abs(a), p.e8m0 != 0);
          if (lane == 0) store_scale(p.scale, row * p.groups_per_row + g, sc, p.e8m0 != 0);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int c = c0 + k * 32 + lane;
            if (k * 32 < p.group && c < p.N) qrow[c] = static_cast<uint8_t>(fp8x2(fp8_quotient(v[k], sc), 0.f));
          }
        }
      }
    }
    __syncthreads();  // the next row overwrites hs
  }
}

template <typename T, typename R>
__global__ void __launch_bounds__(512) addnorm_bwd_any_kernel(const AddNormParams p) {
  extern __shared__ float acc[];  // [N]: column c belongs to thread c % 512
  __shared__ float scratch[2 * 16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int phase = 0;
  grid_dependency_sync();
  trigger_dependents();
  for (int c = threadIdx.x; c < p.N; c += 512) acc[c] = 0.f;
  const float inv_n = 1.f / static_cast<float>(p.N);
  for (int64_t row = blockIdx.x; row < p.M; row += gridDim.x) {
    const T* grow = static_cast<const T*>(p.x) + row * p.x_stride;
    const R* hrow = static_cast<const R*>(p.h) + row * p.h_stride;
    const R* drow = static_cast<const R*>(p.r) + row * p.r_stride;
    T* dxrow = static_cast<T*>(p.y) + row * p.y_stride;
    R* drrow = static_cast<R*>(p.dr) + row * p.dr_stride;
    const float rs = p.rstd[row];
    float s[1] = {0.f};
#pragma unroll 4
    for (int c = threadIdx.x; c < p.N; c += 512) {
      const float w = p.w != nullptr ? load_param(p.w, p.w_dtype, c) : 1.f;
      const float a = to_f32(grow[c]) * (to_f32(hrow[c]) * rs);
      acc[c] += a;
      s[0] = fmaf(w, a, s[0]);
    }
    group_sum<16, 1, 0>(s, scratch, phase, 0, warp, lane);
    const float kh = -s[0] * inv_n * rs * rs;
#pragma unroll 4
    for (int c = threadIdx.x; c < p.N; c += 512) {
      const float w = p.w != nullptr ? load_param(p.w, p.w_dtype, c) : 1.f;
      const float dh = p.r != nullptr ? to_f32(drow[c]) : 0.f;
      const float d = fmaf(w * rs, to_f32(grow[c]), fmaf(to_f32(hrow[c]), kh, dh));
      dxrow[c] = from_f32<T>(d);
      if constexpr (sizeof(R) != sizeof(T)) drrow[c] = from_f32<R>(d);
    }
  }
  if (p.part == nullptr) return;
  for (int c = threadIdx.x; c < p.N; c += 512) p.part[(size_t)blockIdx.x * p.N + c] = acc[c];
}

// ---------------------------------------------------------------------------------------
// What the launch code needs to know of the compiled kernels, one table per (T, R).
// ---------------------------------------------------------------------------------------
struct AddNormShape {  // null: the shape is not for this
  int ld, tpr;
  const void* fwd[2];       // [rows at a common offset]
  const void* fp8[5];       // a scale per row, 32, 64, 128 columns; rows at a common offset
  const void* fp8_ring[5];
  const void* bwd[2];
  const void* bwd_ring[2];
  int capacity() const { return ld * tpr; }  // packets per row
  int threads() const { return addnorm_threads(tpr); }
  int groups() const { return threads() / tpr; }
};
struct AddNormTable {
  int size_t_, size_r;  // bytes per element
  const AddNormShape* shapes;  // ascending capacity
  int n;
  const void *fwd_any, *fp8_any, *bwd_any;
};

const AddNormTable* addnorm_table_f32();
const AddNormTable* addnorm_table_f16();
const AddNormTable* addnorm_table_bf16();
const AddNormTable* addnorm_table_f16_f32();
const AddNormTable* addnorm_table_bf16_f32();

}  // namespace b200norm
