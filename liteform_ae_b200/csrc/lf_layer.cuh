// Element types, activations and sums shared by the operators of a layer: the CSR product with bias,
// activation and residual (lf_spmm_act.cu), its gradients (lf_spmm_act_grad.cu) and the root-mean-square norm
// (lf_rms_norm.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "lf_common.cuh"

namespace lf {

constexpr int kSms = 148;   // of a B200: launches are sized by it, and workspaces, whose sizes are asked for without a device
inline bool is_wide_dtype(int32_t dt) { return dt == LF_DTYPE_F32 || dt == LF_DTYPE_BF16 || dt == LF_DTYPE_F16; }
__host__ __device__ inline int dtype_bytes(int32_t dt) { return dt == LF_DTYPE_F32 ? 4 : dt == LF_DTYPE_E4M3 ? 1 : 2; }
// what a misaligned address would fault on; NULL is aligned
inline bool aligned(const void* p, int bytes) { return (uintptr_t)p % bytes == 0; }
inline bool aligned_for(const void* p, int32_t dt) { return aligned(p, dtype_bytes(dt)); }
inline bool on_grid16(const void* p, int64_t ld, int32_t dt) {   // every row starts on a 16-byte boundary
  return (uintptr_t)p % 16 == 0 && ld * dtype_bytes(dt) % 16 == 0;
}

// `Type<LF_DTYPE_...>`: the stored type, and its way to and from float (rounded to nearest, ties to even)
template <int DT> struct Type;
template <> struct Type<LF_DTYPE_F32> {
  using T = float;
  static __device__ __forceinline__ float get(T v) { return v; }
  static __device__ __forceinline__ T put(float v) { return v; }
};
template <> struct Type<LF_DTYPE_BF16> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float get(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T put(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Type<LF_DTYPE_F16> {
  using T = __half;
  static __device__ __forceinline__ float get(T v) { return __half2float(v); }
  static __device__ __forceinline__ T put(float v) { return __float2half_rn(v); }
};
template <> struct Type<LF_DTYPE_E4M3> {   // put: values beyond 448 become 448, NaN stays NaN
  using T = __nv_fp8_storage_t;
  static __device__ __forceinline__ float get(T v) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3))); }
  static __device__ __forceinline__ T put(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
};

// `n` consecutive elements, from or to an address that is a multiple of their size together (n * bytes <= 16, or
// a multiple of 16)
template <int DT, int n>
struct Pack {
  static constexpr int kBytes = n * (int)sizeof(typename Type<DT>::T);
  static constexpr int kWord = kBytes >= 16 ? 16 : kBytes;
  union {
    typename Type<DT>::T e[n];
    uint4 q[(kBytes + 15) / 16];
    uint2 d;
    uint32_t w;
    uint16_t h;
    uint8_t b;
  };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ void fetch(const void* p) {   // read once, by the thread that may write there later: streaming
    if constexpr (kWord == 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) q[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
    } else if constexpr (kWord == 8) d = __ldcs(reinterpret_cast<const uint2*>(p));
    else if constexpr (kWord == 4) w = __ldcs(reinterpret_cast<const uint32_t*>(p));
    else if constexpr (kWord == 2) h = __ldcs(reinterpret_cast<const uint16_t*>(p));
    else b = __ldcs(reinterpret_cast<const uint8_t*>(p));
  }
  __device__ __forceinline__ void keep(void* p) const {   // what the next launch gathers stays in the L2 if it can
    if constexpr (kWord == 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = q[i];
    } else if constexpr (kWord == 8) *reinterpret_cast<uint2*>(p) = d;
    else if constexpr (kWord == 4) *reinterpret_cast<uint32_t*>(p) = w;
    else if constexpr (kWord == 2) *reinterpret_cast<uint16_t*>(p) = h;
    else *reinterpret_cast<uint8_t*>(p) = b;
  }
  __device__ __forceinline__ void store(void* p) const {   // written once, read by a later launch: streaming
    if constexpr (kWord == 16) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) __stcs(reinterpret_cast<uint4*>(p) + i, q[i]);
    } else if constexpr (kWord == 8) __stcs(reinterpret_cast<uint2*>(p), d);
    else if constexpr (kWord == 4) __stcs(reinterpret_cast<uint32_t*>(p), w);
    else if constexpr (kWord == 2) __stcs(reinterpret_cast<uint16_t*>(p), h);
    else __stcs(reinterpret_cast<uint8_t*>(p), b);
  }
  __device__ __forceinline__ float get(int i) const { return Type<DT>::get(e[i]); }
  __device__ __forceinline__ void put(const float* v) {   // two at a time where the type has such a conversion
    if constexpr (n % 2 == 0 && DT != LF_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < n; i += 2) {
        if constexpr (DT == LF_DTYPE_BF16) *reinterpret_cast<__nv_bfloat162*>(e + i) = __floats2bfloat162_rn(v[i], v[i + 1]);
        else if constexpr (DT == LF_DTYPE_F16) *reinterpret_cast<__half2*>(e + i) = __floats2half2_rn(v[i], v[i + 1]);
        else *reinterpret_cast<__nv_fp8x2_storage_t*>(e + i) = __nv_cvt_float2_to_fp8x2(make_float2(v[i], v[i + 1]), __NV_SATFINITE, __NV_E4M3);
      }
    } else {
#pragma unroll
      for (int i = 0; i < n; ++i) e[i] = Type<DT>::put(v[i]);
    }
  }
};

// one element of a type that is known at run time only (never 8 bits)
__device__ __forceinline__ float get_any(const void* p, int64_t i, int dt) {
  if (dt == LF_DTYPE_F32) return __ldg(reinterpret_cast<const float*>(p) + i);
  if (dt == LF_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(reinterpret_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void put_any(void* p, int64_t i, int dt, float v) {
  if (dt == LF_DTYPE_F32) reinterpret_cast<float*>(p)[i] = v;
  else if (dt == LF_DTYPE_BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
}

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float min_nan(float a, float b) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---- activations ------------------------------------------------------------------------------------
// 2^x (off by 2 units in the last place) and 1 / x (by 1) by the special function unit, results below the normal numbers as 0
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;
// s = 1 / (1 + exp(-u)), and *d = s (1 - s).  FULL: for results in 32 bits.  p = exp(-|u|) does not overflow, and for u < 0 both
// keep their relative accuracy as far as numbers go, about 7 units of 2^-24.  Otherwise rounding -u log2(e) adds |u| units to the
// lower tail, which 16-bit results do not show (2^20 rows of 64 in 8 bits, silu to bfloat16: 667 us, with FULL 688); where the
// exponential overflows s is 0.
template <bool FULL>
__device__ __forceinline__ float sigmoid(float u, float* d) {
  if constexpr (FULL) {
    const float p = expf(-fabsf(u)), r = rcp_approx(1.f + p), pr = p * r;
    *d = pr * r;
    return u < 0.f ? pr : r;   // a NaN stays one
  } else {
    const float s = rcp_approx(1.f + exp2_approx(-kLog2e * u));
    *d = s * (1.f - s);
    return s;
  }
}
// the tanh form of GELU is z * sigmoid(u), u = z (k0 + k0 k1 z^2), since (1 + tanh(u / 2)) / 2 = sigmoid(u)
constexpr float kGelu0 = 1.5957691216057308f, kGelu1 = 0.044715f;

// The normal distribution beyond x >= 0 is e M(x) with e = exp(-x^2 / 2) and M(x) = t P(t), t = 1 / (1 + 0.35 x): P by least squares
// with repeated weights on the relative error (Lawson) for x up to 15, where M is off by 3.2e-8; in 32 bits by 2.9e-7 with t
// rounded rightly.  e's argument adds 3 units of 2^-24 times x^2 / 2.  So the lower tail keeps its relative accuracy, which
// 1 + erf(z / sqrt 2) does not.  (2^18 rows of 256 bfloat16 gradients of gelu with erff and expf: 142 us.)
__device__ __forceinline__ float normal_tail(float x, float* e) {
  const float t = rcp_approx(fmaf(0.35f, x, 1.f));
  *e = exp2_approx(-0.5f * kLog2e * x * x);
  float p = -0.0291638002f;
  p = fmaf(t, p, 0.144060209f);
  p = fmaf(t, p, -0.255900681f);
  p = fmaf(t, p, 0.159391612f);
  p = fmaf(t, p, -0.0232629776f);
  p = fmaf(t, p, 0.105574459f);
  p = fmaf(t, p, 0.119815581f);
  p = fmaf(t, p, 0.139864326f);
  p = fmaf(t, p, 0.139621258f);
  return t * p;
}

// v[i] = act(v[i]) for n values.  The two kinds with a sigmoid share their code: z * sigmoid(z (k0 + k1 z^2)).
template <int n, bool FULL>
__device__ __forceinline__ void activate_all(float* v, int act) {
  if (act == LF_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = max_nan(v[i], 0.f);
  } else if (act == LF_ACT_SILU || act == LF_ACT_GELU_TANH) {
    const float k0 = act == LF_ACT_SILU ? 1.f : kGelu0, k1 = act == LF_ACT_SILU ? 0.f : kGelu0 * kGelu1;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      float d;
      v[i] *= sigmoid<FULL>(v[i] * fmaf(k1 * v[i], v[i], k0), &d);
    }
  } else if (act == LF_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      float e;
      const float q = normal_tail(fabsf(v[i]), &e) * e;
      v[i] *= v[i] < 0.f ? q : 1.f - q;   // a NaN stays one
    }
  }
}

// v[i] = act'(v[i]).  Beyond +-120 the slopes of smooth ones are 0 or 1 to the last bit; so far the formulas stay clear of 0 *
// infinity.
template <int n, bool FULL>
__device__ __forceinline__ void slopes(float* v, int act) {
  if (act == LF_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < n; ++i) v[i] = v[i] <= 0.f ? 0.f : 1.f;   // a NaN lets the gradient through
  } else if (act == LF_ACT_SILU || act == LF_ACT_GELU_TANH) {
    const float k0 = act == LF_ACT_SILU ? 1.f : kGelu0, k1 = act == LF_ACT_SILU ? 0.f : kGelu0 * kGelu1;
#pragma unroll
    for (int i = 0; i < n; ++i) {   // u = z (k0 + k1 z^2): s + z s (1 - s) u'
      float d;
      const float z = min_nan(max_nan(v[i], -120.f), 120.f), zz = k1 * z * z, s = sigmoid<FULL>(z * (k0 + zz), &d);
      v[i] = fmaf(z * d, fmaf(3.f, zz, k0), s);
    }
  } else if (act == LF_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < n; ++i) {
      float e;   // the slope beyond x is e (M(x) - x / sqrt(2 pi)), and 1 less that of -x for x
      const float x = min_nan(fabsf(v[i]), 120.f), m = normal_tail(x, &e), w = fmaf(-0.3989422804014327f, x, m) * e;
      v[i] = v[i] < 0.f ? w : 1.f - w;
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {   // the same sum in every lane
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace lf
