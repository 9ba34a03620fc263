// Root-mean-square norm of the rows of a feature matrix, the residual's addition before it, and its gradients.
#include "lf_layer.cuh"

namespace lf {
namespace {

struct NormArgs {
  const void* x;
  const void* res;     // or NULL
  const void* weight;
  void* sum;           // x + res, or NULL where there is no residual
  void* y;
  float* scale;        // e4m3 only
  float* rstd;         // or NULL
  int64_t rows, ld_x, ld_res, ld_sum, ld_y;
  int N, weight_dtype, y_dtype;
  float eps;
};

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// value and sum over a block of 256 threads; every thread gets it
__device__ __forceinline__ float block_sum(float v, float* smem) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) v += smem[i];
  return v;
}
__device__ __forceinline__ float block_max(float v, float* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = smem[0];
  for (int i = 1; i < (int)blockDim.x / 32; ++i) v = max_nan(v, smem[i]);
  return v;
}

// what a row is multiplied with before it is rounded to e4m3; rows whose largest magnitude is below
// 448 * 2^-126 count as zero
__device__ __forceinline__ float e4m3_scale(float amax, float* inverse) {
  const float scale = amax * (1.f / 448.f);
  const bool zero = scale < 1.17549435e-38f;
  *inverse = zero ? 0.f : 1.f / scale;
  return zero ? 0.f : scale;
}

// One block per row, element by element: any size, stride and alignment.
template <int DT>
__global__ void __launch_bounds__(256)
rms_norm_rows_kernel(NormArgs a) {
  using T = Type<DT>;
  __shared__ float smem[8];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const auto* x = reinterpret_cast<const typename T::T*>(a.x) + row * a.ld_x;
    const auto* res = reinterpret_cast<const typename T::T*>(a.res) + row * a.ld_res;
    auto* sum = reinterpret_cast<typename T::T*>(a.sum) + row * a.ld_sum;
    float ss = 0.f;
    for (int f = threadIdx.x; f < a.N; f += 256) {
      float v = T::get(x[f]);
      if (a.res) {
        const auto h = T::put(v + T::get(res[f]));
        sum[f] = h;
        v = T::get(h);
      }
      ss = fmaf(v, v, ss);
    }
    const float rstd = rsqrtf(block_sum(ss, smem) / (float)a.N + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
    const auto* h = a.res ? sum : x;   // a thread reads what it wrote itself
    float inverse = 1.f;
    if (a.y_dtype == LF_DTYPE_E4M3) {
      float amax = 0.f;
      for (int f = threadIdx.x; f < a.N; f += 256)
        amax = max_nan(amax, fabsf(T::get(h[f]) * rstd * get_any(a.weight, f, a.weight_dtype)));
      const float scale = e4m3_scale(block_max(amax, smem), &inverse);
      if (threadIdx.x == 0) a.scale[row] = scale;
    }
    for (int f = threadIdx.x; f < a.N; f += 256) {
      const float y = T::get(h[f]) * rstd * get_any(a.weight, f, a.weight_dtype);
      if (a.y_dtype == LF_DTYPE_E4M3)
        reinterpret_cast<__nv_fp8_storage_t*>(a.y)[row * a.ld_y + f] = Type<LF_DTYPE_E4M3>::put(y * inverse);
      else
        put_any(a.y, row * a.ld_y + f, a.y_dtype, y);
    }
  }
}

struct NormGradArgs {
  const void* dy;
  const void* h;
  const void* weight;
  const float* rstd;
  const void* dsum;    // gradient that reaches h by other ways, or NULL
  void* dx;
  float* partial;      // [blocks][N]
  int64_t rows, ld_dy, ld_h, ld_dsum, ld_dx;
  int N, weight_dtype;
};

template <int DT>
__global__ void __launch_bounds__(256)
rms_norm_grad_rows_kernel(NormGradArgs a) {
  using T = Type<DT>;
  __shared__ float smem[8];
  float* part = a.partial + (int64_t)blockIdx.x * a.N;
  for (int f = threadIdx.x; f < a.N; f += 256) part[f] = 0.f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const auto* dy = reinterpret_cast<const typename T::T*>(a.dy) + row * a.ld_dy;
    const auto* h = reinterpret_cast<const typename T::T*>(a.h) + row * a.ld_h;
    const auto* ds = reinterpret_cast<const typename T::T*>(a.dsum) + row * a.ld_dsum;
    auto* dx = reinterpret_cast<typename T::T*>(a.dx) + row * a.ld_dx;
    const float rstd = a.rstd[row];
    float dot = 0.f;
    for (int f = threadIdx.x; f < a.N; f += 256)
      dot = fmaf(T::get(dy[f]) * get_any(a.weight, f, a.weight_dtype), T::get(h[f]) * rstd, dot);
    const float c = block_sum(dot, smem) / (float)a.N;
    for (int f = threadIdx.x; f < a.N; f += 256) {
      const float n = T::get(h[f]) * rstd, d = T::get(dy[f]);
      float g = rstd * (d * get_any(a.weight, f, a.weight_dtype) - n * c);
      if (a.dsum) g += T::get(ds[f]);
      dx[f] = T::put(g);
      part[f] = fmaf(d, n, part[f]);
    }
  }
}

// out[f] = sum over `parts` rows of partial, in order
__global__ void __launch_bounds__(256)
column_sum_kernel(const float* __restrict__ partial, int parts, int N, float* __restrict__ out) {
  __shared__ float smem[8][33];
  const int f = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  float s = 0.f;
  if (f < N)
    for (int p = w; p < parts; p += 8) s += partial[(int64_t)p * N + f];
  smem[w][threadIdx.x & 31] = s;
  __syncthreads();
  if (w == 0 && f < N) {
    for (int i = 1; i < 8; ++i) s += smem[i][threadIdx.x];
    out[f] = s;
  }
}

constexpr int kNormGradBlocks = 592;   // 148 SMs x 4

}  // namespace

cudaError_t launch_column_sum(const float* partial, int parts, int N, float* out, cudaStream_t st) {
  column_sum_kernel<<<(N + 31) / 32, 256, 0, st>>>(partial, parts, N, out);
  return cudaGetLastError();
}

}  // namespace lf

using namespace lf;

extern "C" {

int lf_rms_norm(const void* x, int32_t dtype, int64_t ld_x, const void* residual, int64_t ld_residual, void* sum,
                int64_t ld_sum, const void* weight, int32_t weight_dtype, float eps, void* y, int32_t y_dtype,
                int64_t ld_y, float* scale, float* rstd, int64_t rows, int32_t N, void* stream) {
  LF_REQUIRE(rows >= 0 && N >= 1 && ld_x >= N && ld_y >= N, "bad sizes");
  LF_REQUIRE(is_wide_dtype(dtype) && is_wide_dtype(weight_dtype), "x and weight must be float32, bfloat16 or float16");
  LF_REQUIRE(y_dtype == LF_DTYPE_E4M3 || is_wide_dtype(y_dtype), "unknown type of y");
  LF_REQUIRE(eps >= 0.f, "eps must not be negative");
  if (rows == 0) return LF_OK;
  LF_REQUIRE(x && weight && y, "null pointer argument");
  LF_REQUIRE(!residual || (sum && ld_residual >= N && ld_sum >= N), "a residual needs a place for the sum");
  LF_REQUIRE(y_dtype != LF_DTYPE_E4M3 || scale, "8-bit rows need a place for their scales");
  const NormArgs a{x, residual, weight, sum, y, scale, rstd, rows, ld_x, ld_residual, ld_sum, ld_y, N, weight_dtype, y_dtype, eps};
  cudaStream_t st = (cudaStream_t)stream;
  const unsigned grid = (unsigned)(rows < (1 << 20) ? rows : 1 << 20);
  if (dtype == LF_DTYPE_F32) rms_norm_rows_kernel<LF_DTYPE_F32><<<grid, 256, 0, st>>>(a);
  else if (dtype == LF_DTYPE_BF16) rms_norm_rows_kernel<LF_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
  else rms_norm_rows_kernel<LF_DTYPE_F16><<<grid, 256, 0, st>>>(a);
  LF_CUDA_CHECK(cudaGetLastError());
  return LF_OK;
}

size_t lf_rms_norm_backward_workspace_bytes(int64_t rows, int32_t N) {
  if (rows < 1 || N < 1) return 0;
  return (size_t)(rows < kNormGradBlocks ? rows : kNormGradBlocks) * (size_t)N * sizeof(float);
}

int lf_rms_norm_backward(const void* dy, int64_t ld_dy, const void* h, int64_t ld_h, int32_t dtype, const void* weight,
                         int32_t weight_dtype, const float* rstd, const void* dsum, int64_t ld_dsum, void* dx,
                         int64_t ld_dx, float* dweight, int64_t rows, int32_t N, void* workspace,
                         size_t workspace_bytes, void* stream) {
  LF_REQUIRE(rows >= 0 && N >= 1, "bad sizes");
  LF_REQUIRE(is_wide_dtype(dtype) && is_wide_dtype(weight_dtype), "the types must be float32, bfloat16 or float16");
  LF_REQUIRE(dweight, "null pointer argument");
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    LF_CUDA_CHECK(cudaMemsetAsync(dweight, 0, (size_t)N * sizeof(float), st));
    return LF_OK;
  }
  LF_REQUIRE(dy && h && weight && rstd && dx, "null pointer argument");
  LF_REQUIRE(ld_dy >= N && ld_h >= N && ld_dx >= N && (!dsum || ld_dsum >= N), "bad leading dimension");
  if (workspace_bytes < lf_rms_norm_backward_workspace_bytes(rows, N) || !workspace)
    return fail(LF_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace_bytes,
                lf_rms_norm_backward_workspace_bytes(rows, N));
  const NormGradArgs a{dy, h, weight, rstd, dsum, dx, (float*)workspace, rows, ld_dy, ld_h, ld_dsum, ld_dx, N, weight_dtype};
  const unsigned grid = (unsigned)(rows < kNormGradBlocks ? rows : kNormGradBlocks);
  if (dtype == LF_DTYPE_F32) rms_norm_grad_rows_kernel<LF_DTYPE_F32><<<grid, 256, 0, st>>>(a);
  else if (dtype == LF_DTYPE_BF16) rms_norm_grad_rows_kernel<LF_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
  else rms_norm_grad_rows_kernel<LF_DTYPE_F16><<<grid, 256, 0, st>>>(a);
  LF_CUDA_CHECK(cudaGetLastError());
  LF_CUDA_CHECK(launch_column_sum(a.partial, (int)grid, N, dweight, st));
  return LF_OK;
}

}  // extern "C"
