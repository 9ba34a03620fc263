// Gradients of Y = act(A * B + bias) + residual besides that of B (which is the product with A transposed):
// dZ = dY * act'(Z), its sum over the rows for the bias, and the gradient of A's values.
#include "lf_layer.cuh"

namespace lf {

cudaError_t launch_column_sum(const float* partial, int parts, int N, float* out, cudaStream_t st);   // lf_rms_norm.cu

namespace {

struct ActGradArgs {
  const void* dy;
  const void* z;       // or NULL: no activation
  void* dz;            // or NULL
  float* partial;      // [parts][N], or NULL
  int64_t rows, ld_dy, ld_z, ld_dz;
  int N, act, rows_per_part;
};

template <int DT>
__global__ void __launch_bounds__(256)
act_grad_kernel(ActGradArgs a) {
  using T = Type<DT>;
  const int f = blockIdx.y * 256 + threadIdx.x;
  if (f >= a.N) return;
  const int64_t r0 = (int64_t)blockIdx.x * a.rows_per_part, r1 = min(r0 + a.rows_per_part, a.rows);
  float s = 0.f;
  for (int64_t r = r0; r < r1; ++r) {
    float d = T::get(reinterpret_cast<const typename T::T*>(a.dy)[r * a.ld_dy + f]);
    if (a.z) d *= activate_slope(T::get(reinterpret_cast<const typename T::T*>(a.z)[r * a.ld_z + f]), a.act);
    if (a.dz) reinterpret_cast<typename T::T*>(a.dz)[r * a.ld_dz + f] = T::put(d);
    s += d;
  }
  if (a.partial) a.partial[(int64_t)blockIdx.x * a.N + f] = s;
}

struct ValueGradArgs {
  const int64_t* indptr;
  const int32_t* indices;
  int64_t row_begin, rows, nnz;
  const void* dy;
  const void* z;
  const void* B;
  float* dvalues;
  int64_t ld_dy, ld_z, ldb;
  int N, act, dy_dtype;
};

// A warp per row.
template <int DT>
__global__ void __launch_bounds__(256)
value_grad_rows_kernel(ValueGradArgs a) {
  using T = Type<DT>;
  const int lane = threadIdx.x & 31;
  const int64_t base = a.indptr[a.row_begin];
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < a.rows; row += (int64_t)gridDim.x * 8) {
    const int64_t s0 = a.indptr[a.row_begin + row], s1 = min(a.indptr[a.row_begin + row + 1], base + a.nnz);
    for (int64_t e = s0; e < s1; ++e) {
      const auto* b = reinterpret_cast<const typename T::T*>(a.B) + (int64_t)a.indices[e] * a.ldb;
      float s = 0.f;
      for (int f = lane; f < a.N; f += 32) {
        float d = get_any(a.dy, row * a.ld_dy + f, a.dy_dtype);
        if (a.z) d *= activate_slope(get_any(a.z, row * a.ld_z + f, a.dy_dtype), a.act);
        s = fmaf(d, T::get(b[f]), s);
      }
      s = warp_sum(s);
      if (lane == 0) a.dvalues[e - base] = s;
    }
  }
}

constexpr int kParts = 1184;   // 148 SMs x 8

int rows_per_part(int64_t rows) { return (int)ceil_div64(rows, kParts); }

}  // namespace
}  // namespace lf

using namespace lf;

extern "C" {

size_t lf_act_backward_workspace_bytes(int64_t rows, int32_t N) {
  if (rows < 1 || N < 1) return 0;
  return (size_t)ceil_div64(rows, rows_per_part(rows)) * (size_t)N * sizeof(float);
}

int lf_act_backward(const void* dy, int64_t ld_dy, const void* preact, int64_t ld_preact, int32_t dtype,
                    int32_t activation, void* dz, int64_t ld_dz, float* dbias, int64_t rows, int32_t N,
                    void* workspace, size_t workspace_bytes, void* stream) {
  LF_REQUIRE(rows >= 0 && rows < (1ll << 31) - 64 && N >= 1, "bad sizes");
  LF_REQUIRE(is_wide_dtype(dtype), "the type must be float32, bfloat16 or float16");
  LF_REQUIRE(activation >= LF_ACT_NONE && activation <= LF_ACT_GELU_TANH, "unknown activation");
  LF_REQUIRE(dz || dbias, "nothing to compute");
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    if (dbias) LF_CUDA_CHECK(cudaMemsetAsync(dbias, 0, (size_t)N * sizeof(float), st));
    return LF_OK;
  }
  LF_REQUIRE(dy && (preact || activation == LF_ACT_NONE), "null pointer argument");
  LF_REQUIRE(ld_dy >= N && (activation == LF_ACT_NONE || ld_preact >= N) && (!dz || ld_dz >= N), "bad leading dimension");
  if (dbias && (!workspace || workspace_bytes < lf_act_backward_workspace_bytes(rows, N)))
    return fail(LF_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace_bytes,
                lf_act_backward_workspace_bytes(rows, N));
  const ActGradArgs a{dy, activation == LF_ACT_NONE ? nullptr : preact, dz, dbias ? (float*)workspace : nullptr,
                      rows, ld_dy, ld_preact, ld_dz, N, activation, rows_per_part(rows)};
  const int parts = (int)ceil_div64(rows, a.rows_per_part);
  const dim3 grid((unsigned)parts, (unsigned)((N + 255) / 256));
  if (dtype == LF_DTYPE_F32) act_grad_kernel<LF_DTYPE_F32><<<grid, 256, 0, st>>>(a);
  else if (dtype == LF_DTYPE_BF16) act_grad_kernel<LF_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
  else act_grad_kernel<LF_DTYPE_F16><<<grid, 256, 0, st>>>(a);
  LF_CUDA_CHECK(cudaGetLastError());
  if (dbias) LF_CUDA_CHECK(launch_column_sum(a.partial, parts, N, dbias, st));
  return LF_OK;
}

int lf_spmm_csr_grad_values(const int64_t* indptr, const int32_t* indices, int64_t row_begin, int64_t row_end,
                            int64_t nnz, const void* dy, int64_t ld_dy, const void* preact, int64_t ld_preact,
                            int32_t dy_dtype, int32_t activation, const void* B, int32_t b_dtype, int64_t ldb,
                            int32_t N, float* dvalues, void* stream) {
  LF_REQUIRE(N >= 1 && ldb >= N && ldb < (1ll << 30) && ld_dy >= N && ld_dy < (1ll << 30), "bad sizes");
  LF_REQUIRE(0 <= row_begin && row_begin <= row_end && row_end - row_begin < (1ll << 31) - 64 && nnz >= 0, "bad row range");
  LF_REQUIRE(is_wide_dtype(dy_dtype) && is_wide_dtype(b_dtype), "the types must be float32, bfloat16 or float16");
  LF_REQUIRE(activation >= LF_ACT_NONE && activation <= LF_ACT_GELU_TANH, "unknown activation");
  if (row_begin == row_end || nnz == 0) return LF_OK;
  LF_REQUIRE(indptr && indices && dy && B && dvalues, "null pointer argument");
  LF_REQUIRE(activation == LF_ACT_NONE || (preact && ld_preact >= N && ld_preact < (1ll << 30)), "preact missing");
  const ValueGradArgs a{indptr, indices, row_begin, row_end - row_begin, nnz, dy, activation == LF_ACT_NONE ? nullptr : preact,
                        B, dvalues, ld_dy, ld_preact, ldb, N, activation, dy_dtype};
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t blocks = ceil_div64(a.rows, 8);
  const unsigned grid = (unsigned)(blocks < (1 << 20) ? blocks : 1 << 20);
  if (b_dtype == LF_DTYPE_F32) value_grad_rows_kernel<LF_DTYPE_F32><<<grid, 256, 0, st>>>(a);
  else if (b_dtype == LF_DTYPE_BF16) value_grad_rows_kernel<LF_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
  else value_grad_rows_kernel<LF_DTYPE_F16><<<grid, 256, 0, st>>>(a);
  LF_CUDA_CHECK(cudaGetLastError());
  return LF_OK;
}

}  // extern "C"
