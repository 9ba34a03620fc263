// CSR product with the end of a layer in its epilogue: Y = act(A * B + bias) + residual.
#include "lf_layer.cuh"

namespace lf {
namespace {

struct ActArgs {
  const int64_t* indptr;
  const int32_t* indices;
  const float* data;       // or NULL: all ones
  const int32_t* order;    // data of entry e is data[order[e]], or NULL: data[e]
  int64_t row_begin, rows, nnz;
  const void* B;
  const float* b_scale;    // or NULL
  int64_t ldb;
  const void* bias;
  const void* residual;
  void* preact;
  void* C;
  int64_t ld_res, ld_pre, ldc;
  int N, bias_dtype, res_dtype, c_dtype, act;
};

// A warp per row, 128 features at a time.
template <int DT>
__global__ void __launch_bounds__(256)
spmm_csr_act_rows_kernel(ActArgs a) {
  using T = Type<DT>;
  const int lane = threadIdx.x & 31, f0 = blockIdx.y * 128 + lane;
  const int64_t base = a.indptr[a.row_begin];
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < a.rows; row += (int64_t)gridDim.x * 8) {
    const int64_t s0 = a.indptr[a.row_begin + row], s1 = min(a.indptr[a.row_begin + row + 1], base + a.nnz);
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t e = s0; e < s1; ++e) {
      const int32_t col = a.indices[e];
      float v = a.data ? a.data[a.order ? a.order[e] : e] : 1.f;
      if (v == 0.f) continue;
      if (a.b_scale) v *= a.b_scale[col];
      const auto* b = reinterpret_cast<const typename T::T*>(a.B) + (int64_t)col * a.ldb;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (f0 + 32 * i < a.N) acc[i] = fmaf(v, T::get(b[f0 + 32 * i]), acc[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int f = f0 + 32 * i;
      if (f >= a.N) continue;
      const float z = a.bias ? acc[i] + get_any(a.bias, f, a.bias_dtype) : acc[i];
      if (a.preact) put_any(a.preact, row * a.ld_pre + f, a.c_dtype, z);
      float y = activate(z, a.act);
      if (a.residual) y += get_any(a.residual, row * a.ld_res + f, a.res_dtype);
      put_any(a.C, row * a.ldc + f, a.c_dtype, y);
    }
  }
}

}  // namespace
}  // namespace lf

using namespace lf;

extern "C" {

size_t lf_spmm_csr_act_workspace_bytes(int64_t nnz, int32_t N, int32_t b_dtype) { return 0; }

int lf_spmm_csr_act(const int64_t* indptr, const int32_t* indices, const float* data, const int32_t* order,
                    int64_t row_begin, int64_t row_end, int64_t nnz, const void* B, int32_t b_dtype, int64_t ldb,
                    const float* b_scale, void* C, int32_t c_dtype, int64_t ldc, int32_t N, const lf_epilogue* epilogue,
                    void* workspace, size_t workspace_bytes, void* stream) {
  LF_REQUIRE(N >= 1 && ldb >= N && ldc >= N && ldb < (1ll << 30) && ldc < (1ll << 30), "bad sizes");
  LF_REQUIRE(0 <= row_begin && row_begin <= row_end, "bad row range");
  LF_REQUIRE(row_end - row_begin < (1ll << 31) - 64 && nnz >= 0, "bad number of rows or entries");
  LF_REQUIRE(b_dtype == LF_DTYPE_E4M3 || is_wide_dtype(b_dtype), "unknown type of B");
  LF_REQUIRE(b_dtype != LF_DTYPE_E4M3 || b_scale, "8-bit rows need their scales");
  LF_REQUIRE(is_wide_dtype(c_dtype), "C must be float32, bfloat16 or float16");
  const lf_epilogue none = {};
  const lf_epilogue& ep = epilogue ? *epilogue : none;
  LF_REQUIRE(ep.activation >= LF_ACT_NONE && ep.activation <= LF_ACT_GELU_TANH, "unknown activation");
  LF_REQUIRE(!ep.bias || is_wide_dtype(ep.bias_dtype), "the bias must be float32, bfloat16 or float16");
  LF_REQUIRE(!ep.residual || (is_wide_dtype(ep.residual_dtype) && ep.ld_residual >= N), "bad residual");
  LF_REQUIRE(!ep.preact || ep.ld_preact >= N, "bad leading dimension of preact");
  if (row_begin == row_end) return LF_OK;
  LF_REQUIRE(indptr && C, "null pointer argument");
  LF_REQUIRE(nnz == 0 || (indices && B), "indices or B missing");
  LF_REQUIRE(!order || (data && nnz < (1ll << 31)), "order goes with data, for fewer than 2^31 entries");
  const ActArgs a{indptr, indices, data, order, row_begin, row_end - row_begin, nnz, B, b_scale, ldb, ep.bias, ep.residual,
                  ep.preact, C, ep.ld_residual, ep.ld_preact, ldc, N, ep.bias_dtype, ep.residual_dtype, c_dtype, ep.activation};
  cudaStream_t st = (cudaStream_t)stream;
  const int64_t blocks = ceil_div64(a.rows, 8);
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20), (unsigned)((N + 127) / 128));
  if (b_dtype == LF_DTYPE_F32) spmm_csr_act_rows_kernel<LF_DTYPE_F32><<<grid, 256, 0, st>>>(a);
  else if (b_dtype == LF_DTYPE_BF16) spmm_csr_act_rows_kernel<LF_DTYPE_BF16><<<grid, 256, 0, st>>>(a);
  else if (b_dtype == LF_DTYPE_F16) spmm_csr_act_rows_kernel<LF_DTYPE_F16><<<grid, 256, 0, st>>>(a);
  else spmm_csr_act_rows_kernel<LF_DTYPE_E4M3><<<grid, 256, 0, st>>>(a);
  LF_CUDA_CHECK(cudaGetLastError());
  return LF_OK;
}

}  // extern "C"
