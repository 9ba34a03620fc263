// Gradients of Y = act(A * B + bias) + residual besides that of B (which is the product with A transposed):
// dZ = dY * act'(Z), its sum over the rows for the bias, and the gradient of A's values.
#include <type_traits>

#include "lf_layer_rows.cuh"

namespace lf {

cudaError_t launch_column_sum(const float* partial, int parts, int N, float* out, cudaStream_t st);   // lf_rms_norm.cu

namespace {

// ---- dZ and the bias --------------------------------------------------------------------------------
struct ActGradArgs {
  const void* dy;
  const void* z;       // or NULL: no activation
  void* dz;            // or NULL
  float* partial;      // [parts][N], or NULL
  int64_t rows, ld_dy, ld_z, ld_dz;
  int N, act;
  int per_row;         // threads per row, a power of two
};

// A block's threads are 256 / per_row rows side by side, VEC features each; a thread keeps its features while it walks down
// the rows, so that the bias's sum stays in registers.  The inputs are read once and dZ is written once (61 us for 2^18 rows
// of 256 bfloat16).  Under the profiler relu takes 79 us, waiting for loads with half of an SM's warps, and gelu 99, issuing in
// 67 % of the cycles.  48 registers leave five blocks an SM, and the launch has six for each: the last one runs alone.
template <int DT, int OUT, int VEC>   // of dy and z, of dz
__global__ void __launch_bounds__(256)
act_grad_kernel(ActGradArgs a) {
  using E = typename Type<DT>::T;
  using O = typename Type<OUT>::T;
  __shared__ float sums[256 * VEC];
  const int t = threadIdx.x % a.per_row, r = threadIdx.x / a.per_row, side = 256 / a.per_row;
  const int f = (blockIdx.y * a.per_row + t) * VEC;
  float s[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) s[i] = 0.f;
  if (f < a.N) {
#pragma unroll 2
    for (int64_t row = (int64_t)blockIdx.x * side + r; row < a.rows; row += (int64_t)gridDim.x * side) {
      Pack<DT, VEC> d, z;
      d.fetch(reinterpret_cast<const E*>(a.dy) + row * a.ld_dy + f);
      if (a.z) z.fetch(reinterpret_cast<const E*>(a.z) + row * a.ld_z + f);
      float v[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = a.z ? z.get(i) : 0.f;
      if (a.z) slopes<VEC, DT == LF_DTYPE_F32>(v, a.act);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        v[i] = a.z ? d.get(i) * v[i] : d.get(i);
        s[i] += v[i];
      }
      if (a.dz) {
        Pack<OUT, VEC> o;
        o.put(v);
        o.keep(reinterpret_cast<O*>(a.dz) + row * a.ld_dz + f);   // gathered next
      }
    }
  }
  if (!a.partial) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i) sums[threadIdx.x * VEC + i] = s[i];
  __syncthreads();
  const int width = a.per_row * VEC;
  for (int i = threadIdx.x; i < width; i += 256) {
    float v = sums[i];
    for (int k = 1; k < side; ++k) v += sums[k * width + i];
    if (blockIdx.y * width + i < a.N) a.partial[(int64_t)blockIdx.x * a.N + blockIdx.y * width + i] = v;
  }
}

constexpr int kMostParts = kSms * 6;

// ---- gradient of the values -------------------------------------------------------------------------
struct ValueGradArgs {
  const int64_t* indptr;   // of row_begin
  const int32_t* indices;
  int64_t nnz;
  const void* dy;
  const void* z;           // or NULL: no activation
  const void* B;
  float* dvalues;          // first of the row range's entries
  uint32_t pitch_dy, pitch_z, pitch_b;
  int rows, N, dy_dtype, act, lg, slack, f0;
  bool vec;
};

// The group keeps its row of dZ in registers (computed there, not rounded) and multiplies the rows of B that come through the
// ring with it; four dot products at a time are summed up over the lanes, each lane ending with one of them.  A row wider
// than a walk takes several launches, which add to what the ones before wrote.  As in the product, the rows of B and the
// instructions on them bound it (2^18 power-law rows, 3.1 M entries, 256 bfloat16 features, gelu: 302 us, instructions in 71 % of the
// cycles).
// VIO: rows of dy and z have B's type and are known to be on the grid.
template <int DT, int G, int CH, bool VIO>
struct GradWork {
  using S = Share<DT, G, CH>;
  static constexpr bool kPlaces = true;
  static constexpr int kVec = S::kShifted ? 1 : S::VEC, kApart = S::kShifted ? G : G * S::VEC;
  const ValueGradArgs& a;
  int f0, nf, f, left, gl;   // the walk's features; the lane's first, and those from there on
  bool ragged, vec;        // the row's last piece of 16 bytes is not full; rows of dy and z are on the 16-byte grid
  int stop, used;
  int64_t at;
  uint64_t dz[S::kPairs];
  float dot[kAtOnce];

  __device__ __forceinline__ void coming(int row) const {
    prefetch(a.dy, row, a.pitch_dy);
    if (a.z) prefetch(a.z, row, a.pitch_z);
  }
  __device__ __forceinline__ void prefetch(const void* base, int row, uint32_t pitch) const {
    const int bytes = dtype_bytes(a.dy_dtype);
    const char* p = reinterpret_cast<const char*>(row_of_b(base, (uint32_t)row, pitch)) + f0 * bytes;
    for (int i = 0; i < nf * bytes; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + i));
  }
  // VIO: the group's next row is on its way while the steps of this one run (the case above took 455 us with one row of dy
  // and one of z loaded after the other when they were needed, 341 with both at once then).
  uint32_t wd[S::kFloats], wz[S::kFloats];
  int held = -1;
  __device__ __forceinline__ void fetch(int row) {
    const int64_t at = f * dtype_bytes(DT);
    load_blocks<S::kPieces, S::VEC>(reinterpret_cast<const char*>(row_of_b(a.dy, (uint32_t)row, a.pitch_dy)) + at, DT, kApart, left, wd);
    if (a.z) load_blocks<S::kPieces, S::VEC>(reinterpret_cast<const char*>(row_of_b(a.z, (uint32_t)row, a.pitch_z)) + at, DT, kApart, left, wz);
    held = row;
  }
  __device__ __forceinline__ void ahead(int row) {
    if constexpr (VIO) {
      if (row >= 0) fetch(row);
    }
  }
  // the lane's features of rows of dy and z, as floats; what lies behind the rows' end is anything
  __device__ __forceinline__ void load(int row, float* d, float* z) {
    if constexpr (VIO) {
      if (held != row) fetch(row);
      use_blocks<S::kPieces, S::VEC>(wd, DT, d, [](float, float y) { return y; });
      if (a.z) use_blocks<S::kPieces, S::VEC>(wz, DT, z, [](float, float y) { return y; });
    } else {
      load_any(a.dy, row, a.pitch_dy, d);
      if (a.z) load_any(a.z, row, a.pitch_z, z);
    }
  }
  __device__ __forceinline__ void load_any(const void* base, int row, uint32_t pitch, float* v) const {
    const char* p = reinterpret_cast<const char*>(row_of_b(base, (uint32_t)row, pitch)) + f * dtype_bytes(a.dy_dtype);
    if (vec) {
      __align__(16) uint32_t w[S::kFloats];
      if constexpr (!S::kShifted) {
        load_blocks<S::kPieces, S::VEC>(p, a.dy_dtype, kApart, left, w);
        use_blocks<S::kPieces, S::VEC>(w, a.dy_dtype, v, [](float, float y) { return y; });
      }
      return;
    }
    if (a.dy_dtype == LF_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < S::kFloats; ++i) {
        const int k = i / kVec * kApart + i % kVec;
        v[i] = k < left ? __ldg(reinterpret_cast<const float*>(p) + k) : 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < S::kFloats; ++i) {
        const int k = i / kVec * kApart + i % kVec;
        const uint32_t h = k < left ? __ldg(reinterpret_cast<const uint16_t*>(p) + k) : 0u;
        v[i] = a.dy_dtype == LF_DTYPE_BF16 ? __uint_as_float(h << 16) : __half2float(__ushort_as_half((unsigned short)h));
      }
    }
  }
  __device__ __forceinline__ void begin(int row, bool, int, int64_t at_, int end_) {
    at = at_;
    stop = end_;
    used = 0;
    float d[S::kFloats];
    if (row >= 0) {
      float z[S::kFloats];
      load(row, d, z);
      if (a.z) {
        slopes<S::kFloats, !VIO || DT == LF_DTYPE_F32>(z, a.act);
#pragma unroll
        for (int i = 0; i < S::kFloats; ++i) d[i] *= z[i];
      }
#pragma unroll
      for (int i = 0; i < S::kFloats; ++i)
        if (i / kVec * kApart + i % kVec >= left) d[i] = 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < S::kFloats; ++i) d[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < S::kPairs; ++i) dz[i] = as_pair(__float_as_uint(d[2 * i]), __float_as_uint(d[2 * i + 1]));
  }
  __device__ __forceinline__ void step(float, const unsigned char* x) {
    uint64_t y[S::kPairs], s = 0;
    S::floats(x, gl, y);
    // What lies behind the row's end may be anything, and a 0 in dz does not make up for it: a last piece that is not full is
    // cleared here, and pieces that no lane copies hold the zeros the kernel began with.
    if (!VIO && ragged) {
#pragma unroll
      for (int i = 0; i < S::kPairs; ++i) {
        const int k = 2 * i / kVec * kApart + 2 * i % kVec, k1 = (2 * i + 1) / kVec * kApart + (2 * i + 1) % kVec;
        const float2 p = as_floats(y[i]);
        y[i] = as_pair(k < left ? __float_as_uint(p.x) : 0u, k1 < left ? __float_as_uint(p.y) : 0u);
      }
    }
    uint64_t t = 0;   // two chains
#pragma unroll
    for (int i = 0; i < S::kPairs; i += 2) {
      s = fma_pair(dz[i], y[i], s);
      t = fma_pair(dz[i + 1], y[i + 1], t);
    }
    s = add_pair(s, t);
    dot[used++ % kAtOnce] = as_floats(s).x + as_floats(s).y;
  }
  __device__ __forceinline__ void steps_done(int place, bool in) {
    used = 0;
    // lane gl ends with the dot product of place + (gl & 3)
    const bool up = gl & 2, odd = gl & 1;
    float k0 = up ? dot[2] : dot[0], k1 = up ? dot[3] : dot[1];
    k0 += __shfl_xor_sync(kAllLanes, up ? dot[0] : dot[2], 2);
    k1 += __shfl_xor_sync(kAllLanes, up ? dot[1] : dot[3], 2);
    float s = odd ? k1 : k0;
    s += __shfl_xor_sync(kAllLanes, odd ? k0 : k1, 1);
#pragma unroll
    for (int o = 4; o < G; o <<= 1) s += __shfl_xor_sync(kAllLanes, s, o);
    if (in && gl < 4 && place + gl < stop) {
      float* p = a.dvalues + at + place + gl;
      *p = a.f0 > 0 ? *p + s : s;
    }
  }
  __device__ __forceinline__ void end(int, bool, int) const {}
};

template <int DT, int G, int CH, bool VIO>
__global__ void __launch_bounds__(kWalkThreads, kWalkBlocks)
value_grad_kernel(const __grid_constant__ ValueGradArgs a) {
  using S = Share<DT, G, CH>;
  extern __shared__ __align__(16) unsigned char grad_smem[];
  const int lane = threadIdx.x, first = S::feature(0, lane % G);
  const int nf = min(a.N - a.f0, S::kFeatures);
  RowStarts ptr;
  ptr.init(a.indptr, a.rows, a.nnz);
  const int64_t q = blockIdx.x;
  if ((q << a.lg) >= ptr.total) return;
  WalkSmem& walk = *reinterpret_cast<WalkSmem*>(grad_smem);
  uint4* ring = reinterpret_cast<uint4*>(walk.ring);
  for (int i = lane; i < kRingBytes / 16 + 1; i += 32) ring[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncwarp();
  const WalkArgs wa{a.indices + ptr.base, nullptr, nullptr, nullptr, reinterpret_cast<const char*>(a.B) + (int64_t)a.f0 * dtype_bytes(DT), a.pitch_b, nf};
  GradWork<DT, G, CH, VIO> work{a, a.f0, nf, a.f0 + first, nf - first, lane % G, S::kShifted || a.N % S::VEC != 0, !S::kShifted && a.vec && a.N % S::VEC == 0};
  RowWalk<DT, G, CH, false, GradWork<DT, G, CH, VIO>>(wa, ptr, walk, work).range(q, a.lg, a.slack);
}

template <int DT, int G, int CH, bool VIO>
cudaError_t launch_value_grad_as(ValueGradArgs a, cudaStream_t st) {
  constexpr auto kernel = value_grad_kernel<DT, G, CH, VIO>;
  constexpr int smem = (int)sizeof(WalkSmem);
  cudaError_t e = allow_smem<kernel>(smem);
  const unsigned grid = (unsigned)ceil_div64(a.nnz, (int64_t)1 << a.lg);
  for (a.f0 = 0; a.f0 < a.N && e == cudaSuccess; a.f0 += Share<DT, G, CH>::kFeatures) {
    kernel<<<grid, kWalkThreads, smem, st>>>(a);
    e = cudaGetLastError();
  }
  return e;
}

template <int DT>
cudaError_t launch_value_grad(const ValueGradArgs& a, cudaStream_t st) {
  return with_row_shape<DT>((uintptr_t)a.B % 16 == 0 && a.pitch_b % 16 == 0, a.N, [&](auto G, auto CH) {
    if constexpr (CH.value > 0) {
      if (a.vec && a.dy_dtype == DT && a.N % Share<DT, G.value, CH.value>::VEC == 0) return launch_value_grad_as<DT, G.value, CH.value, true>(a, st);
    }
    return launch_value_grad_as<DT, G.value, CH.value, false>(a, st);
  });
}

}  // namespace
}  // namespace lf

using namespace lf;

extern "C" {

size_t lf_act_backward_workspace_bytes(int64_t rows, int32_t N) {
  if (rows < 1 || N < 1) return 0;
  return (size_t)(rows < kMostParts ? rows : kMostParts) * (size_t)N * sizeof(float);
}

int lf_act_backward(const void* dy, int64_t ld_dy, const void* preact, int64_t ld_preact, int32_t dtype,
                    int32_t activation, void* dz, int64_t ld_dz, float* dbias, int64_t rows, int32_t N,
                    void* workspace, size_t workspace_bytes, void* stream) {
  return lf_act_backward_as(dy, ld_dy, preact, ld_preact, dtype, activation, dz, dtype, ld_dz, dbias, rows, N, workspace,
                            workspace_bytes, stream);
}

int lf_act_backward_as(const void* dy, int64_t ld_dy, const void* preact, int64_t ld_preact, int32_t dtype,
                       int32_t activation, void* dz, int32_t dz_dtype, int64_t ld_dz, float* dbias, int64_t rows,
                       int32_t N, void* workspace, size_t workspace_bytes, void* stream) {
  LF_REQUIRE(rows >= 0 && rows < (1ll << 31) - 64 && N >= 1, "bad sizes");
  LF_REQUIRE(is_wide_dtype(dtype), "the type must be float32, bfloat16 or float16");
  LF_REQUIRE(!dz || dz_dtype == dtype || dz_dtype == LF_DTYPE_F32, "dz must have dy's type or float32");
  LF_REQUIRE(activation >= LF_ACT_NONE && activation <= LF_ACT_GELU_TANH, "unknown activation");
  LF_REQUIRE(dz || dbias, "nothing to compute");
  cudaStream_t st = (cudaStream_t)stream;
  if (rows == 0) {
    if (dbias) LF_CUDA_CHECK(cudaMemsetAsync(dbias, 0, (size_t)N * sizeof(float), st));
    return LF_OK;
  }
  LF_REQUIRE(dy && (preact || activation == LF_ACT_NONE), "null pointer argument");
  LF_REQUIRE(ld_dy >= N && (activation == LF_ACT_NONE || ld_preact >= N) && (!dz || ld_dz >= N), "bad leading dimension");
  LF_REQUIRE(aligned_for(dy, dtype) && (activation == LF_ACT_NONE || aligned_for(preact, dtype)) && aligned_for(dz, dz_dtype) && aligned(dbias, 4) &&
                 (!dbias || aligned(workspace, 4)),
             "an address is not a multiple of its type's size");
  if (dbias && (!workspace || workspace_bytes < lf_act_backward_workspace_bytes(rows, N)))
    return fail(LF_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace_bytes,
                lf_act_backward_workspace_bytes(rows, N));
  const void* z = activation == LF_ACT_NONE ? nullptr : preact;
  const int per = 16 / dtype_bytes(dtype);
  const bool vec = N % per == 0 && on_grid16(dy, ld_dy, dtype) && (!z || on_grid16(z, ld_preact, dtype)) && (!dz || on_grid16(dz, ld_dz, dz_dtype));
  const int pieces = vec ? N / per : N;
  int per_row = 4;
  while (per_row < pieces && per_row < 256) per_row *= 2;
  const ActGradArgs a{dy, z, dz, dbias ? (float*)workspace : nullptr, rows, ld_dy, ld_preact, ld_dz, N, activation, per_row};
  const int64_t want = ceil_div64(rows, 256 / per_row);
  const int parts = (int)(want < kMostParts ? want : kMostParts);
  const dim3 grid((unsigned)parts, (unsigned)((pieces + per_row - 1) / per_row));
  LF_REQUIRE(grid.y < 65536, "too many features");
  const bool wide = dz && dz_dtype != dtype;
#define LF_GO(DT_, OUT_, VEC_) \
  if (vec) act_grad_kernel<DT_, OUT_, VEC_><<<grid, 256, 0, st>>>(a); \
  else act_grad_kernel<DT_, OUT_, 1><<<grid, 256, 0, st>>>(a)
  if (dtype == LF_DTYPE_F32) { LF_GO(LF_DTYPE_F32, LF_DTYPE_F32, 4); }
  else if (dtype == LF_DTYPE_BF16 && !wide) { LF_GO(LF_DTYPE_BF16, LF_DTYPE_BF16, 8); }
  else if (dtype == LF_DTYPE_BF16) { LF_GO(LF_DTYPE_BF16, LF_DTYPE_F32, 8); }
  else if (!wide) { LF_GO(LF_DTYPE_F16, LF_DTYPE_F16, 8); }
  else { LF_GO(LF_DTYPE_F16, LF_DTYPE_F32, 8); }
#undef LF_GO
  LF_CUDA_CHECK(cudaGetLastError());
  if (dbias) LF_CUDA_CHECK(launch_column_sum(a.partial, parts, N, dbias, st));
  return LF_OK;
}

int lf_spmm_csr_grad_values(const int64_t* indptr, const int32_t* indices, int64_t row_begin, int64_t row_end,
                            int64_t nnz, const void* dy, int64_t ld_dy, const void* preact, int64_t ld_preact,
                            int32_t dy_dtype, int32_t activation, const void* B, int32_t b_dtype, int64_t ldb,
                            int32_t N, float* dvalues, void* stream) {
  LF_REQUIRE(N >= 1 && N <= (1 << 22) && ldb >= N && ldb < (1ll << 30) && ld_dy >= N && ld_dy < (1ll << 30), "bad sizes");
  LF_REQUIRE(0 <= row_begin && row_begin <= row_end && row_end - row_begin < (1ll << 31) - 64 && nnz >= 0, "bad row range");
  LF_REQUIRE(is_wide_dtype(dy_dtype) && is_wide_dtype(b_dtype), "the types must be float32, bfloat16 or float16");
  LF_REQUIRE(activation >= LF_ACT_NONE && activation <= LF_ACT_GELU_TANH, "unknown activation");
  if (row_begin == row_end || nnz == 0) return LF_OK;
  LF_REQUIRE(indptr && indices && dy && B && dvalues, "null pointer argument");
  LF_REQUIRE(activation == LF_ACT_NONE || (preact && ld_preact >= N && ld_preact < (1ll << 30)), "preact missing");
  LF_REQUIRE(aligned(indptr, 8) && aligned(indices, 4) && aligned(dvalues, 4) && aligned_for(dy, dy_dtype) &&
                 (activation == LF_ACT_NONE || aligned_for(preact, dy_dtype)) && aligned_for(B, b_dtype),
             "an address is not a multiple of its type's size");
  const int lg = range_log(nnz, row_end - row_begin);
  LF_REQUIRE((nnz >> lg) < (1ll << 31) - 1, "too many entries");
  const uint32_t bytes = (uint32_t)dtype_bytes(dy_dtype);
  const ValueGradArgs a{indptr + row_begin, indices, nnz, dy, activation == LF_ACT_NONE ? nullptr : preact, B, dvalues,
                        (uint32_t)ld_dy * bytes, (uint32_t)ld_preact * bytes, (uint32_t)ldb * dtype_bytes(b_dtype),
                        (int)(row_end - row_begin), N, dy_dtype, activation, lg, range_slack(lg), 0,
                        on_grid16(dy, ld_dy, dy_dtype) && (activation == LF_ACT_NONE || on_grid16(preact, ld_preact, dy_dtype))};
  cudaStream_t st = (cudaStream_t)stream;
  if (b_dtype == LF_DTYPE_F32) LF_CUDA_CHECK(launch_value_grad<LF_DTYPE_F32>(a, st));
  else if (b_dtype == LF_DTYPE_BF16) LF_CUDA_CHECK(launch_value_grad<LF_DTYPE_BF16>(a, st));
  else LF_CUDA_CHECK(launch_value_grad<LF_DTYPE_F16>(a, st));
  return LF_OK;
}

}  // extern "C"
