// Root-mean-square norm of the rows of a feature matrix, the residual's addition before it, and its gradients.
#include <type_traits>

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

// Rows of e4m3.  y / scale = 448 h w / max|h w| has no rstd in it, so it is made from p = h (448 w) alone, which is exact for
// bfloat16 rows and weights: halves between two stored values, frequent among numbers of few bits, go to the even one (from y =
// h rstd w and a reciprocal of the scale 17 000 of 134 million went to the other).  Rows whose largest |y| is below 448 * 2^-126
// count as zero.
struct E4m3Row {
  float scale;     // what the stored values are multiples of
  float top;       // max|h w|
  float inverse;   // 1 / top, or 0 for a row of zeros
  __device__ __forceinline__ E4m3Row(float most, float rstd) {   // most: the largest |p|
    top = __fdiv_rn(most, 448.f);
    scale = rstd * top * (1.f / 448.f);
    const bool zero = scale < 1.17549435e-38f;   // a NaN is none
    inverse = zero ? 0.f : __frcp_rn(top);
    if (zero) scale = 0.f;
  }
  // A top so small that its reciprocal may overflow (only beside an eps far below 10^-30): p and top are taken 2^100-fold.
  __device__ __forceinline__ bool tiny() const { return top < 0x1p-100f; }
  __device__ __forceinline__ float lift() {
    top *= 0x1p100f;
    if (inverse != 0.f) inverse = __frcp_rn(top);
    return 0x1p100f;
  }
  // p / top: a product with the reciprocal, and what is left of p added
  __device__ __forceinline__ float quotient(float p) const {
    const float t = p * inverse;
    return fmaf(fmaf(-t, top, p), inverse, t);
  }
};

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
    if (a.y_dtype != LF_DTYPE_E4M3) {
      for (int f = threadIdx.x; f < a.N; f += 256)
        put_any(a.y, row * a.ld_y + f, a.y_dtype, T::get(h[f]) * rstd * get_any(a.weight, f, a.weight_dtype));
      continue;
    }
    float most = 0.f;
    for (int f = threadIdx.x; f < a.N; f += 256)
      most = max_nan(most, fabsf(T::get(h[f]) * (448.f * get_any(a.weight, f, a.weight_dtype))));
    E4m3Row to(block_max(most, smem), rstd);
    if (threadIdx.x == 0) a.scale[row] = to.scale;
    const float lift = to.tiny() ? to.lift() : 1.f;
    auto* y = reinterpret_cast<__nv_fp8_storage_t*>(a.y) + row * a.ld_y;
    for (int f = threadIdx.x; f < a.N; f += 256)
      y[f] = Type<LF_DTYPE_E4M3>::put(to.quotient(T::get(h[f]) * (448.f * get_any(a.weight, f, a.weight_dtype)) * lift));
  }
}

// Sum or maximum over the L threads that share a row: part of a warp, or the whole block (L > 32).
template <int L, bool MAX>
__device__ __forceinline__ float row_reduce(float v, float* smem) {
#pragma unroll
  for (int o = (L > 32 ? 16 : L / 2); o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, v, o);
    v = MAX ? max_nan(v, u) : v + u;
  }
  if constexpr (L > 32) {
    constexpr int W = L / 32;
    if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
    __syncthreads();
    v = smem[threadIdx.x & (W - 1)];
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
      const float u = __shfl_xor_sync(0xffffffffu, v, o);
      v = MAX ? max_nan(v, u) : v + u;
    }
    __syncthreads();
  }
  return v;
}

// The chunks of one row that a thread holds: C of VEC elements, L * VEC apart.  `left`: elements from its first one
// to the end of the row.
template <int DT, int VEC, int L, int C>
struct RowPart {
  using E = typename Type<DT>::T;
  Pack<DT, VEC> p[C];
  __device__ __forceinline__ void fetch(const E* first, int left) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (c * L * VEC < left) p[c].fetch(first + c * L * VEC);
  }
};

// Whether the next row of a thread is fetched before this one is done: as far as registers go.
template <int VEC, int L, int C> constexpr bool kFetchAhead = C * VEC <= 16;

// A row in the registers of L threads.  Every input is read once and every output written once, so memory bounds
// it, if the instructions per element are few: conversions go in pairs, y is kept between the row's maximum and
// its rounding, and what is done once a row (sums over the threads, root, quotient) is done for 32 / L rows at a
// time.  2^20 rows of 128 bfloat16 with a residual, to 8 bits: 150 us, 6.3 TB/s (a copy of as much 145).
template <int DT, int OUT, int VEC, int L, int C>
__global__ void __launch_bounds__(L > 32 ? L : 256)
rms_norm_kernel(NormArgs a) {
  using E = typename Type<DT>::T;
  using O = typename Type<OUT>::T;
  constexpr int GROUPS = L > 32 ? 1 : 256 / L;
  constexpr bool AHEAD = kFetchAhead<VEC, L, C>;
  __shared__ float smem[32];
  const int t = L > 32 ? threadIdx.x : threadIdx.x % L, group = L > 32 ? 0 : threadIdx.x / L;
  const int left = a.N - t * VEC;
  const bool add = a.res != nullptr;
  const float inv_n = 1.f / (float)a.N;
  float w[C][VEC];
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) w[c][i] = c * L * VEC < left ? (OUT == LF_DTYPE_E4M3 ? 448.f : 1.f) * get_any(a.weight, (t + c * L) * VEC + i, a.weight_dtype) : 0.f;
  }
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const E* px = reinterpret_cast<const E*>(a.x) + row * a.ld_x + t * VEC;
  const E* pr = reinterpret_cast<const E*>(a.res) + row * a.ld_res + t * VEC;
  E* ps = reinterpret_cast<E*>(a.sum) + row * a.ld_sum + t * VEC;
  O* py = reinterpret_cast<O*>(a.y) + row * a.ld_y + t * VEC;
  RowPart<DT, VEC, L, C> x, r;
  auto fetch = [&](bool there) {
    if (there) {
      x.fetch(px, left);
      if (add) r.fetch(pr, left);
    }
    px += step * a.ld_x;
    pr += step * a.ld_res;
  };
  if (AHEAD) fetch(row < a.rows);
  for (; row - group < a.rows; row += step) {   // the same number of turns for the whole block
    const bool ok = row < a.rows;
    if (!AHEAD) fetch(ok);
    float y[C][VEC], ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const bool in = ok && c * L * VEC < left;
#pragma unroll
      for (int i = 0; i < VEC; ++i) y[c][i] = x.p[c].get(i);
      if (add) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[c][i] += r.p[c].get(i);
        Pack<DT, VEC> h;
        h.put(y[c]);
        if (in) h.store(ps + c * L * VEC);
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[c][i] = h.get(i);   // the norm is that of the sum as it is kept
      }
      float sc = 0.f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) sc = fmaf(y[c][i], y[c][i], sc);
      ss += in ? sc : 0.f;
    }
    if (AHEAD) fetch(row + step < a.rows);
    const float rstd = rsqrtf(row_reduce<L, false>(ss, smem) * inv_n + a.eps);
    if (a.rstd && t == 0 && ok) a.rstd[row] = rstd;
    if constexpr (OUT == LF_DTYPE_E4M3) {
      float most = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float mc = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          y[c][i] *= w[c][i];
          mc = max_nan(mc, fabsf(y[c][i]));
        }
        if (c * L * VEC < left) most = max_nan(most, mc);
      }
      E4m3Row to(row_reduce<L, true>(most, smem), rstd);
      if (t == 0 && ok) a.scale[row] = to.scale;
      if (to.tiny()) {
        const float lift = to.lift();
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) y[c][i] *= lift;
        }
      }
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[c][i] = to.quotient(y[c][i]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) y[c][i] *= rstd * w[c][i];
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      Pack<OUT, VEC> o;
      o.put(y[c]);
      if (ok && c * L * VEC < left) o.keep(py + c * L * VEC);
    }
    ps += step * a.ld_sum;
    py += step * a.ld_y;
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

// Blocks of the gradient's kernel that an SM holds at a time; the launch has as many, since each walks over an equal
// share of the rows (2^18 rows of 512 bfloat16: 3 held and 592 launched 236 us, 444 181: 5.9 TB/s).  Wider rows have one, and nothing
// on its way between a row's two barriers: 2^15 rows of 4096 bfloat16 335 us where the bytes take 164; 257 to 512 float32
// features spill (2^18 rows of 384: 360 us for 246), and rows off the grid beyond 4096 go element by element, their sums in
// memory (2^14 rows of 4099 bfloat16: 845 us for 82).
template <int VEC, int L, int C> constexpr int kGradResident = L <= 256 && C * VEC <= 16 ? 3 : 1;

// The same for the gradients, row after row; the weight's is summed over the rows that a thread sees, then over the groups of its
// block, and the blocks' sums by column_sum_kernel: one order, whatever block runs first.
template <int DT, int VEC, int L, int C>
__global__ void __launch_bounds__(L > 32 ? L : 256, kGradResident<VEC, L, C>)
rms_norm_grad_kernel(NormGradArgs a) {
  using E = typename Type<DT>::T;
  constexpr int GROUPS = L > 32 ? 1 : 256 / L;
  __shared__ float smem[32];
  __shared__ float sums[GROUPS > 1 ? 256 * C * VEC : 1];
  const int t = L > 32 ? threadIdx.x : threadIdx.x % L, group = L > 32 ? 0 : threadIdx.x / L;
  float w[C][VEC], dw[C][VEC];
#pragma unroll
  for (int c = 0; c < C; ++c) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int f = (t + c * L) * VEC + i;
      w[c][i] = f < a.N ? get_any(a.weight, f, a.weight_dtype) : 0.f;
      dw[c][i] = 0.f;
    }
  }
  const float inv_n = 1.f / (float)a.N;
  const int left = a.N - t * VEC;
  const bool add = a.dsum != nullptr;
  RowPart<DT, VEC, L, C> dy, h, ds;
  float rstd = 0.f;
  int64_t row = (int64_t)blockIdx.x * GROUPS + group;
  const int64_t step = (int64_t)gridDim.x * GROUPS;
  const E* pdy = reinterpret_cast<const E*>(a.dy) + row * a.ld_dy + t * VEC;
  const E* ph = reinterpret_cast<const E*>(a.h) + row * a.ld_h + t * VEC;
  const E* pds = reinterpret_cast<const E*>(a.dsum) + row * a.ld_dsum + t * VEC;
  E* pdx = reinterpret_cast<E*>(a.dx) + row * a.ld_dx + t * VEC;
  auto fetch = [&](int64_t from) {
    if (from < a.rows) {
      dy.fetch(pdy, left);
      h.fetch(ph, left);
      if (add) ds.fetch(pds, left);
      rstd = __ldg(a.rstd + from);
    }
    pdy += step * a.ld_dy;
    ph += step * a.ld_h;
    pds += step * a.ld_dsum;
  };
  for (; row - group < a.rows; row += step) {   // the same number of turns for the whole block
    const bool ok = row < a.rows;
    fetch(row);
    float dot = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (ok && c * L * VEC < left) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float dn = dy.p[c].get(i) * (h.p[c].get(i) * rstd);
          dw[c][i] += dn;
          dot = fmaf(dn, w[c][i], dot);
        }
      }
    }
    const float mean = row_reduce<L, false>(dot, smem) * inv_n;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (ok && c * L * VEC < left) {
        float g[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          g[i] = rstd * (dy.p[c].get(i) * w[c][i] - h.p[c].get(i) * rstd * mean);
          if (add) g[i] += ds.p[c].get(i);
        }
        Pack<DT, VEC> o;
        o.put(g);
        o.store(pdx + c * L * VEC);
      }
    }
    pdx += step * a.ld_dx;
  }
  float* part = a.partial + (int64_t)blockIdx.x * a.N;
  if constexpr (GROUPS > 1) {
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) sums[group * (L * C * VEC) + (t + c * L) * VEC + i] = dw[c][i];
    }
    __syncthreads();
    for (int f = threadIdx.x; f < a.N; f += 256) {
      float s = 0.f;
#pragma unroll
      for (int g = 0; g < GROUPS; ++g) s += sums[g * (L * C * VEC) + f];
      part[f] = s;
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if ((t + c * L) * VEC + i < a.N) part[(t + c * L) * VEC + i] = dw[c][i];
    }
  }
}

// out[f] = sum over the `parts` rows of partial: 32 threads take every 32nd row of a column, then their sums in turn
// (444 rows of 512: 6 us, latency)
__global__ void __launch_bounds__(1024)
column_sum_kernel(const float* __restrict__ partial, int parts, int N, float* __restrict__ out) {
  __shared__ float smem[32][33];
  const int f = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  float s = 0.f;
  if (f < N) {
#pragma unroll 8
    for (int p = w; p < parts; p += 32) s += partial[(int64_t)p * N + f];
  }
  smem[threadIdx.x & 31][w] = s;
  __syncthreads();
  s = warp_sum(smem[w][threadIdx.x & 31]);
  const int g = blockIdx.x * 32 + w;
  if ((threadIdx.x & 31) == 0 && g < N) out[g] = s;
}

}  // namespace

cudaError_t launch_column_sum(const float* partial, int parts, int N, float* out, cudaStream_t st) {
  column_sum_kernel<<<(N + 31) / 32, 1024, 0, st>>>(partial, parts, N, out);
  return cudaGetLastError();
}

namespace {

constexpr int kNormGradBlocks = 3 * kSms;

inline bool rows_on(const void* p, int64_t ld, int bytes, int grid) { return (uintptr_t)p % grid == 0 && ld * bytes % grid == 0; }

// Threads and chunks per row.  Chunks of 16 bytes where every row starts on such a boundary and holds whole
// chunks, else single elements.  A few chunks a thread, so that a warp holds several narrow rows; a block and its
// barriers only for rows that a warp has no registers for.
template <int DT, class F>
cudaError_t with_norm_shape(bool vec, int N, F&& go) {
  constexpr int V = 16 / (int)sizeof(typename Type<DT>::T);
#define LF_SHAPE(VEC_, L_, C_) \
  if (N <= VEC_ * L_ * C_) return go(std::integral_constant<int, VEC_>(), std::integral_constant<int, L_>(), \
                                     std::integral_constant<int, C_>())
  if (vec) {
    LF_SHAPE(V, 4, 2);
    LF_SHAPE(V, 8, 2);
    LF_SHAPE(V, 16, 2);
    LF_SHAPE(V, 32, 2);
    LF_SHAPE(V, 32, 4);
    LF_SHAPE(V, 256, 1);
    LF_SHAPE(V, 512, 1);
    LF_SHAPE(V, 512, 2);
    LF_SHAPE(V, 512, 4);
  } else {
    LF_SHAPE(1, 8, 8);
    LF_SHAPE(1, 16, 8);
    LF_SHAPE(1, 32, 8);
    LF_SHAPE(1, 256, 4);
    LF_SHAPE(1, 512, 8);
  }
#undef LF_SHAPE
  return cudaErrorNotSupported;   // wider: the kernel that walks over the row
}

template <int DT>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t st) {
  const int e = (int)sizeof(typename Type<DT>::T), v = 16 / e;
  const bool vec = a.N % v == 0 && rows_on(a.x, a.ld_x, e, 16) && (!a.res || (rows_on(a.res, a.ld_res, e, 16) && rows_on(a.sum, a.ld_sum, e, 16))) &&
                   rows_on(a.y, a.ld_y, dtype_bytes(a.y_dtype), v * dtype_bytes(a.y_dtype) < 16 ? v * dtype_bytes(a.y_dtype) : 16);
  const cudaError_t done = with_norm_shape<DT>(vec, a.N, [&](auto VEC, auto L, auto C) {
    constexpr int threads = L.value > 32 ? L.value : 256, rpb = threads / L.value;
    const int64_t blocks = ceil_div64(a.rows, rpb), most = kSms * 12 * 256 / threads;   // the weight is read once per block
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    if (a.y_dtype == LF_DTYPE_E4M3) rms_norm_kernel<DT, LF_DTYPE_E4M3, VEC.value, L.value, C.value><<<grid, threads, 0, st>>>(a);
    else if (a.y_dtype == LF_DTYPE_F32) rms_norm_kernel<DT, LF_DTYPE_F32, VEC.value, L.value, C.value><<<grid, threads, 0, st>>>(a);
    else if (a.y_dtype == LF_DTYPE_BF16) rms_norm_kernel<DT, LF_DTYPE_BF16, VEC.value, L.value, C.value><<<grid, threads, 0, st>>>(a);
    else rms_norm_kernel<DT, LF_DTYPE_F16, VEC.value, L.value, C.value><<<grid, threads, 0, st>>>(a);
    return cudaGetLastError();
  });
  if (done != cudaErrorNotSupported) return done;
  rms_norm_rows_kernel<DT><<<(unsigned)(a.rows < (1 << 20) ? a.rows : 1 << 20), 256, 0, st>>>(a);
  return cudaGetLastError();
}

template <int DT>
cudaError_t launch_norm_grad(const NormGradArgs& a, float* dweight, cudaStream_t st) {
  const int e = (int)sizeof(typename Type<DT>::T), v = 16 / e;
  const bool vec = a.N % v == 0 && rows_on(a.dy, a.ld_dy, e, 16) && rows_on(a.h, a.ld_h, e, 16) && rows_on(a.dx, a.ld_dx, e, 16) &&
                   (!a.dsum || rows_on(a.dsum, a.ld_dsum, e, 16));
  int blocks = (int)(a.rows < kNormGradBlocks ? a.rows : kNormGradBlocks);
  cudaError_t done = with_norm_shape<DT>(vec, a.N, [&](auto VEC, auto L, auto C) {
    constexpr int threads = L.value > 32 ? L.value : 256, rpb = threads / L.value;
    const int64_t want = ceil_div64(a.rows, rpb), most = kSms * kGradResident<VEC.value, L.value, C.value>;
    blocks = (int)(want < most ? want : most);
    rms_norm_grad_kernel<DT, VEC.value, L.value, C.value><<<blocks, threads, 0, st>>>(a);
    return cudaGetLastError();
  });
  if (done == cudaErrorNotSupported) {
    rms_norm_grad_rows_kernel<DT><<<blocks, 256, 0, st>>>(a);
    done = cudaGetLastError();
  }
  return done == cudaSuccess ? launch_column_sum(a.partial, blocks, a.N, dweight, st) : done;
}

}  // namespace
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
  LF_REQUIRE(aligned_for(x, dtype) && aligned_for(residual, dtype) && (!residual || aligned_for(sum, dtype)) && aligned_for(weight, weight_dtype) &&
                 aligned_for(y, y_dtype) && (y_dtype != LF_DTYPE_E4M3 || aligned(scale, 4)) && aligned(rstd, 4),
             "an address is not a multiple of its type's size");
  const NormArgs a{x, residual, weight, sum, y, scale, rstd, rows, ld_x, ld_residual, ld_sum, ld_y, N, weight_dtype, y_dtype, eps};
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == LF_DTYPE_F32) LF_CUDA_CHECK(launch_norm<LF_DTYPE_F32>(a, st));
  else if (dtype == LF_DTYPE_BF16) LF_CUDA_CHECK(launch_norm<LF_DTYPE_BF16>(a, st));
  else LF_CUDA_CHECK(launch_norm<LF_DTYPE_F16>(a, st));
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
  LF_REQUIRE(aligned_for(dy, dtype) && aligned_for(h, dtype) && aligned_for(dsum, dtype) && aligned_for(dx, dtype) && aligned_for(weight, weight_dtype) &&
                 aligned(rstd, 4) && aligned(dweight, 4) && aligned(workspace, 4),
             "an address is not a multiple of its type's size");
  if (workspace_bytes < lf_rms_norm_backward_workspace_bytes(rows, N) || !workspace)
    return fail(LF_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace_bytes,
                lf_rms_norm_backward_workspace_bytes(rows, N));
  const NormGradArgs a{dy, h, weight, rstd, dsum, dx, (float*)workspace, rows, ld_dy, ld_h, ld_dsum, ld_dx, N, weight_dtype};
  if (dtype == LF_DTYPE_F32) LF_CUDA_CHECK(launch_norm_grad<LF_DTYPE_F32>(a, dweight, st));
  else if (dtype == LF_DTYPE_BF16) LF_CUDA_CHECK(launch_norm_grad<LF_DTYPE_BF16>(a, dweight, st));
  else LF_CUDA_CHECK(launch_norm_grad<LF_DTYPE_F16>(a, dweight, st));
  return LF_OK;
}

}  // extern "C"
