// CSR product with the end of a layer in its epilogue: Y = act(A * B + bias) + residual.
//
// What it has to move: the entries (8 bytes each), C and the residual once; what bounds it are the rows of B, one for each
// entry, out of the L2 and, as far as B is larger than that, out of memory, and the instructions that unpack and add them.
// 2^20 power-law rows with 13.2 M entries: 128 bfloat16 features 555 us (3.4 GB of rows of B, 6.1 TB/s), the same in 8 bits
// 584; the entries, one read of B and C and the residual would take 0.14 and 0.12 ms.
//
// Two launches.  In the first a warp takes a range of entries and does the rows in it (lf_layer_rows.cuh); a group of
// lanes that has summed up its row runs the epilogue on its registers, the residual having been fetched along with the rows
// of B.  The second launch adds up, in order, the pieces of rows that several ranges share, and does the rows without
// entries.
#include <type_traits>

#include "lf_layer_rows.cuh"

namespace lf {
namespace {

struct ActArgs {
  const int64_t* indptr;   // of row_begin
  const int32_t* indices;
  const float* data;       // or NULL: all ones
  const int32_t* order;    // data of entry e is data[order[e]], or NULL: data[e]
  int64_t nnz;
  const void* B;
  const float* b_scale;    // or NULL
  const void* bias;
  const void* residual;
  void* preact;
  void* C;
  float* partial;          // [2 * ranges][ld_partial]: sums of a range's first row, where it started earlier, and
  int64_t ld_partial;      //   of its last row, where it goes on
  uint32_t pitch_b, pitch_res, pitch_pre, pitch_c;   // bytes between rows
  int rows, N, bias_dtype, res_dtype, c_dtype, act;
  int lg, slack;           // entries of a range: 1 << lg; how far a row may reach behind it
  bool vec;                // rows of C, residual and preact start on 16-byte boundaries, N is a multiple of 8
};

// ---- epilogue ---------------------------------------------------------------------------------------
__device__ __forceinline__ char* row_at(const void* base, int row, uint32_t pitch) {
  return reinterpret_cast<char*>(const_cast<void*>(row_of_b(base, (uint32_t)row, pitch)));
}

// What a lane has of a row: BLOCKS of n neighbouring features, `apart` from one block to the next, `left` of them from the
// first on to the row's end.  vec: the row is on the 16-byte grid and holds whole eights, so blocks move as they are, and
// `w` holds them side by side; otherwise one by one, one a word.  (In a loop over memory, as each is needed once: 80 802 rows with 1.3 M
// entries, 168 features in 8 bits, 326 us for 130.)
template <int BLOCKS, int n, bool FULL>   // FULL: activations for results in 32 bits
struct RowIo {
  static __device__ __forceinline__ void load(const char* p, int dt, bool vec, int apart, int left, uint32_t* w) {
    if (vec) {
      load_blocks<BLOCKS, n>(p, dt, apart, left, w);
    } else if (dt == LF_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < BLOCKS * n; ++i)
        if (i / n * apart + i % n < left) w[i] = __ldcs(reinterpret_cast<const uint32_t*>(p) + i / n * apart + i % n);
    } else {
#pragma unroll
      for (int i = 0; i < BLOCKS * n; ++i)
        if (i / n * apart + i % n < left) w[i] = __ldcs(reinterpret_cast<const uint16_t*>(p) + i / n * apart + i % n);
    }
  }
  static __device__ __forceinline__ void add(const uint32_t* w, int dt, bool vec, float* v) {
    if (vec) {
      use_blocks<BLOCKS, n>(w, dt, v, [](float x, float y) { return x + y; });
      return;
    }
#pragma unroll
    for (int i = 0; i < BLOCKS * n; ++i)
      v[i] += dt == LF_DTYPE_F32 ? __uint_as_float(w[i]) : dt == LF_DTYPE_BF16 ? __uint_as_float(w[i] << 16) : __half2float(__ushort_as_half((unsigned short)w[i]));
  }
  static __device__ __forceinline__ void store(char* p, int dt, bool vec, int apart, int left, const float* v) {
    if (vec) {
      const int bytes = dtype_bytes(dt);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        if (b * apart >= left) break;
        char* q = p + b * apart * bytes;
        if (dt == LF_DTYPE_F32) {
#pragma unroll
          for (int i = 0; i < n; i += 4) __stcs(reinterpret_cast<float4*>(q + i * 4), make_float4(v[b * n + i], v[b * n + i + 1], v[b * n + i + 2], v[b * n + i + 3]));
        } else {
          uint32_t h[n / 2 > 0 ? n / 2 : 1];
#pragma unroll
          for (int i = 0; i < n; i += 2) {
            if (dt == LF_DTYPE_BF16) *reinterpret_cast<__nv_bfloat162*>(h + i / 2) = __floats2bfloat162_rn(v[b * n + i], v[b * n + i + 1]);
            else *reinterpret_cast<__half2*>(h + i / 2) = __floats2half2_rn(v[b * n + i], v[b * n + i + 1]);
          }
          if constexpr (n == 4) {
            __stcs(reinterpret_cast<uint2*>(q), make_uint2(h[0], h[1]));
          } else {
#pragma unroll
            for (int i = 0; i < n / 2; i += 4) __stcs(reinterpret_cast<uint4*>(q + i * 4), make_uint4(h[i], h[i + 1], h[i + 2], h[i + 3]));
          }
        }
      }
    } else if (dt == LF_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < BLOCKS * n; ++i)
        if (i / n * apart + i % n < left) reinterpret_cast<float*>(p)[i / n * apart + i % n] = v[i];
    } else {
#pragma unroll
      for (int i = 0; i < BLOCKS * n; ++i) {
        const unsigned short h = dt == LF_DTYPE_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v[i])) : __half_as_ushort(__float2half_rn(v[i]));
        if (i / n * apart + i % n < left) reinterpret_cast<unsigned short*>(p)[i / n * apart + i % n] = h;
      }
    }
  }
  // z = A * B for features f on, `bias` theirs, w their residual -> what the call returns
  static __device__ __forceinline__ void finish(const ActArgs& a, int c_dtype, int res_dtype, bool vec, int row, int f, int apart, int left, const float* bias, const uint32_t* w, float* z) {
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) {
#pragma unroll
      for (int i = 0; i < n; ++i) z[b * n + i] += bias[b * apart + i];
    }
    const int at = f * dtype_bytes(c_dtype);
    if (a.preact) store(row_at(a.preact, row, a.pitch_pre) + at, c_dtype, vec, apart, left, z);
    activate_all<BLOCKS * n, FULL>(z, a.act);
    if (a.residual) add(w, res_dtype, vec, z);
    store(row_at(a.C, row, a.pitch_c) + at, c_dtype, vec, apart, left, z);
  }
};
// eight features, the residual fetched here
__device__ __forceinline__ void finish8(const ActArgs& a, int row, int f, const float* bias, float* z) {
  __align__(16) uint32_t w[8];
  if (a.residual) RowIo<1, 8, true>::load(row_at(a.residual, row, a.pitch_res) + f * dtype_bytes(a.res_dtype), a.res_dtype, a.vec, 8, a.N - f, w);
  RowIo<1, 8, true>::finish(a, a.c_dtype, a.res_dtype, a.vec, row, f, 8, a.N - f, bias, w, z);
}

// ---- the walk ---------------------------------------------------------------------------------------
// What is known of C, residual and preact when the kernel is compiled (the first launch alone, 2^20 power-law rows, 128 bfloat16
// features: 566 us with kAnyRows, 551 with kOnGrid, 540 with kTyped; in 8 bits 595 and 579 with the latter two; 2^20 uniform rows of 64 features in 8
// bits 790 with the first and 724 with the second).  Other types than kTyped's are compiled for the grid only from 8 bits, where
// there is no type of its own for C.
enum Rows { kAnyRows, kOnGrid, kTyped };   // on the grid: on 16-byte boundaries and of whole pieces; typed: of kOwn as well
template <int DT> constexpr int kOwn = DT == LF_DTYPE_E4M3 ? LF_DTYPE_BF16 : DT;

template <int DT, int G, int CH, Rows IO>
struct ActWork {
  using S = Share<DT, G, CH>;
  // the lane's share of a row in memory
  static constexpr int kBlock = S::kShifted ? 1 : S::VEC < 8 ? S::VEC : 8, kBlocks = S::kFloats / kBlock;   // whole blocks in a row of whole eights
  static constexpr int kApart = S::kShifted ? G : S::VEC > 8 ? 8 : G * S::VEC;
  using Io = RowIo<kBlocks, kBlock, IO != kTyped || kOwn<DT> == LF_DTYPE_F32>;
  const ActArgs& a;
  const float* bias;    // in shared memory, from the lane's first feature on
  int64_t slots;        // of the range in `partial`
  int f0, nf;           // the walk's features
  int f, left, gl;      // the lane's first feature; features from there to the end of the walk
  bool vec_;
  uint64_t sum[S::kPairs];
  __align__(16) uint32_t res[S::kFloats];

  __device__ __forceinline__ void coming(int row) const {   // the residual, 128 bytes at a time
    if (!a.residual) return;
    const int bytes = dtype_bytes(a.res_dtype);
    const char* p = row_at(a.residual, row, a.pitch_res) + f0 * bytes;
    for (int i = 0; i < nf * bytes; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(p + i));
  }
  static constexpr bool kPlaces = false;
  __device__ __forceinline__ bool vec() const { return IO != kAnyRows || vec_; }
  __device__ __forceinline__ int c_dtype() const { return IO == kTyped ? kOwn<DT> : a.c_dtype; }
  __device__ __forceinline__ int res_dtype() const { return IO == kTyped ? kOwn<DT> : a.res_dtype; }
  // The residual is on its way while the row is summed up, where its words take no more registers than the sums' rows of B; 16
  // bits of either kind are loaded alike.  (Any residual so, 16 words held for 8 used:
  // the 8-bit case above 630 us for 596.)
  __device__ __forceinline__ const char* residual_of(int row) const { return row_at(a.residual, row, a.pitch_res) + f * dtype_bytes(res_dtype()); }
  __device__ __forceinline__ bool early() const { return !S::kShifted && a.residual && vec() && (DT == LF_DTYPE_F32 || res_dtype() != LF_DTYPE_F32); }
  __device__ __forceinline__ void begin(int row, bool whole, int piece, int64_t, int) {
#pragma unroll
    for (int i = 0; i < S::kPairs; ++i) sum[i] = 0;
    if constexpr (!S::kShifted) {
      if (early() && row >= 0 && !(whole && piece >= 0))
        load_blocks<kBlocks, kBlock>(residual_of(row), DT == LF_DTYPE_F32 ? res_dtype() : LF_DTYPE_BF16, kApart, left, res);
    }
  }
  __device__ __forceinline__ void step(float v, const unsigned char* x) {
    uint64_t y[S::kPairs];
    S::floats(x, gl, y);
    const uint64_t vv = as_pair(__float_as_uint(v), __float_as_uint(v));
#pragma unroll
    for (int i = 0; i < S::kPairs; ++i) sum[i] = fma_pair(vv, y[i], sum[i]);
  }
  __device__ __forceinline__ void steps_done(int, bool) const {}
  __device__ __forceinline__ void end(int row, bool whole, int piece) {
    if (whole) {
#pragma unroll
      for (int o = G; o < 32; o <<= 1) {
#pragma unroll
        for (int i = 0; i < S::kPairs; ++i) sum[i] = add_pair(sum[i], __shfl_xor_sync(kAllLanes, (unsigned long long)sum[i], o));
      }
      if ((threadIdx.x & 31) >= G) return;
    }
    if (row < 0) return;
    float z[S::kFloats];
#pragma unroll
    for (int i = 0; i < S::kPairs; ++i) {
      const float2 p = as_floats(sum[i]);
      z[2 * i] = p.x;
      z[2 * i + 1] = p.y;
    }
    if (whole && piece >= 0) {   // as it is
      float* p = a.partial + (slots + piece) * a.ld_partial + f;
#pragma unroll
      for (int i = 0; i < S::kFloats; ++i)
        if (i / kBlock * kApart + i % kBlock < left) p[i / kBlock * kApart + i % kBlock] = z[i];
    } else {
      if (a.residual && !early()) Io::load(residual_of(row), res_dtype(), vec(), kApart, left, res);
      Io::finish(a, c_dtype(), res_dtype(), vec(), row, f, kApart, left, bias, res, z);
    }
  }
};

template <int DT, int G, int CH, bool IND, Rows IO>
__global__ void __launch_bounds__(kWalkThreads, kWalkBlocks)
spmm_csr_act_kernel(const __grid_constant__ ActArgs a) {
  using S = Share<DT, G, CH>;
  extern __shared__ __align__(16) unsigned char act_smem[];
  WalkSmem& walk = *reinterpret_cast<WalkSmem*>(act_smem);
  float* bias = reinterpret_cast<float*>(act_smem + sizeof(WalkSmem));
  let_dependents_launch();
  const int lane = threadIdx.x;
  const int f0 = blockIdx.y * S::kFeatures, nf = min(a.N - f0, S::kFeatures);
  for (int f = lane; f < S::kSpan; f += 32) bias[f] = a.bias && f < nf ? get_any(a.bias, f0 + f, a.bias_dtype) : 0.f;
  __syncwarp();
  RowStarts ptr;
  ptr.init(a.indptr, a.rows, a.nnz);
  const int64_t q = blockIdx.x;
  if ((q << a.lg) >= ptr.total) return;
  const WalkArgs wa{a.indices + ptr.base, a.data && !a.order ? a.data + ptr.base : a.data, a.order ? a.order + ptr.base : nullptr, a.b_scale,
                    reinterpret_cast<const char*>(a.B) + (int64_t)f0 * dtype_bytes(DT), a.pitch_b, nf};
  const int first = S::feature(0, lane % G);
  ActWork<DT, G, CH, IO> work{a, bias + first, 2 * q, f0, nf, f0 + first, nf - first, lane % G, !S::kShifted && a.vec};
  RowWalk<DT, G, CH, IND, ActWork<DT, G, CH, IO>>(wa, ptr, walk, work).range(q, a.lg, a.slack);
}

// Rows without entries, and rows that several ranges share: their pieces in order.  Most of its time goes into looking
// at row pointers (2^20 rows: 16 us).  A lane has eight features; rows of few pieces
// are a warp's, rows of many the block's, whose warps take every eighth piece.  Six blocks an SM, for the looking, leave 40 registers:
// the epilogue and the adding up spill (308 bytes), and act(bias) is computed for every row without entries.  Those are written at
// 3.3 TB/s.
constexpr int kLongPieces = 8;

__device__ __forceinline__ void bias8(const ActArgs& a, int f, float* b) {
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = a.bias && f + i < a.N ? get_any(a.bias, f + i, a.bias_dtype) : 0.f;
}
__device__ __forceinline__ void add_piece(const ActArgs& a, int64_t slot, int f, float* z) {
  const float4* p = reinterpret_cast<const float4*>(a.partial + slot * a.ld_partial + f);
  const float4 x = __ldcg(p), y = __ldcg(p + 1);
  z[0] += x.x; z[1] += x.y; z[2] += x.z; z[3] += x.w;
  z[4] += y.x; z[5] += y.y; z[6] += y.z; z[7] += y.w;
}

__global__ void __launch_bounds__(kThreads, 6)   // most blocks only look at row pointers: many of them at a time
finish_rows_kernel(const __grid_constant__ ActArgs a, int span) {   // span: rows of a block at a time, at most its threads
  __shared__ int rows_of[kThreads / 32][32], long_rows[kThreads], num_long;
  __shared__ int64_t starts_of[kThreads / 32][32], ends_of[kThreads / 32][32];
  __shared__ float sums[kThreads / 32][256 + 8];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  RowStarts ptr;
  ptr.init(a.indptr, a.rows, a.nnz);
  const int chunks = (a.N + 7) / 8;
  for (int64_t row0 = (int64_t)blockIdx.x * span; row0 < a.rows; row0 += (int64_t)gridDim.x * span) {
    if (threadIdx.x == 0) num_long = 0;
    __syncthreads();
    const int64_t row = row0 + threadIdx.x;
    int64_t s = 0, e = 0;
    bool mine = false;
    if (row < a.rows && threadIdx.x < span) {
      s = ptr((int)row);
      e = ptr((int)row + 1);
      mine = s >= e;
      if (!mine && row_is_cut(s, e, a.lg, a.slack)) {
        mine = ((e - 1) >> a.lg) - (s >> a.lg) < kLongPieces;
        if (!mine) long_rows[atomicAdd(&num_long, 1)] = (int)row;   // in any order: each row is one block's from here on
      }
    }
    const unsigned todo = __ballot_sync(kAllLanes, mine);
    if (mine) {
      const int i = __popc(todo & ((1u << lane) - 1u));
      rows_of[w][i] = (int)row;
      starts_of[w][i] = s;
      ends_of[w][i] = e;
    }
    __syncwarp();
    wait_for_prior_grid();   // the pieces are there
    const int per = chunks < 32 ? chunks : 32;   // lanes per row
    for (int c = lane % per; c < chunks && lane < 32 / per * per; c += per) {
      float bias[8];
      if (todo) bias8(a, c * 8, bias);
      for (int i = lane / per; i < __popc(todo); i += 32 / per) {
        const int64_t s1 = starts_of[w][i], e1 = ends_of[w][i];
        float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (s1 < e1) {
          const int64_t q0 = s1 >> a.lg, q1 = (e1 - 1) >> a.lg;
          add_piece(a, 2 * q0 + 1, c * 8, z);
#pragma unroll 8
          for (int64_t q = q0 + 1; q <= q1; ++q) add_piece(a, 2 * q, c * 8, z);
        }
        finish8(a, rows_of[w][i], c * 8, bias, z);
      }
    }
    __syncthreads();
    for (int i = 0; i < num_long; ++i) {
      const int r = long_rows[i];
      const int64_t q0 = ptr(r) >> a.lg, q1 = (ptr(r + 1) - 1) >> a.lg;
      for (int f0 = 0; f0 < a.N; f0 += 256) {
        const int f = f0 + lane * 8;
        float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (f < a.N) {
          if (w == 0) add_piece(a, 2 * q0 + 1, f, z);
#pragma unroll 8
          for (int64_t q = q0 + 1 + w; q <= q1; q += kThreads / 32) add_piece(a, 2 * q, f, z);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) sums[w][lane * 8 + k] = z[k];
        __syncthreads();
        if (w == 0 && f < a.N) {
          for (int v = 1; v < kThreads / 32; ++v) {
#pragma unroll
            for (int k = 0; k < 8; ++k) z[k] += sums[v][lane * 8 + k];
          }
          float bias[8];
          bias8(a, f, bias);
          finish8(a, r, f, bias, z);
        }
        __syncthreads();
      }
    }
    __syncthreads();
  }
}

template <int DT, int G, int CH, bool IND, Rows IO>
cudaError_t launch_walk_as(const ActArgs& a, cudaStream_t st) {
  using S = Share<DT, G, CH>;
  constexpr auto kernel = spmm_csr_act_kernel<DT, G, CH, IND, IO>;
  constexpr int smem = (int)sizeof(WalkSmem) + S::kSpan * 4;
  const cudaError_t e = allow_smem<kernel>(smem);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)ceil_div64(a.nnz, (int64_t)1 << a.lg), (unsigned)((a.N + S::kFeatures - 1) / S::kFeatures));
  kernel<<<grid, kWalkThreads, smem, st>>>(a);
  return cudaGetLastError();
}

template <int DT>
cudaError_t launch_walk(const ActArgs& a, cudaStream_t st) {
  return with_row_shape<DT>((uintptr_t)a.B % 16 == 0 && a.pitch_b % 16 == 0, a.N, [&](auto G, auto CH) {
    const auto launch = [&](auto io) {
      if constexpr (DT != LF_DTYPE_E4M3) {
        if (!a.b_scale && !a.order) return launch_walk_as<DT, G.value, CH.value, false, io.value>(a, st);
      }
      return launch_walk_as<DT, G.value, CH.value, true, io.value>(a, st);
    };
    if constexpr (CH.value > 0) {
      if (a.vec) {
        if (a.c_dtype == kOwn<DT> && (!a.residual || a.res_dtype == kOwn<DT>)) return launch(std::integral_constant<Rows, kTyped>());
        if constexpr (DT == LF_DTYPE_E4M3) return launch(std::integral_constant<Rows, kOnGrid>());
      }
    }
    return launch(std::integral_constant<Rows, kAnyRows>());
  });
}

}  // namespace
}  // namespace lf

using namespace lf;

extern "C" {

size_t lf_spmm_csr_act_workspace_bytes(int64_t nnz, int32_t N, int32_t b_dtype) {
  if (nnz < 1 || N < 1) return 0;
  const int64_t ranges = ceil_div64(nnz, (int64_t)1 << range_log(nnz, nnz + 1));   // the shorter ones, for any number of rows
  return (size_t)ranges * 2 * align_up((size_t)N, 8) * sizeof(float);
}

int lf_spmm_csr_act(const int64_t* indptr, const int32_t* indices, const float* data, const int32_t* order,
                    int64_t row_begin, int64_t row_end, int64_t nnz, const void* B, int32_t b_dtype, int64_t ldb,
                    const float* b_scale, void* C, int32_t c_dtype, int64_t ldc, int32_t N, const lf_epilogue* epilogue,
                    void* workspace, size_t workspace_bytes, void* stream) {
  LF_REQUIRE(N >= 1 && ldb >= N && ldc >= N && ldb < (1ll << 30) && ldc < (1ll << 30), "bad sizes");
  LF_REQUIRE(N <= (1 << 22), "more than 2^22 features");
  LF_REQUIRE(0 <= row_begin && row_begin <= row_end, "bad row range");
  LF_REQUIRE(row_end - row_begin < (1ll << 31) - 64 && nnz >= 0, "bad number of rows or entries");
  LF_REQUIRE(b_dtype == LF_DTYPE_E4M3 || is_wide_dtype(b_dtype), "unknown type of B");
  LF_REQUIRE(b_dtype != LF_DTYPE_E4M3 || b_scale, "8-bit rows need their scales");
  LF_REQUIRE(is_wide_dtype(c_dtype), "C must be float32, bfloat16 or float16");
  const lf_epilogue none = {};
  const lf_epilogue& ep = epilogue ? *epilogue : none;
  LF_REQUIRE(ep.activation >= LF_ACT_NONE && ep.activation <= LF_ACT_GELU_TANH, "unknown activation");
  LF_REQUIRE(!ep.bias || is_wide_dtype(ep.bias_dtype), "the bias must be float32, bfloat16 or float16");
  LF_REQUIRE(!ep.residual || (is_wide_dtype(ep.residual_dtype) && ep.ld_residual >= N && ep.ld_residual < (1ll << 30)), "bad residual");
  LF_REQUIRE(!ep.preact || (ep.ld_preact >= N && ep.ld_preact < (1ll << 30)), "bad leading dimension of preact");
  if (row_begin == row_end) return LF_OK;
  LF_REQUIRE(indptr && C, "null pointer argument");
  LF_REQUIRE(nnz == 0 || (indices && B), "indices or B missing");
  LF_REQUIRE(aligned(indptr, 8) && aligned(indices, 4) && aligned(data, 4) && aligned(order, 4) && aligned(b_scale, 4) && aligned_for(B, b_dtype) &&
                 aligned_for(C, c_dtype) && aligned_for(ep.bias, ep.bias_dtype) && aligned_for(ep.residual, ep.residual_dtype) && aligned_for(ep.preact, c_dtype),
             "an address is not a multiple of its type's size");
  LF_REQUIRE(!order || (data && nnz < (1ll << 31)), "order goes with data, for fewer than 2^31 entries");
  const size_t need = lf_spmm_csr_act_workspace_bytes(nnz, N, b_dtype);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return fail(LF_ERR_WORKSPACE_TOO_SMALL, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
  LF_REQUIRE((uintptr_t)workspace % 16 == 0, "the workspace must start on a 16-byte boundary");
  LF_REQUIRE(nnz == 0 || (B != C && B != ep.preact), "C and preact must not start where B does, nor lie in it at all: every row reads B");
  LF_REQUIRE(C != ep.preact, "C and preact must not be the same");
  const int lg = range_log(nnz, row_end - row_begin);
  LF_REQUIRE((nnz >> lg) < (1ll << 31) - 1, "too many entries");
  const bool vec = N % 8 == 0 && on_grid16(C, ldc, c_dtype) && (!ep.residual || on_grid16(ep.residual, ep.ld_residual, ep.residual_dtype)) &&
                   (!ep.preact || on_grid16(ep.preact, ep.ld_preact, c_dtype));
  const ActArgs a{indptr + row_begin, indices, data, order, nnz, B, b_scale, ep.bias, ep.residual, ep.preact, C, (float*)workspace,
                  (int64_t)align_up((size_t)N, 8), (uint32_t)ldb * dtype_bytes(b_dtype), (uint32_t)ep.ld_residual * dtype_bytes(ep.residual_dtype),
                  (uint32_t)ep.ld_preact * dtype_bytes(c_dtype), (uint32_t)ldc * dtype_bytes(c_dtype), (int)(row_end - row_begin), N,
                  ep.bias_dtype, ep.residual_dtype, c_dtype, ep.activation, lg, range_slack(lg), vec};
  cudaStream_t st = (cudaStream_t)stream;
  if (nnz > 0) {
    if (b_dtype == LF_DTYPE_F32) LF_CUDA_CHECK(launch_walk<LF_DTYPE_F32>(a, st));
    else if (b_dtype == LF_DTYPE_BF16) LF_CUDA_CHECK(launch_walk<LF_DTYPE_BF16>(a, st));
    else if (b_dtype == LF_DTYPE_F16) LF_CUDA_CHECK(launch_walk<LF_DTYPE_F16>(a, st));
    else LF_CUDA_CHECK(launch_walk<LF_DTYPE_E4M3>(a, st));
  }
  // few rows per block while that fills the chip: a block's long rows are done one after the other (16384 rows, 64 of them
  // with 2048 entries: 35 us with 256 rows a block, 17 with 32)
  int span = 32;
  while (span < kThreads && a.rows > (int64_t)span * kSms * 8) span *= 2;
  const int64_t blocks = ceil_div64(a.rows, span);
  LF_CUDA_CHECK(launch_dep(finish_rows_kernel, dim3((unsigned)(blocks < (1 << 16) ? blocks : 1 << 16)), kThreads, st, nnz > 0, a, span));
  return LF_OK;
}

}  // extern "C"
