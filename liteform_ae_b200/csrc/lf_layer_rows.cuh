// Walking over the rows of a CSR matrix, a warp per range of entries: what the product with an epilogue
// (lf_spmm_act.cu) and the gradient of the values (lf_spmm_act_grad.cu) share.
//
// A warp is R = 32 / G groups of G lanes; a row of B is CH pieces of 16 bytes per lane of a group.  The warp takes up to 32
// consecutive rows at a time, brings their columns and values into shared memory, sorts the rows by length and does R of
// them side by side, a group each; rows of more than 64 entries are done by all groups together.  Either way the rows of
// B come through a ring in shared memory that cp.async fills 8 KB ahead, across the rows' ends.
//
// Why sorted rows: graphs have most of their rows at a few entries and most of their entries in a few rows.  Groups that
// end their rows at different steps run the epilogue one after the other; rows of about one length end together, and
// nothing has to notice where a row ends.  2^20 power-law rows, 13.2 M entries, 128 bfloat16 features, bias, relu and
// residual (the graph below): groups that walk over entries at an even pace, finished rows in a queue, 985 us; thread blocks
// that stage row starts in the place of entries 1193; sorted rows with four gathers per group in registers instead of the ring
// 1441; the first form with the ring 624; now 555, both launches.  Figures of a choice beside others were taken when it was made.
#pragma once

#include "lf_layer.cuh"
#include "lf_spmm_group.cuh"

namespace lf {

// Entries of a warp's range: the most that still gives each SM 20 warps (it holds 17 to 19 at a time), three times
// over where there are enough, from 64 to 2048 (2^20 uniform rows, 33.5 M entries: 735 us with 1024 each, 707 with 2048; the
// graph above 620 with 512, 615 with 1024).  From 16 where most rows have no entry, since there each may take a search
// for its row (332 469 rows with 40 entries: 196 us for 64, 85 for 16; 3497 rows with 56 000, some of them long: 27 and 34).
inline int range_log(int64_t nnz, int64_t rows) {
  int lg = 11;
  while (lg > (rows > nnz ? 4 : 6) && (nnz >> lg) < kSms * 20 * (lg > 8 ? 3 : 1)) --lg;
  return lg;
}
// A row that starts in a range and ends at most so far behind its nominal end belongs to it whole; only longer ones are
// cut, at the nominal ends.  Their pieces are added up in order by a later launch.
inline int range_slack(int lg) { return lg > 7 ? 1 << (lg - 2) : 32; }
__device__ __forceinline__ bool row_is_cut(int64_t a, int64_t b, int lg, int slack) { return b > (((a >> lg) + 1) << lg) + slack; }

// Row pointers of a row range, relative to its first entry and never beyond the `nnz` the caller gave, so that what
// follows from them stays inside the arrays whatever the matrix holds.
struct RowStarts {
  const int64_t* __restrict__ indptr;   // of the first row of the range
  int64_t base, total;
  int rows;
  __device__ __forceinline__ void init(const int64_t* range_indptr, int rows_, int64_t nnz) {
    indptr = range_indptr;
    rows = rows_;
    base = __ldg(indptr);
    total = min(__ldg(indptr + rows) - base, nnz);
  }
  __device__ __forceinline__ int64_t operator()(int row) const {   // rows beyond the last start at the end
    const int64_t s = __ldg(indptr + min(row, rows)) - base;
    return s < 0 ? 0 : min(s, total);
  }
};

// The last rows that start at or before COUNT entries e[], by the whole warp: 33-ary search, a probe per lane, the searches
// side by side.
template <int COUNT>
__device__ __forceinline__ void find_rows(const RowStarts& ptr, const int64_t* e, int lane, int* row) {
  int lo[COUNT], hi[COUNT];   // start of lo <= e, answer in [lo, hi)
#pragma unroll
  for (int i = 0; i < COUNT; ++i) {
    lo[i] = 0;
    hi[i] = ptr.rows;
  }
  for (;;) {
    bool more = false;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) more |= hi[i] - lo[i] > 1;
    if (!more) break;
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const int span = hi[i] - lo[i];
      int q = lo[i] + (int)(((int64_t)(lane + 1) * span) / 33);
      if (q <= lo[i]) q = lo[i] + 1;
      const int cnt = __popc(__ballot_sync(kAllLanes, span > 1 && ptr(q) <= e[i]));   // probes are monotone
      const int qlo = __shfl_sync(kAllLanes, q, cnt > 0 ? cnt - 1 : 0), qhi = __shfl_sync(kAllLanes, q, cnt < 32 ? cnt : 31);
      if (span > 1) {
        if (cnt > 0) lo[i] = qlo;
        if (cnt < 32) hi[i] = min(qhi, hi[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < COUNT; ++i) row[i] = lo[i];
}

// Where a range begins.
struct RangeStart {
  int64_t entry;   // its first entry
  int row;         // that entry's row, where it is a cut row that started earlier; else the row before the next that starts
  bool open;       // the former
};
// The starts of the range `q` and of the one after it.
__device__ __forceinline__ void find_range(const RowStarts& ptr, int64_t q, int lg, int slack, int lane, RangeStart* out) {
  const int64_t s[2] = {q << lg, min((q + 1) << lg, ptr.total - 1)};
  int row[2];
  find_rows<2>(ptr, s, lane, row);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int64_t e = (q + i) << lg;
    const int64_t a = ptr(row[i]), b = ptr(row[i] + 1);
    if (e >= ptr.total) out[i] = {ptr.total, ptr.rows - 1, false};
    else if (a >= e) out[i] = {e, row[i] - 1, false};
    else if (row_is_cut(a, b, lg, slack)) out[i] = {e, row[i], true};
    else out[i] = {b, row[i], false};
  }
}

// ---- rows of B as they are stored -----------------------------------------------------------------------------
template <int DT> constexpr int kPerPiece = 16 / (int)sizeof(typename Type<DT>::T);   // elements in 16 bytes

// 16 bytes to floats, in pairs
template <int DT>
__device__ __forceinline__ void pairs_of(const uint4& x, uint64_t* f) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  if constexpr (DT == LF_DTYPE_F32) {
    f[0] = as_pair(w[0], w[1]);
    f[1] = as_pair(w[2], w[3]);
  } else if constexpr (DT == LF_DTYPE_BF16) {   // a bf16 is the upper half of the float with the same value
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = as_pair(w[i] << 16, w[i] & 0xffff0000u);
  } else if constexpr (DT == LF_DTYPE_F16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(w + i));
      f[i] = as_pair(__float_as_uint(v.x), __float_as_uint(v.y));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {   // e4m3 is exact in float16
      const float2 v = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i & 1))), __NV_E4M3)));
      f[i] = as_pair(__float_as_uint(v.x), __float_as_uint(v.y));
    }
  }
}

// The share of a row that a lane of a group has: CH pieces of 16 bytes, G pieces apart (features (gl + G c) VEC + i), or,
// where rows are off the 16-byte grid (CH == 0), VEC single elements (features gl + G i) behind the row's shift in the G
// aligned pieces that cover it.
template <int DT, int G, int CH>
struct Share {
  static constexpr bool kShifted = CH == 0;
  static constexpr int VEC = kPerPiece<DT>, kPieces = CH ? CH : 1, kFloats = kPieces * VEC, kPairs = kFloats / 2;
  // of a walk; where a row takes several, each starts at a multiple of eight features
  static constexpr int kFeatures = !kShifted ? G * kFloats : G == 32 ? (G - 1) * VEC / 8 * 8 : (G - 1) * VEC;
  static constexpr int kSpan = G * kFloats;   // features that the lanes have places for
  static __device__ __forceinline__ int feature(int i, int gl) { return kShifted ? gl + G * i : (gl + G * (i / VEC)) * VEC + i % VEC; }
  // the lane's share of a row in the ring, as floats; x: the lane's first piece, or the row's first feature
  static __device__ __forceinline__ void floats(const unsigned char* x, int gl, uint64_t* f) {
    if constexpr (!kShifted) {
#pragma unroll
      for (int c = 0; c < CH; ++c) pairs_of<DT>(*reinterpret_cast<const uint4*>(x + c * 512), f + c * (VEC / 2));
    } else {
      const auto* p = reinterpret_cast<const typename Type<DT>::T*>(x) + gl;   // past the row's end: what the ring holds, dropped
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i)
        f[i] = as_pair(__float_as_uint(Type<DT>::get(p[G * 2 * i])), __float_as_uint(Type<DT>::get(p[G * (2 * i + 1)])));
    }
  }
};

// Calls go(G, CH) with lanes per group and pieces per lane as constants: groups as narrow as the row, 512 bytes of wider ones
// at a time; two pieces per lane where that is no more than 16 features.  Shifted rows: CH = 0.
template <int DT, class F>
inline cudaError_t with_row_shape(bool grid16, int N, F&& go) {
#define LF_GO(G_, CH_) return go(std::integral_constant<int, G_>(), std::integral_constant<int, CH_>())
  const int64_t bytes = (int64_t)N * dtype_bytes(DT);
  if (!grid16) {
    if (bytes <= 48) LF_GO(4, 0);
    if (bytes <= 112) LF_GO(8, 0);
    if (bytes <= 240) LF_GO(16, 0);
    LF_GO(32, 0);
  }
  constexpr bool kTwo = DT != LF_DTYPE_E4M3;
  if (bytes <= 64) LF_GO(4, 1);
  if (bytes <= 128) LF_GO(8, 1);
  if constexpr (kTwo) {
    if (bytes <= 256) LF_GO(8, 2);
    LF_GO(16, 2);
  } else {
    if (bytes <= 256) LF_GO(16, 1);
    LF_GO(32, 1);
  }
#undef LF_GO
}

// BLOCKS of n neighbouring elements of a row in memory, `apart` from one block to the next, as they are stored: `left` of them
// from the first on to the row's end.  Blocks of 16 bytes and halves of them move as they are.
template <int BLOCKS, int n>
__device__ __forceinline__ void load_blocks(const char* p, int dt, int apart, int left, uint32_t* w) {
  const int bytes = dtype_bytes(dt);
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b) {
    if (b * apart >= left) break;
    const char* q = p + b * apart * bytes;
    if (dt == LF_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < n; i += 4) *reinterpret_cast<uint4*>(w + b * n + i) = __ldcs(reinterpret_cast<const uint4*>(q + i * 4));
    } else if (n == 4) {
      *reinterpret_cast<uint2*>(w + b * n) = __ldcs(reinterpret_cast<const uint2*>(q));
    } else {
#pragma unroll
      for (int i = 0; i < n; i += 8) *reinterpret_cast<uint4*>(w + b * n + i / 2) = __ldcs(reinterpret_cast<const uint4*>(q + i * 2));
    }
  }
}
// v[i] = op(v[i], the element)
template <int BLOCKS, int n, class Op>
__device__ __forceinline__ void use_blocks(const uint32_t* w, int dt, float* v, Op op) {
  if (dt == LF_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < BLOCKS * n; ++i) v[i] = op(v[i], __uint_as_float(w[i]));
  } else if (dt == LF_DTYPE_BF16) {
#pragma unroll
    for (int i = 0; i < BLOCKS * n; ++i) {
      const uint32_t h = w[i / n * n + i % n / 2];
      v[i] = op(v[i], __uint_as_float(i & 1 ? h & 0xffff0000u : h << 16));
    }
  } else {
#pragma unroll
    for (int i = 0; i < BLOCKS * n; i += 2) {
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(w + i / n * n + i % n / 2));
      v[i] = op(v[i], x.x);
      if (i + 1 < BLOCKS * n) v[i + 1] = op(v[i + 1], x.y);
    }
  }
}

// ---- the walk ---------------------------------------------------------------------------------------------------
// What a walk is made of.
struct WalkArgs {
  const int32_t* cols;     // of the row range's first entry
  const float* vals;       // same, or NULL: all ones (with order: the values of all entries)
  const int32_t* order;    // same, or NULL
  const float* scale;      // per row of B, or NULL
  const char* B;           // first feature of the walk
  uint32_t pitch;          // bytes between rows of B
  int nf;                  // features from there on, at most kFeatures
};

constexpr int kWalkThreads = 32;    // a warp: a block of two keeps its place until the slower is done (589 us on the graph above for 561)
// Blocks per SM that the registers have to allow; shared memory allows 17 to 19 with the span of the bias.  16 are four to each of
// the SM's register files, so 128 registers; 17 to 20 are five, so 96 without spills, but the compiler orders instructions for the
// number it is given.  16, 17, 18, 20: 588, 558, 560, 563 us on the graph above, in 8 bits 651, 584, 607, 613.
constexpr int kWalkBlocks = 17;
constexpr int kWindow = 256;        // entries of the rows taken at a time, rows rounded up to fours
constexpr int kShortRow = 64;       // longest row that one group does (16 / 32 / 64 / 128: 713 / 622 / 606 / 642 us on the graph above, in an earlier form)
constexpr int kAtOnce = 4;          // steps (a row of B per group) that are copied and added up together
constexpr int kRingBytes = 8192;
constexpr uint32_t kNothing = 0x80000000u;   // mark of a column whose row of B is not read

struct WalkSmem {
  unsigned char ring[kRingBytes + 16];   // shifted rows are read up to their shift past the ring's end
  __align__(16) uint32_t col[kWindow];   // or with the mark; a group's row, or its share of one, from a multiple of four on
  float val[kWindow];
  int32_t sorted[32];                    // rows of the window that have entries, the shortest first: number, place, size in fours
};

// Copies the lane's pieces of a row of B into the ring (PIECES of 16 bytes, `STRIDE` apart in the row), those that are
// `on`, or zeros for an entry that gathers nothing: the sums need not look, since what they multiply with its value 0 is 0.
// Predicates and immediate offsets, since this is a third of what the walk executes.
template <int PIECES, int STRIDE, int TO>
__device__ __forceinline__ void copy_row(uint32_t dst, const void* src, uint32_t col, int on1, int on2) {
  if constexpr (PIECES == 2) {
    asm volatile(
        "{\n .reg .pred z, a, b;\n setp.lt.s32 z, %2, 0;\n setp.ne.s32 a, %3, 0;\n setp.ne.s32 b, %4, 0;\n"
        " @a cp.async.cg.shared.global [%0 + %6], [%1], 16, z;\n @b cp.async.cg.shared.global [%0 + %7], [%1 + %5], 16, z;\n}" ::"r"(dst),
        "l"(src), "r"((int)col), "r"(on1), "r"(on2), "n"(STRIDE), "n"(TO), "n"(TO + 512)
        : "memory");
  } else {
    asm volatile(
        "{\n .reg .pred z, a;\n setp.lt.s32 z, %2, 0;\n setp.ne.s32 a, %3, 0;\n @a cp.async.cg.shared.global [%0 + %4], [%1], 16, z;\n}" ::"r"(dst),
        "l"(src), "r"((int)col), "r"(on1), "n"(TO)
        : "memory");
  }
}

// A walk over the rows of one range.  IND: there may be scales or an order.  `Work` has
//   coming(row)              a row of the window, by one of its lanes
//   begin(row, whole, piece, at, end)   every group begins a row (row < 0: the group has none), or, `whole`, all groups the
//                            same one; its entries are at places below `end`, and the one at place p is entry at + p (both
//                            only where Work::kPlaces)
//   ahead(row)               the group's next row of the window, or -1 (only where Work::kPlaces)
//   step(val, x)             an entry of the row (one that the group does not have has the value 0): x is the lane's share of
//                            its row of B, as Share::floats takes it
//   steps_done(k, in)        after four steps: k is the place of the first of them in the window; in: they are the group's
//   end(row, whole, piece)   the row is done; piece: -1 the whole row, 0 a piece of one that started in an earlier range,
//                            1 of one that goes on in the next
// Each is called at one place: what the walk executes has to stay in the instruction cache (with the epilogue at several
// places and unrolled for every type, 114 KB a kernel, 4.8 of 12 cycles of a warp went into waiting for instructions).
template <int DT, int G, int CH, bool IND, class Work>
struct RowWalk {
  using S = Share<DT, G, CH>;
  static constexpr int R = 32 / G, U = kAtOnce, kStep = S::kPieces * 512, kBatch = U * kStep, kBatches = kRingBytes / kBatch;
  const WalkArgs& a;
  const RowStarts& ptr;
  WalkSmem& sm;
  Work& work;
  int lane, g, gl;
  const char* Bl;
  uint32_t ring_s;
  bool in1, in2;
  int over, in_slot, out_slot;

  // A group's row (or -1) and its places in the window, in fours; steps: the longest row's of the groups.
  struct Batch {
    int row, from, own, steps, end;
    int64_t at;
    __device__ __forceinline__ bool has(int k) const { return k < own; }
    __device__ __forceinline__ int place(int k) const { return has(k) ? from + k * U : 0; }
  };
  __device__ __forceinline__ RowWalk(const WalkArgs& a_, const RowStarts& p_, WalkSmem& s_, Work& w_) : a(a_), ptr(p_), sm(s_), work(w_) {
    lane = threadIdx.x & 31;
    g = lane / G;
    gl = lane % G;
    Bl = a.B + (S::kShifted ? 0 : gl * 16);
    in1 = S::kShifted || gl * S::VEC < a.nf;
    in2 = CH == 2 && (gl + G) * S::VEC < a.nf;
    over = S::kShifted ? gl * 16 - a.nf * (16 / S::VEC) : 0;   // piece gl is needed while the shift is larger than this
    ring_s = (uint32_t)__cvta_generic_to_shared(sm.ring) + lane * 16;
    in_slot = out_slot = 0;
  }

  // Entry e + index(i) of the matrix (index < 0: none) to place i of the window, for i < places.  All loads of a kind are on
  // their way together.
  template <class Index>
  __device__ __forceinline__ void stage(int64_t e, int places, Index index) {
    constexpr int T = kWindow / 32;
    int at[T];
    uint32_t c[T];
    float v[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
      at[t] = t * 32 < places ? index(t * 32 + lane) : -1;
      c[t] = kNothing;
      v[t] = 0.f;
      if (at[t] >= 0) {
        c[t] = (uint32_t)__ldcs(a.cols + e + at[t]);
        if (IND && a.order) at[t] = __ldcs(a.order + e + at[t]);
        else v[t] = a.vals ? __ldcs(a.vals + e + at[t]) : 1.f;
      }
    }
    if constexpr (IND) {
      if (a.order) {
#pragma unroll
        for (int t = 0; t < T; ++t)
          if (at[t] >= 0) v[t] = __ldg(a.vals + at[t]);
      }
      if (a.scale) {   // (as copies beside the rows of B, multiplied when they are used: 633 -> 651 us in 8 bits, more instructions)
        float s[T];
#pragma unroll
        for (int t = 0; t < T; ++t) s[t] = v[t] != 0.f ? __ldg(a.scale + c[t]) : 0.f;
#pragma unroll
        for (int t = 0; t < T; ++t) at[t] = v[t] != 0.f, v[t] = v[t] != 0.f ? v[t] * s[t] : 0.f;
      } else {
#pragma unroll
        for (int t = 0; t < T; ++t) at[t] = v[t] != 0.f;
      }
    }
#pragma unroll
    for (int t = 0; t < T; ++t) {
      if (t * 32 < places) {
        const bool gathers = IND ? at[t] > 0 : v[t] != 0.f;   // an entry of value 0 reads nothing of B, nor its scale
        sm.col[t * 32 + lane] = gathers ? c[t] : kNothing;
        sm.val[t * 32 + lane] = v[t];
      }
    }
  }
  __device__ __forceinline__ int shift(uint32_t c) const { return (int)(((uint32_t)reinterpret_cast<uintptr_t>(a.B) + (c & ~kNothing) * a.pitch) & 15u); }
  template <int STEP>
  __device__ __forceinline__ void issue_step(uint32_t dst, uint32_t c, int on1, int on2) {
    const char* src = reinterpret_cast<const char*>(row_of_b(Bl, c & ~kNothing, a.pitch));
    if constexpr (S::kShifted) {
      on1 = on1 && shift(c) > over;
      src = reinterpret_cast<const char*>(reinterpret_cast<uint64_t>(src) & ~15ull) + gl * 16;
    }
    copy_row<S::kPieces, G * 16, STEP * kStep>(dst, src, c, on1, on2);
  }
  // starts the copies of the window's places k .. k + 3, if the group has them
  __device__ __forceinline__ void issue(int k, bool in) {
    const uint32_t dst = ring_s + in_slot * kBatch;
    const uint4 c4 = *reinterpret_cast<const uint4*>(sm.col + k);
    const uint32_t c[U] = {c4.x, c4.y, c4.z, c4.w};
    const int on1 = in && in1, on2 = in && in2;
    issue_step<0>(dst, c[0], on1, on2);
    issue_step<1>(dst, c[1], on1, on2);
    issue_step<2>(dst, c[2], on1, on2);
    issue_step<3>(dst, c[3], on1, on2);
    in_slot = in_slot + 1 == kBatches ? 0 : in_slot + 1;
  }
  // their sums
  __device__ __forceinline__ void take(int k, bool in) {
    const float4 v4 = *reinterpret_cast<const float4*>(sm.val + k);
    const float v[U] = {v4.x, v4.y, v4.z, v4.w};
    int h[U] = {0, 0, 0, 0};
    if constexpr (S::kShifted) {
      const uint4 c4 = *reinterpret_cast<const uint4*>(sm.col + k);
      h[0] = shift(c4.x); h[1] = shift(c4.y); h[2] = shift(c4.z); h[3] = shift(c4.w);
    }
    cp_async_wait<kBatches - 1>();            // the copies of these steps have landed
    if constexpr (S::kShifted) __syncwarp();  // lanes read words that other lanes copied
    const unsigned char* x = sm.ring + out_slot * kBatch + (S::kShifted ? g * G * 16 : lane * 16);
    if (in) {
#pragma unroll
      for (int u = 0; u < U; ++u) work.step(v[u], x + u * kStep + h[u]);
    }
    if constexpr (S::kShifted) __syncwarp();  // every lane has read before the place is refilled
    out_slot = out_slot + 1 == kBatches ? 0 : out_slot + 1;
  }

  __device__ __forceinline__ void range(int64_t q, int lg, int slack) {
    RangeStart at[2];
    find_range(ptr, q, lg, slack, lane, at);
    int64_t e = at[0].entry;
    const int64_t end = at[1].entry;
    int row = at[0].row, piece = 0;
    int64_t left = 0;   // of a row that all groups do, from e on
    bool begun = false, skipped = false;
    if (at[0].open) left = min(ptr(row + 1), end) - e;
    else ++row;
    int64_t ends = ptr(row + lane + 1);   // where row + lane ends
    while (e < end && row < ptr.rows) {
      int64_t after;
      int n, held = R, length = 0, size = 0, from = 0, first = 0, places, share = 0, rows = 0;   // share: of a group, of a row that all do
      if (left <= 0) {
        const int64_t before = __shfl_up_sync(kAllLanes, ends, 1), starts = lane == 0 ? e : before;
        const bool goes_on = starts < end && ends > end;
        length = starts < end ? (int)min((int64_t)0x3fffffff, min(ends, end) - starts) : 0;
        const unsigned longs = __ballot_sync(kAllLanes, length > kShortRow || goes_on || length < 0);
        if (longs & 1u) {   // the first row is one for all groups
          left = __shfl_sync(kAllLanes, length, 0);
          piece = __shfl_sync(kAllLanes, goes_on, 0) ? 1 : -1;
          begun = false;
          if (left <= 0) break;   // (only where row pointers do not ascend)
          continue;
        }
        // rows up to the next long one, as many as the window holds
        const int upto = longs ? __ffs(longs) - 1 : 32;
        size = lane < upto ? (length + U - 1) / U : kWindow;
        const int sum = warp_inclusive_scan(size);
        from = (sum - size) * U;
        const bool in = sum * U <= kWindow && starts >= e;
        rows = __popc(__ballot_sync(kAllLanes, in));   // monotone
        if (!in) size = 0;
        places = __shfl_sync(kAllLanes, sum, max(rows - 1, 0)) * U;
        n = rows > 0 ? (int)min((int64_t)kWindow, __shfl_sync(kAllLanes, min(ends, end), rows - 1) - e) : 0;
        if (n <= 0 || places > kWindow) {   // rows without entries: on to the row of the next entry
          if (skipped) break;   // (only where row pointers do not ascend)
          find_rows<1>(ptr, &e, lane, &row);
          ends = ptr(row + lane + 1);
          skipped = true;
          continue;
        }
        // by length, in fours
        held = 0;
        int place = 0;
#pragma unroll 1
        for (int c = 1; c <= kShortRow / U; ++c) {
          const unsigned m = __ballot_sync(kAllLanes, size == c);
          if (size == c) place = held + __popc(m & ((1u << lane) - 1u));
          held += __popc(m);
        }
        __syncwarp();
        if (size > 0) {
          sm.sorted[place] = lane | from << 8 | size << 20;
          work.coming(row + lane);
        }
        after = ptr(row + rows + lane + 1);
        first = (int)(starts - e);
      } else {
        n = length = (int)min((int64_t)kWindow, left);
        after = ptr(row + lane + 2);
        share = (n + R * U - 1) / (R * U) * U;
        places = R * share;
        rows = 1;
        __syncwarp();
      }
      stage(e, places, [&](int i) {   // place i is of the last row that starts at or before it
        if (left > 0 || places == n) return i < n ? i : -1;   // (no row was rounded up)
        int of = 0;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1)
          if (__shfl_sync(kAllLanes, from, (of + d) & 31) <= i && of + d < rows) of += d;
        const int k = i - __shfl_sync(kAllLanes, from, of), f = __shfl_sync(kAllLanes, first, of);
        return k < __shfl_sync(kAllLanes, length, of) && i < places ? f + k : -1;
      });
      skipped = false;
      const bool whole = left > 0, closes = left <= kWindow;   // closes: nothing of the row is left after this window
      __syncwarp();
      // Side by side: every group its own of the sorted rows from p on, or its share of the one row.
      auto batch = [&](int p) {
        Batch b;
        if (whole) {
          b = {row, g * share, share / U, share / U, n, e};
        } else {
          const int mine = p + g < held ? sm.sorted[p + g] : 0;
          b.own = mine >> 20;
          b.row = b.own > 0 ? row + (mine & 31) : -1;
          b.from = (mine >> 8) & 0xfff;
          b.steps = sm.sorted[min(p + R, held) - 1] >> 20;
          if constexpr (Work::kPlaces) {
            b.end = b.from + __shfl_sync(kAllLanes, length, mine & 31);
            b.at = e + __shfl_sync(kAllLanes, first, mine & 31) - b.from;
          }
        }
        return b;
      };
      // the copies run kBatches fours ahead of the sums, through the same rows
      int pa = 0, ka = 0;
      Batch ahead = batch(0);
      auto next = [&]() {
        if (pa < held) {
          issue(ahead.place(ka), ahead.has(ka));
          if (++ka == ahead.steps) {
            ka = 0;
            pa += R;
            if (pa < held) ahead = batch(pa);
          }
        }
        cp_async_commit();
      };
#pragma unroll 1
      for (int t = 0; t < kBatches; ++t) next();
#pragma unroll 1
      for (int p = 0; p < held; p += R) {
        const Batch now = batch(p);
        if (!whole || !begun || Work::kPlaces) work.begin(now.row, whole, piece, now.at, now.end);
        if constexpr (Work::kPlaces) work.ahead(!whole && p + R + g < held ? row + (sm.sorted[p + R + g] & 31) : -1);
#pragma unroll 1
        for (int k = 0; k < now.steps; ++k) {
          take(now.place(k), now.has(k));
          work.steps_done(now.place(k), now.has(k));
          next();
        }
        if (!whole || closes) work.end(now.row, whole, piece);
      }
      e += n;
      if (whole) {
        left -= n;
        begun = true;
        if (left > 0) continue;
        if (piece == 1) break;
        rows = 1;
      }
      row += rows;
      ends = after;
    }
  }
};

}  // namespace lf
