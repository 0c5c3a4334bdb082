// C ABI: the end of a block whose partial outputs lie on the members of a team, and its gradient
// (rsm_norm_to_all, rsm_norm_to_all_grad; no counterpart in the reference).
//
// With s the members' sum of a row, C its length, r(v) = 1 / sqrt(mean(v^2) + eps) and o the weight
// offset:
//   z  = s r(s) (o + w_post)   (RSM_NORM_POST; z = s otherwise)
//   x' = a x + b g z           x the residual stream, a and b its and the block's scale, g the gate
//   h  = x' r(x') (o + w_pre)  the next block's input, on every member
// and backwards, with dh the members' sum of the gradients of h and n = x' r(x'), u = s r(s):
//   t  = dh (o + w_pre)        D = dx' + r(x') (t - n mean(t n))      dw_pre = sum_rows dh n
//   dx = a D                   f = b D g       dg = sum_rows b D z    dw_post = sum_rows f u
//   ds = r(s) (q - u mean(q u)), q = f (o + w_post)   (RSM_NORM_POST; ds = f otherwise)
//
// Sums, means and everything between a load and a store are 32-bit floats; every output is rounded
// to its type once.  Members are summed in ascending order, so every run gives the same bits.
#include <cfloat>
#include <cmath>

#include "roc_shmem.hpp"
#include "rocshmem_device/rows.hpp"
#include "rows_common.hpp"

using namespace rocshmem;
using namespace rocshmem::detail;

namespace {

constexpr int kMaxCols = 16384;

// What both kernels know of a call.  Pointers are the first member's copies, `step` bytes lead to
// the next member's; row strides are in elements.
struct NormShape {
  int rows, cols, members, share;   // row i is held by member i / share (its owner)
  int rows_per_gate;
  int64_t step;
  int64_t partial_ld, residual_ld, normed_ld;
  float eps, inv_cols, residual_scale, block_scale;
  float pre_offset, post_offset;    // what is added to the weights: weight_offset, or 1 where there are none
  bool post, replicated;
};

struct NormForward {
  NormShape s;
  const char *source, *residual, *pre_weight, *post_weight, *gate;
  char *residual_out, *normed, *total;
};

struct NormBackward {
  NormShape s;
  const char *grad_normed, *residual_out, *total, *grad_residual_out, *pre_weight, *post_weight, *gate;
  char *grad_source, *grad_residual, *grad_gate;
  float *part_pre, *part_post, *part_gate;   // [units][part_ld], null where nobody asks for them
  int part_ld;
  // A unit (the lanes that hold a row) walks rows of its own.  `direct`: rows_per_unit in a row, whole
  // gate groups; otherwise units_per_gate units share a group and each takes every units_per_gate-th
  // row of it, so that all units together sweep one compact window of every array.
  int units, units_per_gate, rows_per_unit;
  bool direct;
};

template <typename T>
__device__ __forceinline__ const T *row_at(const char *base, int64_t bytes, int64_t row, int64_t ld, int col) {
  return reinterpret_cast<const T *>(base + bytes) + row * ld + col;
}
template <typename T>
__device__ __forceinline__ T *row_at(char *base, int64_t bytes, int64_t row, int64_t ld, int col) {
  return reinterpret_cast<T *>(base + bytes) + row * ld + col;
}

// How a row ends (kEnd).  kWhole: with a whole vector.  kShifted: inside one; the lane that holds the end
// moves back to the row's last whole vector and makes some elements that its neighbour makes too, to
// the same bits - rows are loaded, and stored, without a question - and leaves them out of sums over
// the row.  kNarrow: rows shorter than a vector, element by element.
enum RowEnd { kWhole = 0, kShifted = 1, kNarrow = 2 };

// First column of a lane's vector v, kept inside the row.
template <typename T, int kLanes, int kEnd>
__device__ __forceinline__ int column(int cols, int lane, int v) {
  const int c = (v * kLanes + lane) * kRowVec<T>;
  return kEnd == kShifted && c < cols && c > cols - kRowVec<T> ? cols - kRowVec<T> : c;
}
// What a lane's element e of vector v counts in a sum over the row: its value, or 0 where the
// neighbour counts it.  Every factor that may be infinite goes through here: inf * 0 is NaN.
template <typename T, int kLanes, int kEnd>
__device__ __forceinline__ float counted(int cols, int lane, int v, int e, float value) {
  if constexpr (kEnd != kShifted) return value;
  const int c = (v * kLanes + lane) * kRowVec<T>;
  return column<T, kLanes, kEnd>(cols, lane, v) + e >= c ? value : 0.f;
}

constexpr int kFoldDepth = 8;   // vectors of a lane, of several members, whose loads are in flight together

// Sum over the members of one row's elements that this lane holds.
template <typename T, int kLanes, int NV, int kEnd, bool kNt, int kAtOnce = kFoldDepth>
__device__ __forceinline__ void fold_members(const NormShape &s, int members, const char *base, int64_t row, int64_t ld,
                                             int lane, float (&acc)[NV][kRowVec<T>]) {
  constexpr int V = kRowVec<T>;
  constexpr int kDepth = kAtOnce / NV < 1 ? 1 : kAtOnce / NV;
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[v][e] = 0.f;
  for (int m = 0; m < members; m += kDepth) {
    u32x4 raw[kDepth][NV];
#pragma unroll
    for (int k = 0; k < kDepth; ++k) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = column<T, kLanes, kEnd>(s.cols, lane, v);
        raw[k][v] = u32x4{0u, 0u, 0u, 0u};
        if (m + k < members) raw[k][v] = row_load<T, kEnd == kNarrow, kNt>(row_at<T>(base, (m + k) * s.step, row, ld, c), s.cols - c);
      }
    }
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[v][e] += row_get<T>(raw[k][v], e);
  }
}

template <typename T, int kLanes, int NV, int kEnd, bool kNt = false>
__device__ __forceinline__ void load_row(const T *p, int cols, int lane, u32x4 (&raw)[NV]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = column<T, kLanes, kEnd>(cols, lane, v);
    raw[v] = row_load<T, kEnd == kNarrow, kNt>(p + c, cols - c);
  }
}

// A row that need not be there: elsewhere its elements have the bits `bits` stand for (0, or kOnes), so
// that the arithmetic behind it asks no questions.
template <typename T>
constexpr uint32_t kOnes = sizeof(T) == 4 ? 0x3f800000u : 0x3f803f80u;
template <typename T, int kLanes, int NV, int kEnd, bool kNt = false>
__device__ __forceinline__ void load_row_or(bool there, uint32_t bits, const T *p, int cols, int lane, u32x4 (&raw)[NV]) {
  if (there) {
    load_row<T, kLanes, NV, kEnd, kNt>(p, cols, lane, raw);
  } else {
#pragma unroll
    for (int v = 0; v < NV; ++v) raw[v] = u32x4{bits, bits, bits, bits};
  }
}

// Ends the life of everything derived from raw vectors: what follows unpacks them again.  Without it
// the compiler carries the floats of bfloat16 rows, twice the registers, from one sum over the row to
// what depends on it.
template <int NV>
__device__ __forceinline__ void keep_packed(u32x4 (&raw)[NV]) {
#pragma unroll
  for (int v = 0; v < NV; ++v) __asm__ volatile("" : "+v"(raw[v]));
}

// The row to `copies` members, `step` bytes apart.
template <typename T, int kLanes, int NV, int kEnd>
__device__ __forceinline__ void store_row(T *p, int64_t step, int copies, int cols, int lane,
                                          const float (&f)[NV][kRowVec<T>]) {
  u32x4 raw[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) raw[v] = row_pack<T>(f[v]);
  for (int m = 0; m < copies; ++m) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = column<T, kLanes, kEnd>(cols, lane, v);
      row_store<T, kEnd == kNarrow, true>(bytes_on(p, m * step) + c, cols - c, raw[v]);
    }
  }
}

template <int kLanes>
constexpr int kWgLanes = kLanes < 256 ? 256 : kLanes;

// A row stays in the registers of its lanes from the loads to the last store: every operand crosses memory
// once, which is what bounds the kernel (8192 x 4096 bf16 over 8 members, sums kept: 1.28 GB in 205 to 225 us
// by process, 5.7-6.2 TB/s; the library's best copy reaches 6.1-6.7).  One row to a workgroup: two to four
// rows, other orders of rows over the chip, and slots on the clock for loads and for stores gave no more.
// One row of 8192 takes 5.1 us, of which an empty launch is about 4.
template <typename T, int kLanes, int NV, int kEnd, bool kNt>
__global__ void __launch_bounds__(kWgLanes<kLanes>) norm_kernel(NormForward p) {
  constexpr int V = kRowVec<T>;
  __shared__ float slots[2 * (kWgLanes<kLanes> / 64)];
  int turn = 0;
  const NormShape &s = p.s;
  const int lane = threadIdx.x % kLanes;
  const int row = uniform(static_cast<int>(blockIdx.x * (kWgLanes<kLanes> / kLanes) + threadIdx.x / kLanes));
  if (row >= s.rows) return;   // a whole wave of a workgroup of one-wave rows; no barrier follows
  const int owner = uniform(row / s.share);
  const int64_t home = owner * s.step;
  const int64_t held = s.replicated ? row : row - owner * s.share;

  u32x4 x[NV], wpre[NV], wpost[NV], gate[NV];
  load_row<T, kLanes, NV, kEnd, kNt>(row_at<T>(p.residual, home, held, s.residual_ld, 0), s.cols, lane, x);
  load_row_or<T, kLanes, NV, kEnd>(p.pre_weight, 0u, row_at<T>(p.pre_weight, home, 0, 0, 0), s.cols, lane, wpre);
  load_row_or<T, kLanes, NV, kEnd>(p.post_weight, 0u, row_at<T>(p.post_weight, home, 0, 0, 0), s.cols, lane, wpost);
  load_row_or<T, kLanes, NV, kEnd>(p.gate, kOnes<T>, row_at<T>(p.gate, home, row / s.rows_per_gate, s.cols, 0), s.cols,
                                    lane, gate);

  float acc[NV][V];
  fold_members<T, kLanes, NV, kEnd, kNt>(s, s.members, p.source, row, s.partial_ld, lane, acc);
  if (p.total) store_row<T, kLanes, NV, kEnd>(row_at<T>(p.total, home, row - owner * s.share, s.cols, 0), 0, 1, s.cols, lane, acc);

  if (s.post) {
    float ss[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float sc = counted<T, kLanes, kEnd>(s.cols, lane, v, e, acc[v][e]);
        ss[0] = fmaf(sc, sc, ss[0]);
      }
    row_sums<kLanes>(ss, slots, turn);
    const float r = rsqrtf(fmaf(ss[0], s.inv_cols, s.eps));
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) acc[v][e] *= r * (s.post_offset + row_get<T>(wpost[v], e));
  }
  float ss[1] = {0.f};
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float z = acc[v][e] * row_get<T>(gate[v], e);
      acc[v][e] = fmaf(s.residual_scale, row_get<T>(x[v], e), s.block_scale * z);
      const float xc = counted<T, kLanes, kEnd>(s.cols, lane, v, e, acc[v][e]);
      ss[0] = fmaf(xc, xc, ss[0]);
    }
  // The row may be stored over what a shifted lane of another wave still loads.
  if (kEnd == kShifted && kLanes > 64 && !s.post) __syncthreads();
  store_row<T, kLanes, NV, kEnd>(row_at<T>(p.residual_out, s.replicated ? 0 : home, held, s.residual_ld, 0), s.step,
                                 s.replicated ? s.members : 1, s.cols, lane, acc);
  if (!p.normed) return;
  row_sums<kLanes>(ss, slots, turn);
  const float r = rsqrtf(fmaf(ss[0], s.inv_cols, s.eps));
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < V; ++e) acc[v][e] *= r * (s.pre_offset + row_get<T>(wpre[v], e));
  store_row<T, kLanes, NV, kEnd>(row_at<T>(p.normed, 0, row, s.normed_ld, 0), s.step, s.members, s.cols, lane, acc);
}

// Four floats of row `at` of an array of sums, from column c on if the row has it.  part_ld is a multiple
// of 4, so that a narrow row's four stay inside the array.
__device__ __forceinline__ void store_part(float *part, int64_t at, int ld, int cols, int c, float4 f) {
  if (c < cols) row_store<float, false>(part + at * ld + c, 4, row_pack<float>({f.x, f.y, f.z, f.w}));
}

// Every operand crosses memory once here too (8192 x 4096 bf16 over 8 members: 1.34 GB in 230 to 251 us, and
// part_sums_kernel's 7); what the rows leave for the sums over rows stays on the compute unit until its
// rows are done (25 MB of it in all there).
template <typename T, int kLanes, int NV, int kEnd, bool kNt>
__global__ void __launch_bounds__(kWgLanes<kLanes>) norm_grad_kernel(NormBackward p) {
  constexpr int V = kRowVec<T>;
  __shared__ float slots[2 * 3 * (kWgLanes<kLanes> / 64)];
  __shared__ float slots1[2 * (kWgLanes<kLanes> / 64)];
  // The sums of the two weights' gradients over the unit's rows, each lane's own: in LDS, since in
  // registers they would halve the workgroups of a compute unit or, at 1024 lanes, spill.
  __shared__ float4 sums_of[2][NV * V / 4][kWgLanes<kLanes>];
  int turn = 0, turn1 = 0;
  const NormShape &s = p.s;
  const int lane = threadIdx.x % kLanes;
  const int unit = uniform(static_cast<int>(blockIdx.x * (kWgLanes<kLanes> / kLanes) + threadIdx.x / kLanes));
  if (unit >= p.units) return;   // as in norm_kernel
  int64_t first, last, step = 1;
  if (p.direct) {
    first = static_cast<int64_t>(unit) * p.rows_per_unit;
    last = first + p.rows_per_unit;
  } else {
    const int64_t group = unit / p.units_per_gate;
    first = group * s.rows_per_gate + unit % p.units_per_gate;
    last = (group + 1) * s.rows_per_gate;
    step = p.units_per_gate;
  }
  if (last > s.rows) last = s.rows;

  float sum_gate[NV][V];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int e = 0; e < V; ++e) sum_gate[v][e] = 0.f;
#pragma unroll
  for (int k = 0; k < NV * V / 4; ++k) sums_of[0][k][threadIdx.x] = sums_of[1][k][threadIdx.x] = float4{0.f, 0.f, 0.f, 0.f};
  // The weights' copies on the first member serve every row of the unit.  Rows of 16 elements to a lane
  // (kTight) leave no registers for them: those loads are made again for every row, where the values are
  // used, as is the gate's.
  constexpr bool kTight = NV * V >= 16;
  u32x4 wpre[NV], wpost[NV], g[NV];
  auto load_pre = [&] {
    load_row_or<T, kLanes, NV, kEnd>(p.pre_weight, 0u, row_at<T>(p.pre_weight, 0, 0, 0, 0), s.cols, lane, wpre);
  };
  auto load_post = [&] {
    load_row_or<T, kLanes, NV, kEnd>(p.post_weight, 0u, row_at<T>(p.post_weight, 0, 0, 0, 0), s.cols, lane, wpost);
  };
  if constexpr (!kTight) {
    load_pre();
    load_post();
  }

  auto add_to = [](auto &of, int v, const float (&f)[V]) {
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
      float4 &sum = of[v * (V / 4) + k][threadIdx.x];
      sum = float4{sum.x + f[4 * k], sum.y + f[4 * k + 1], sum.z + f[4 * k + 2], sum.w + f[4 * k + 3]};
    }
  };
  for (int64_t row = first; row < last; row += step) {
    const int owner = uniform(static_cast<int>(row) / s.share);
    const int64_t home = owner * s.step, shared = row - static_cast<int64_t>(owner) * s.share;
    const int64_t held = s.replicated ? row : shared;
    const int gate_row = uniform(static_cast<int>(row) / s.rows_per_gate);
    u32x4 x[NV], tot[NV], din[NV];
    load_row_or<T, kLanes, NV, kEnd, kNt>(p.grad_normed, 0u, row_at<T>(p.residual_out, home, held, s.residual_ld, 0), s.cols,
                                           lane, x);
    load_row_or<T, kLanes, NV, kEnd, kNt>(p.total, 0u, row_at<T>(p.total, home, shared, s.cols, 0), s.cols, lane, tot);
    load_row_or<T, kLanes, NV, kEnd, kNt>(p.grad_residual_out, 0u,
                                           row_at<T>(p.grad_residual_out, home, held, s.residual_ld, 0), s.cols, lane, din);
    auto load_gate = [&] {
      load_row_or<T, kLanes, NV, kEnd>(p.gate, kOnes<T>, row_at<T>(p.gate, home, gate_row, s.cols, 0), s.cols, lane, g);
    };
    if constexpr (!kTight) load_gate();
    float d[NV][V];
    if constexpr (kTight) load_pre();
    fold_members<T, kLanes, NV, kEnd, kNt, kTight ? 4 : kFoldDepth>(s, p.grad_normed ? s.members : 0, p.grad_normed, row,
                                                                    s.normed_ld, lane, d);
    // sum x'^2, sum t x' and sum s^2 in one go: the second mean is r(x') times a plain sum
    float sums[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float xc = counted<T, kLanes, kEnd>(s.cols, lane, v, e, row_get<T>(x[v], e));
        const float sc = counted<T, kLanes, kEnd>(s.cols, lane, v, e, row_get<T>(tot[v], e));
        const float t = d[v][e] * (s.pre_offset + row_get<T>(wpre[v], e));
        sums[0] = fmaf(xc, xc, sums[0]);
        sums[1] = fmaf(counted<T, kLanes, kEnd>(s.cols, lane, v, e, t), xc, sums[1]);
        sums[2] = fmaf(sc, sc, sums[2]);
      }
    row_sums<kLanes>(sums, slots, turn);
    keep_packed(x);
    keep_packed(tot);
    keep_packed(din);
    if constexpr (kTight) keep_packed(wpre);
    const float r2 = rsqrtf(fmaf(sums[0], s.inv_cols, s.eps));
    const float mean_tn = sums[1] * r2 * s.inv_cols;
    const float r1 = s.post ? rsqrtf(fmaf(sums[2], s.inv_cols, s.eps)) : 1.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float to_pre[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float n = row_get<T>(x[v], e) * r2;
        const float t = d[v][e] * (s.pre_offset + row_get<T>(wpre[v], e));
        to_pre[e] = d[v][e] * n;
        d[v][e] = fmaf(r2, fmaf(-n, mean_tn, t), row_get<T>(din[v], e));
      }
      if (p.part_pre) add_to(sums_of[0], v, to_pre);
    }
    if (p.grad_residual) {
      float dx[NV][V];
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < V; ++e) dx[v][e] = s.residual_scale * d[v][e];
      store_row<T, kLanes, NV, kEnd>(row_at<T>(p.grad_residual, s.replicated ? 0 : home, held, s.residual_ld, 0), s.step,
                                      s.replicated ? s.members : 1, s.cols, lane, dx);
    }
    // from here on d is f, and then q
    if constexpr (kTight) {
      load_gate();
      load_post();
    }
    float qs[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float to_post[V];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float w = s.post_offset + row_get<T>(wpost[v], e), u = row_get<T>(tot[v], e) * r1;
        float f = s.block_scale * d[v][e];
        sum_gate[v][e] = fmaf(f, u * w, sum_gate[v][e]);
        f *= row_get<T>(g[v], e);
        to_post[e] = f * u;
        f *= w;
        qs[0] = fmaf(counted<T, kLanes, kEnd>(s.cols, lane, v, e, f), counted<T, kLanes, kEnd>(s.cols, lane, v, e, u), qs[0]);
        d[v][e] = f;
      }
      if (p.part_post) add_to(sums_of[1], v, to_post);
    }
    if (s.post) {
      row_sums<kLanes>(qs, slots1, turn1);
      keep_packed(tot);
      const float mean_qu = qs[0] * s.inv_cols;
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < V; ++e) d[v][e] = r1 * fmaf(-mean_qu * r1, row_get<T>(tot[v], e), d[v][e]);
    }
    store_row<T, kLanes, NV, kEnd>(row_at<T>(p.grad_source, 0, row, s.partial_ld, 0), s.step, s.members, s.cols, lane, d);
    if (p.direct && p.grad_gate && (row + 1 == last || (row + 1) % s.rows_per_gate == 0)) {
      for (int m = 0; m < s.members; ++m) {
        float *out = reinterpret_cast<float *>(p.grad_gate + m * s.step) + static_cast<int64_t>(gate_row) * s.cols;
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int k = 0; k < V; k += 4) {
            const int c = column<T, kLanes, kEnd>(s.cols, lane, v) + k;
            row_store<float, kEnd == kNarrow, true>(out + c, s.cols - c, row_pack<float>({sum_gate[v][k], sum_gate[v][k + 1], sum_gate[v][k + 2], sum_gate[v][k + 3]}));
          }
      }
#pragma unroll
      for (int v = 0; v < NV; ++v)
#pragma unroll
        for (int e = 0; e < V; ++e) sum_gate[v][e] = 0.f;
    }
  }
  auto leave = [&](float *part, auto of) {
    if (!part) return;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int k = 0; k < V; k += 4)
        store_part(part, unit, p.part_ld, s.cols, column<T, kLanes, kEnd>(s.cols, lane, v) + k, of(v, k));
  };
  leave(p.part_pre, [&](int v, int k) { return sums_of[0][(v * V + k) / 4][threadIdx.x]; });
  leave(p.part_post, [&](int v, int k) { return sums_of[1][(v * V + k) / 4][threadIdx.x]; });
  leave(p.part_gate, [&](int v, int k) { return float4{sum_gate[v][k], sum_gate[v][k + 1], sum_gate[v][k + 2], sum_gate[v][k + 3]}; });
}

// The units' sums, added up in a fixed order: workgroup (x, y) makes columns 32 x .. 32 x + 31 of sum y
// (0: pre_weight, 1: post_weight, then the gate rows) and writes them to every member.  32 columns, so
// that two sums of 4096 columns already make 256 workgroups; 128 lanes share a column's units, which are
// up to some thousand.
constexpr int kSumQuads = 8, kSumRanks = 128, kSumFold = 16;
struct PartSums {
  const float *part_pre, *part_post, *part_gate;
  char *grad_pre, *grad_post, *grad_gate;
  int units, units_per_gate, part_ld, cols, members;
  int64_t step;
};

__global__ void __launch_bounds__(kSumQuads * kSumRanks) part_sums_kernel(PartSums p) {
  __shared__ float4 sums[kSumRanks][kSumQuads];
  const int y = blockIdx.y;
  const float *part = y == 0 ? p.part_pre : y == 1 ? p.part_post : p.part_gate;
  char *out = y == 0 ? p.grad_pre : y == 1 ? p.grad_post : p.grad_gate;
  if (!out) return;
  const int quad = threadIdx.x % kSumQuads, rank = threadIdx.x / kSumQuads;
  const int c = (blockIdx.x * kSumQuads + quad) * 4;
  int first = 0, count = p.units;
  if (y >= 2) {
    first = (y - 2) * p.units_per_gate;
    count = p.units_per_gate;
  }
  float4 sum{0.f, 0.f, 0.f, 0.f};
  if (c < p.cols) {
#pragma unroll 8
    for (int u = rank; u < count; u += kSumRanks) {
      const float4 a = *reinterpret_cast<const float4 *>(part + static_cast<int64_t>(first + u) * p.part_ld + c);
      sum.x += a.x;
      sum.y += a.y;
      sum.z += a.z;
      sum.w += a.w;
    }
  }
  auto add_up = [&](int from, int to) {   // ranks from .. to - 1 onto rank `from`
    for (int k = from + 1; k < to; ++k) {
      const float4 a = sums[k][quad];
      sum.x += a.x;
      sum.y += a.y;
      sum.z += a.z;
      sum.w += a.w;
    }
  };
  // by groups of kSumFold ranks first, then the groups
  sums[rank][quad] = sum;
  __syncthreads();
  if (rank % kSumFold == 0) add_up(rank, rank + kSumFold);
  __syncthreads();
  if (rank % kSumFold == 0) sums[rank / kSumFold][quad] = sum;
  __syncthreads();
  if (rank != 0 || c >= p.cols) return;
  add_up(0, kSumRanks / kSumFold);
  const float each[4] = {sum.x, sum.y, sum.z, sum.w};
  for (int m = 0; m < p.members; ++m) {
    float *to = reinterpret_cast<float *>(out + m * p.step) + (y >= 2 ? static_cast<int64_t>(y - 2) * p.cols : 0);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < p.cols) to[c + e] = each[e];
  }
}

// ---- host side ------------------------------------------------------------------------------------

// Lanes per row and vectors per lane: the fewest of either that hold the row.  The backward pass holds
// several rows at a time; at 1024 lanes a compute unit has room for one workgroup of it, so 512 lanes
// with more vectors come before.
struct RowLanes {
  int lanes, vecs;
};
RowLanes lanes_for(int cols, int vec, bool backward) {
  static const RowLanes forward_choices[] = {{64, 1}, {64, 2}, {256, 1}, {512, 1}, {1024, 1}, {1024, 2}, {1024, 4}};
  static const RowLanes backward_bf16[] = {{64, 1}, {64, 2}, {256, 1}, {512, 1}, {512, 2}, {1024, 2}};
  static const RowLanes backward_float[] = {{64, 1}, {64, 2}, {256, 1}, {512, 1}, {1024, 1}, {512, 4}, {1024, 4}};
  const RowLanes *c = !backward ? forward_choices : vec == 8 ? backward_bf16 : backward_float;
  while (c->lanes * c->vecs * vec < cols) ++c;   // the last of each holds kMaxCols elements
  return *c;
}

template <typename T, int kLanes, int NV, typename P, int kEnd, bool kNt>
void launch_rows(const P &p, int units, hipStream_t stream) {
  const unsigned per_wg = kWgLanes<kLanes> / kLanes;
  const dim3 grid((static_cast<unsigned>(units) + per_wg - 1) / per_wg), block(kWgLanes<kLanes>);
  if constexpr (std::is_same<P, NormForward>::value)
    hipLaunchKernelGGL((norm_kernel<T, kLanes, NV, kEnd, kNt>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((norm_grad_kernel<T, kLanes, NV, kEnd, kNt>), grid, block, 0, stream, p);
}

// How a call goes: how its rows end, and whether the Infinity Cache could not hold its operands.
struct Manner {
  RowEnd end;
  bool once;
};

template <typename T, int kLanes, int NV, typename P>
void launch_lanes(const P &p, int units, Manner m, hipStream_t stream) {
  if (m.end == kWhole) {
    if (m.once) launch_rows<T, kLanes, NV, P, kWhole, true>(p, units, stream);
    else launch_rows<T, kLanes, NV, P, kWhole, false>(p, units, stream);
  } else if (m.end == kShifted) {
    if (m.once) launch_rows<T, kLanes, NV, P, kShifted, true>(p, units, stream);
    else launch_rows<T, kLanes, NV, P, kShifted, false>(p, units, stream);
  } else if constexpr (kLanes == 64 && NV == 1) {
    launch_rows<T, kLanes, NV, P, kNarrow, false>(p, units, stream);
  }
}

template <typename T, typename P>
void launch_for(const P &p, int units, RowLanes l, bool once, hipStream_t stream) {
  const Manner m{p.s.cols < kRowVec<T> ? kNarrow : p.s.cols % kRowVec<T> ? kShifted : kWhole, once};
  constexpr bool kBackward = std::is_same<P, NormBackward>::value, kBf16 = sizeof(T) == 2;
  switch (l.lanes * 8 + l.vecs) {
    case 64 * 8 + 1: return launch_lanes<T, 64, 1>(p, units, m, stream);
    case 64 * 8 + 2: return launch_lanes<T, 64, 2>(p, units, m, stream);
    case 256 * 8 + 1: return launch_lanes<T, 256, 1>(p, units, m, stream);
    case 512 * 8 + 1: return launch_lanes<T, 512, 1>(p, units, m, stream);
    case 512 * 8 + 2:
      if constexpr (kBackward && kBf16) return launch_lanes<T, 512, 2>(p, units, m, stream);
      break;
    case 512 * 8 + 4:
      if constexpr (kBackward && !kBf16) return launch_lanes<T, 512, 4>(p, units, m, stream);
      break;
    case 1024 * 8 + 1:
      if constexpr (!kBackward || !kBf16) return launch_lanes<T, 1024, 1>(p, units, m, stream);
      break;
    case 1024 * 8 + 2:
      if constexpr (!kBackward || kBf16) return launch_lanes<T, 1024, 2>(p, units, m, stream);
      break;
    default:
      if constexpr (!kBf16) return launch_lanes<T, 1024, 4>(p, units, m, stream);
  }
}

template <typename P>
void launch_typed(int dtype, const P &p, int units, RowLanes l, bool once, hipStream_t stream) {
  if (dtype == RSM_BF16) launch_for<__hip_bfloat16>(p, units, l, once, stream);
  else launch_for<float>(p, units, l, once, stream);
}

size_t type_size(int dtype) { return dtype == RSM_FLOAT ? 4 : dtype == RSM_BF16 ? 2 : 0; }

// What a call's sizes and numbers come to, or false with the error set.  A = either argument struct.
template <typename A>
bool shape_of(const A &a, const char *call, size_t partial_ld, size_t normed_ld, rsm::Members *members, NormShape *out) {
  auto refuse = [&](const char *why) {
    rsm::fail(std::string(call) + ": " + why);
    return false;
  };
  if (!type_size(a.dtype)) return refuse("dtype must be RSM_FLOAT or RSM_BF16");
  if (a.flags & ~(RSM_NORM_POST | RSM_NORM_REPLICATED)) return refuse("unknown flags");
  if (a.cols < 1 || a.cols > kMaxCols) return refuse("cols must be in [1, 16384]");
  if (a.rows >= 1u << 22) return refuse("rows must be below 2^22");
  if (partial_ld < a.cols || normed_ld < a.cols || (a.residual_ld && a.residual_ld < a.cols))
    return refuse("a row stride is shorter than a row");
  const size_t far = ~size_t{0} >> 24;
  if (partial_ld > far / (a.rows + 1) || normed_ld > far / (a.rows + 1) || a.residual_ld > far / (a.rows + 1))
    return refuse("a row stride is too long");
  if (!(a.eps >= FLT_MIN) || !std::isfinite(a.eps)) return refuse("eps must be a positive (normal) number");
  if (!std::isfinite(a.residual_scale) || !std::isfinite(a.block_scale) || !std::isfinite(a.weight_offset))
    return refuse("scales and the weight offset must be finite");
  if (a.post_weight && !(a.flags & RSM_NORM_POST)) return refuse("post_weight without RSM_NORM_POST");
  if (!rsm::members_of(a.team, call, members)) return false;
  const rsm::Members &team = *members;
  NormShape s{};
  s.rows = static_cast<int>(a.rows);
  s.cols = static_cast<int>(a.cols);
  s.members = team.size;
  s.share = static_cast<int>((a.rows + team.size - 1) / team.size);
  if (s.share < 1) s.share = 1;
  // without a gate all rows are one group, whatever the field says
  const bool one_group = !a.gate || a.rows_per_gate == 0 || a.rows_per_gate > a.rows;
  s.rows_per_gate = one_group ? (s.rows ? s.rows : 1) : static_cast<int>(a.rows_per_gate);
  s.step = team.step;
  s.partial_ld = static_cast<int64_t>(partial_ld);
  s.normed_ld = static_cast<int64_t>(normed_ld);
  s.residual_ld = static_cast<int64_t>(a.residual_ld ? a.residual_ld : a.cols);
  s.eps = a.eps;
  s.inv_cols = static_cast<float>(1.0 / static_cast<double>(a.cols));
  s.residual_scale = a.residual_scale;
  s.block_scale = a.block_scale;
  s.pre_offset = a.pre_weight ? a.weight_offset : 1.f;
  s.post_offset = a.post_weight ? a.weight_offset : 1.f;
  s.post = (a.flags & RSM_NORM_POST) != 0;
  s.replicated = (a.flags & RSM_NORM_REPLICATED) != 0;
  *out = s;
  return true;
}

size_t gate_rows(const NormShape &s) { return s.rows ? (static_cast<size_t>(s.rows) + s.rows_per_gate - 1) / s.rows_per_gate : 0; }

// How the rows of a backward pass are dealt to units, and the room their sums take.
struct GradPlan {
  RowLanes lanes;
  int units, units_per_gate, rows_per_unit, part_ld;
  bool direct;
  size_t part_bytes;   // of one of the arrays of sums
  int parts;           // how many arrays there are
};

GradPlan plan_of(const NormShape &s, int dtype, bool has_gate) {
  GradPlan g{};
  g.lanes = lanes_for(s.cols, dtype == RSM_BF16 ? 8 : 4, true);
  // Enough units to fill the chip's 256 compute units, no more: each leaves its sums behind.  (Rows of a
  // wave, 8192 x 64 bf16 over 8 members: 1024 units 26.6 us, 2048 21.2, 4096 21.8.  Rows of 256 lanes, 512
  // units and 1024: 8192 x 2048 bf16 over 8 members 127 and 137, over 4 83 and 91, 8192 x 1200 over 3 62 and 52:
  // width and members change together there, and the rule puts it down to the members, whose fewer loads leave
  // a unit's lanes waiting; 106 of 256 lanes without an element may do it as well.  Rows of 512 lanes, 512
  // units and 1024: 8192 x 4096 over 4 members 162 and 167, over 1 98 and 109.)
  const int64_t target = g.lanes.lanes == 64 ? 2048 : g.lanes.lanes == 256 && s.members < 4 ? 1024 : g.lanes.lanes == 1024 ? 256 : 512;
  const int64_t per_unit = (s.rows + target - 1) / target;
  const int64_t group = s.rows_per_gate;
  g.part_ld = (s.cols + 3) & ~3;
  if (group <= per_unit && has_gate && gate_rows(s) > 1) {
    g.direct = true;
    g.rows_per_unit = static_cast<int>((per_unit + group - 1) / group * group);
    g.units_per_gate = 0;
    g.units = static_cast<int>((s.rows + g.rows_per_unit - 1) / g.rows_per_unit);
  } else {
    g.direct = false;
    g.units_per_gate = static_cast<int>((group + per_unit - 1) / (per_unit ? per_unit : 1));
    if (g.units_per_gate < 1) g.units_per_gate = 1;
    g.units = g.units_per_gate * static_cast<int>(gate_rows(s));
  }
  g.parts = 1 + (s.post ? 1 : 0) + (has_gate && !g.direct ? 1 : 0);
  g.part_bytes = static_cast<size_t>(g.units) * g.part_ld * sizeof(float);
  return g;
}

// What a call moves: every member's rows in and out, and `more` rows on the owners.
size_t rows_bytes(const NormShape &s, size_t size, size_t more) {
  return static_cast<size_t>(s.rows) * s.cols * size * (2 * static_cast<size_t>(s.members) + more);
}

const char *moved(const void *p, int64_t bytes) { return p ? static_cast<const char *>(p) + bytes : nullptr; }
char *moved(void *p, int64_t bytes) { return p ? static_cast<char *>(p) + bytes : nullptr; }

}  // namespace

extern "C" {

int rsm_norm_to_all(const rsm_norm_args_t *args, void *stream) {
  RSM_ENTRY;
  const char *call = "norm_to_all";
  if (!args) return rsm::fail("norm_to_all: arguments are NULL");
  const rsm_norm_args_t &a = *args;
  rsm::Members team;
  NormShape s;
  const size_t source_ld = a.source_ld ? a.source_ld : a.cols, normed_ld = a.normed_ld ? a.normed_ld : a.cols;
  if (!a.source || !a.residual || !a.residual_out) return rsm::fail("norm_to_all: source, residual and residual_out must be given");
  if (a.pre_weight && !a.normed) return rsm::fail("norm_to_all: pre_weight without normed");
  if (!shape_of(a, call, source_ld, normed_ld, &team, &s)) return -1;
  if (a.rows == 0) return 0;
  const size_t size = type_size(a.dtype), held = s.replicated ? a.rows : s.share, ld = static_cast<size_t>(s.residual_ld);
  rsm::Operands o(call);
  const int source = o.matrix(a.source, "source", a.rows, a.cols, source_ld, size, false);
  const int residual = o.matrix(a.residual, "residual", held, a.cols, ld, size, false);
  o.add(a.pre_weight, "pre_weight", a.cols * size, size, false);
  o.add(a.post_weight, "post_weight", a.cols * size, size, false);
  o.add(a.gate, "gate", gate_rows(s) * a.cols * size, size, false);
  o.matrix(a.residual_out, "residual_out", held, a.cols, ld, size, true, residual);
  o.matrix(a.normed, "normed", a.rows, a.cols, normed_ld, size, true, normed_ld == source_ld ? source : o.kNone);
  o.matrix(a.total, "total", s.share, a.cols, a.cols, size, true);
  if (!o.ok()) return -1;
  NormForward p{};
  p.s = s;
  p.source = moved(a.source, team.first);
  p.residual = moved(a.residual, team.first);
  p.pre_weight = moved(a.pre_weight, team.first);
  p.post_weight = moved(a.post_weight, team.first);
  p.gate = moved(a.gate, team.first);
  p.residual_out = moved(a.residual_out, team.first);
  p.normed = moved(a.normed, team.first);
  p.total = moved(a.total, team.first);
  launch_typed(a.dtype, p, s.rows, lanes_for(s.cols, a.dtype == RSM_BF16 ? 8 : 4, false),
               rows_bytes(s, size, 2) > rsm::kInfinityCacheBytes, static_cast<hipStream_t>(stream));
  return rsm::after_launch(call);
}

int rsm_norm_grad_work_bytes(const rsm_norm_grad_args_t *args, size_t *bytes) {
  RSM_ENTRY;
  const char *call = "norm_grad_work_bytes";
  if (!args || !bytes) return rsm::fail("norm_grad_work_bytes: an argument is NULL");
  rsm::Members team;
  NormShape s;
  if (!shape_of(*args, call, args->cols, args->cols, &team, &s)) return -1;
  const GradPlan g = plan_of(s, args->dtype, args->gate != nullptr);
  *bytes = g.part_bytes * g.parts;
  return 0;
}

int rsm_norm_to_all_grad(const rsm_norm_grad_args_t *args, void *stream) {
  RSM_ENTRY;
  const char *call = "norm_to_all_grad";
  if (!args) return rsm::fail("norm_to_all_grad: arguments are NULL");
  const rsm_norm_grad_args_t &a = *args;
  rsm::Members team;
  NormShape s;
  const size_t source_ld = a.source_ld ? a.source_ld : a.cols, normed_ld = a.normed_ld ? a.normed_ld : a.cols;
  if (!a.grad_source) return rsm::fail("norm_to_all_grad: grad_source must be given");
  if (!a.grad_normed && !a.grad_residual_out) return rsm::fail("norm_to_all_grad: neither grad_normed nor grad_residual_out is given");
  if (a.grad_normed && !a.residual_out) return rsm::fail("norm_to_all_grad: grad_normed needs residual_out");
  if (((a.flags & RSM_NORM_POST) || a.grad_gate) && !a.total) return rsm::fail("norm_to_all_grad: total must be given (with RSM_NORM_POST, or for grad_gate)");
  if (a.grad_pre_weight && !a.grad_normed) return rsm::fail("norm_to_all_grad: grad_pre_weight without grad_normed");
  if (a.grad_post_weight && !(a.flags & RSM_NORM_POST)) return rsm::fail("norm_to_all_grad: grad_post_weight without RSM_NORM_POST");
  if (a.grad_gate && !a.gate) return rsm::fail("norm_to_all_grad: grad_gate without gate");
  if (!shape_of(a, call, source_ld, normed_ld, &team, &s)) return -1;
  const GradPlan g = plan_of(s, a.dtype, a.gate != nullptr);
  const bool sums = a.grad_pre_weight || a.grad_post_weight || (a.grad_gate && !g.direct);
  if (sums && s.rows && !a.work) return rsm::fail("norm_to_all_grad: work must be given (rsm_norm_grad_work_bytes)");
  const size_t size = type_size(a.dtype), held = s.replicated ? a.rows : s.share, ld = static_cast<size_t>(s.residual_ld);
  const size_t mine = a.rows ? held : 0, shared = a.rows ? s.share : 0;
  rsm::Operands o(call);
  const int grad_normed = o.matrix(a.grad_normed, "grad_normed", a.rows, a.cols, normed_ld, size, false);
  o.matrix(a.residual_out, "residual_out", mine, a.cols, ld, size, false);
  o.matrix(a.total, "total", shared, a.cols, a.cols, size, false);
  const int grad_residual_out = o.matrix(a.grad_residual_out, "grad_residual_out", mine, a.cols, ld, size, false);
  o.add(a.pre_weight, "pre_weight", a.cols * size, size, false);
  o.add(a.post_weight, "post_weight", a.cols * size, size, false);
  o.add(a.gate, "gate", gate_rows(s) * a.cols * size, size, false);
  o.matrix(a.grad_source, "grad_source", a.rows, a.cols, source_ld, size, true, source_ld == normed_ld ? grad_normed : o.kNone);
  o.matrix(a.grad_residual, "grad_residual", mine, a.cols, ld, size, true, grad_residual_out);
  o.add(a.grad_pre_weight, "grad_pre_weight", a.cols * 4, 4, true);
  o.add(a.grad_post_weight, "grad_post_weight", a.cols * 4, 4, true);
  o.add(a.grad_gate, "grad_gate", gate_rows(s) * a.cols * 4, 4, true);
  if (sums) o.add(a.work, "work (rsm_norm_grad_work_bytes)", g.part_bytes * g.parts, 16, true);
  if (!o.ok()) return -1;
  if (!a.grad_gate && !sums && a.rows == 0) return 0;

  NormBackward p{};
  p.s = s;
  p.grad_normed = moved(a.grad_normed, team.first);
  p.residual_out = moved(a.residual_out ? a.residual_out : a.grad_residual_out, team.first);
  p.total = moved(a.total, team.first);
  p.grad_residual_out = moved(a.grad_residual_out, team.first);
  p.pre_weight = moved(a.pre_weight, team.first);
  p.post_weight = moved(a.post_weight, team.first);
  p.gate = moved(a.gate, team.first);
  p.grad_source = moved(a.grad_source, team.first);
  p.grad_residual = moved(a.grad_residual, team.first);
  p.grad_gate = moved(a.grad_gate, team.first);
  float *part = reinterpret_cast<float *>(moved(a.work, team.first));
  const size_t part_floats = g.part_bytes / sizeof(float);
  if (a.grad_pre_weight) p.part_pre = part;
  if (a.grad_post_weight) p.part_post = part + part_floats;
  if (a.grad_gate && !g.direct) p.part_gate = part + part_floats * (s.post ? 2 : 1);
  p.part_ld = g.part_ld;
  p.units = g.units;
  p.units_per_gate = g.units_per_gate;
  p.rows_per_unit = g.rows_per_unit;
  p.direct = g.direct;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (g.units) launch_typed(a.dtype, p, g.units, g.lanes, rows_bytes(s, size, 4) > rsm::kInfinityCacheBytes, st);
  if (sums) {
    PartSums r{};
    r.part_pre = p.part_pre;
    r.part_post = p.part_post;
    r.part_gate = p.part_gate;
    r.grad_pre = moved(a.grad_pre_weight, team.first);
    r.grad_post = moved(a.grad_post_weight, team.first);
    r.grad_gate = p.part_gate ? p.grad_gate : nullptr;
    r.units = g.units;
    r.units_per_gate = g.units_per_gate;
    r.part_ld = g.part_ld;
    r.cols = s.cols;
    r.members = s.members;
    r.step = s.step;
    const unsigned gates = p.part_gate ? static_cast<unsigned>(gate_rows(s)) : 0;
    hipLaunchKernelGGL(part_sums_kernel, dim3((s.cols + 4 * kSumQuads - 1) / (4 * kSumQuads), 2 + gates), dim3(kSumQuads * kSumRanks), 0, st, r);
  }
  return rsm::after_launch(call);
}

}  // extern "C"
