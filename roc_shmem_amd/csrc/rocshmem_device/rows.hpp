// Building blocks of the row collectives (norm_to_all, logprob_to_all and their gradients): rows of
// float or bfloat16 read and written 16 bytes per lane at any element alignment, held as float, and
// sums over the lanes of a row.
#ifndef ROCSHMEM_MI355X_DEVICE_ROWS_HPP
#define ROCSHMEM_MI355X_DEVICE_ROWS_HPP

#include <hip/hip_bf16.h>

#include "copy.hpp"
#include "reduce.hpp"
#include "wave.hpp"

namespace rocshmem {
namespace detail {

typedef u32x4 u32x4_a2 __attribute__((aligned(2)));

// Elements of T in a 16-byte vector.
template <typename T>
constexpr int kRowVec = 16 / static_cast<int>(sizeof(T));

// The kRowVec<T> elements at `p` as raw bits.  `left` elements of the row remain: the rest of the
// vector is not read and comes back as `fill` bits.  A row may start at any element: the hardware
// reads a 16-byte vector at any address (kTail false: `left` is a multiple of kRowVec<T>).
// kNt: past the caches' allocation, for data that is read once and would not stay in them.
template <typename T, bool kTail, bool kNt = false>
__device__ __forceinline__ u32x4 row_load(const T *p, int left, uint32_t fill = 0) {
  u32x4 v = {fill, fill, fill, fill};
  if (!kTail ? left > 0 : left >= kRowVec<T>) {
    if constexpr (kNt) v = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2 *>(p));
    else v = *reinterpret_cast<const u32x4_a2 *>(p);
  } else if (kTail && left > 0) {
    if constexpr (sizeof(T) == 4) {
      const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
#pragma unroll
      for (int e = 0; e < 3; ++e)
        if (e < left) v[e] = q[e];
    } else {
      const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
      for (int e = 0; e < 7; ++e)
        if (e < left)
          v[e / 2] = e % 2 ? (v[e / 2] & 0xffffu) | static_cast<uint32_t>(q[e]) << 16
                           : (v[e / 2] & 0xffff0000u) | q[e];
    }
  }
  return v;
}

// Element e of a raw vector as float.
template <typename T>
__device__ __forceinline__ float row_get(u32x4 v, int e) {
  if constexpr (sizeof(T) == 4) return __uint_as_float(v[e]);
  else return __uint_as_float(e % 2 ? v[e / 2] & 0xffff0000u : v[e / 2] << 16);
}

// Two floats rounded to bfloat16 (nearest even), the first in the low half.
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b16x2 __attribute__((ext_vector_type(2)));
  const b16x2 b = __builtin_convertvector((f32x2{lo, hi}), b16x2);
  return __builtin_bit_cast(uint32_t, b);
}

// Floats rounded once to T, as raw bits.
template <typename T>
__device__ __forceinline__ u32x4 row_pack(const float (&f)[kRowVec<T>]) {
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == 4) v[k] = __float_as_uint(f[k]);
    else v[k] = pack_bf16(f[2 * k], f[2 * k + 1]);
  }
  return v;
}

// The first `left` elements of a vector, fewer than all of them: in pieces of 8, 4 and 2 bytes.
typedef uint32_t u32_a2 __attribute__((aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_a2 __attribute__((aligned(2)));
template <typename T>
__device__ __forceinline__ void row_store_tail(T *p, int left, u32x4 v) {
  const int bytes = left * static_cast<int>(sizeof(T));
  char *q = reinterpret_cast<char *>(p);
  if (bytes & 8) *reinterpret_cast<u32x2_a2 *>(q) = u32x2{v[0], v[1]};
  if (bytes & 4) *reinterpret_cast<u32_a2 *>(q + (bytes & 8)) = bytes & 8 ? v[2] : v[0];
  if (bytes & 2) {
    uint32_t w = v[0];
#pragma unroll
    for (int k = 1; k < 4; ++k)
      if ((bytes & 12) == 4 * k) w = v[k];
    *reinterpret_cast<uint16_t *>(q + (bytes & 12)) = static_cast<uint16_t>(w);
  }
}

template <typename T, bool kTail, bool kNt = false>
__device__ __forceinline__ void row_store(T *p, int left, u32x4 v) {
  if (!kTail ? left > 0 : left >= kRowVec<T>) {
    if constexpr (kNt) __builtin_nontemporal_store(v, reinterpret_cast<u32x4_a2 *>(p));
    else *reinterpret_cast<u32x4_a2 *>(p) = v;
  } else if (kTail && left > 0) {
    row_store_tail(p, left, v);
  }
}

// `p` moved by `bytes`.  Pointer arithmetic: an address that has been an integer is one of the flat
// address space to the compiler, and flat stores share the counter that LDS results are waited for on.
template <typename T>
__device__ __forceinline__ T *bytes_on(T *p, int64_t bytes) {
  return reinterpret_cast<T *>(reinterpret_cast<char *>(p) + bytes);
}

// Value of `v` under a DPP control word; lanes the control leaves out get 0.
template <int kCtrl, int kRowMask = 0xf>
__device__ __forceinline__ float dpp_or_zero(float v) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), kCtrl, kRowMask, 0xf, false));
}

// Sum over the 64 lanes, the same in every lane.  Within rows of 16 lanes by quad permutes and
// rotations, then row 0 into 1 and 2 into 3, then row 1 into 3: lane 63 holds the sum.  All in the
// vector unit, without a trip through LDS for each of the six steps.
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp_or_zero<0xB1>(v);         // quad_perm [1,0,3,2]
  v += dpp_or_zero<0x4E>(v);         // quad_perm [2,3,0,1]
  v += dpp_or_zero<0x124>(v);        // row_ror:4
  v += dpp_or_zero<0x128>(v);        // row_ror:8
  v += dpp_or_zero<0x142, 0xa>(v);   // row_bcast:15 into rows 1 and 3
  v += dpp_or_zero<0x143, 0xc>(v);   // row_bcast:31 into rows 2 and 3
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}

// Largest of the lanes' values, the same in every lane; none of them is NaN.
__device__ __forceinline__ float wave_max(float v) {
#define RSM_MAX_STEP(ctrl, rows)                                                                       \
  v = fmaxf(v, __uint_as_float(__builtin_amdgcn_update_dpp(__float_as_uint(v), __float_as_uint(v), ctrl, rows, 0xf, false)))
  RSM_MAX_STEP(0xB1, 0xf);
  RSM_MAX_STEP(0x4E, 0xf);
  RSM_MAX_STEP(0x124, 0xf);
  RSM_MAX_STEP(0x128, 0xf);
  RSM_MAX_STEP(0x142, 0xa);
  RSM_MAX_STEP(0x143, 0xc);
#undef RSM_MAX_STEP
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63));
}

// Sums of kN values over the kLanes lanes that hold a row (a wave, or the whole workgroup), the same
// in every lane.  `slots` is LDS for 2 x (kLanes / 64) x kN floats and `turn` picks its half, which
// alternates from call to call: a lane that writes the half again has passed the barrier of the call
// in between, behind which nobody reads the older sums any more.
template <int kLanes, int kN>
__device__ __forceinline__ void row_sums(float (&v)[kN], float *slots, int &turn) {
#pragma unroll
  for (int k = 0; k < kN; ++k) v[k] = wave_sum(v[k]);
  if constexpr (kLanes > 64) {
    constexpr int kWaves = kLanes / 64;
    float *mine = slots + turn * kWaves * kN;
    turn ^= 1;
    if (lane_id() == 0) {
#pragma unroll
      for (int k = 0; k < kN; ++k) mine[(threadIdx.x / 64) * kN + k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) s += mine[w * kN + k];
      v[k] = s;
    }
  }
}

}  // namespace detail
}  // namespace rocshmem

#endif
