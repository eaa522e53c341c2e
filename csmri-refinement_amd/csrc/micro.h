// Block-scaled number formats (shared by act8.hip, lnorm.hip, mx4.hip): 32 consecutive channels of a pixel share one
// power-of-two scale, stored as its biased exponent in a byte (E8M0).
//
//   e = max(floor(log2(largest magnitude of the block)), MICRO_MIN_EXP)
//   kept activations   scale 2^(e - 7), elements e4m3: |x / scale| < 256, nothing saturates (the format ends at 448)
//   4-bit operands     scale 2^(e - 2), elements e2m1 {0, .5, 1, 1.5, 2, 3, 4, 6}: |x / scale| < 8, saturating at 6
//
// Dividing by the scale is exact, so the only rounding is the conversion's, to nearest even.  A block that holds an
// infinity or a NaN gets the scale byte 255 and reads back as NaN throughout: it is not silently made finite.
#pragma once
#include "common.h"

#define MICRO_BLOCK 32
#define MICRO_MIN_EXP (-100)     // scales and their inverses stay normal fp32 numbers
#define MICRO_NAN 255

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// the magnitude's bits order like an unsigned integer, infinities and NaN above every finite number
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ bool micro_finite(unsigned amax) { return amax < 0x7f800000u; }
__device__ __forceinline__ int micro_exp(unsigned amax) {
  const int e = (int)(amax >> 23) - 127;
  return e < MICRO_MIN_EXP ? MICRO_MIN_EXP : e;
}

// Values of neighbouring lanes through the data-parallel paths of the vector unit (a shuffle through LDS takes ten times as
// long): lane ^ 1, lane ^ 2, and the mirror images inside 8 and 16 lanes, which stand for lane ^ 4 and lane ^ 8 once the
// lanes of a quad (of an eighth) agree.
#define DPP_XOR1 0xB1
#define DPP_XOR2 0x4E
#define DPP_MIRROR8 0x141
#define DPP_MIRROR16 0x140
template <int CTRL> __device__ __forceinline__ unsigned dpp_u(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
template <int CTRL> __device__ __forceinline__ float dpp_f(float v) { return __uint_as_float(dpp_u<CTRL>(__float_as_uint(v))); }

// sums over aligned groups of `group` lanes (4 .. 64, a power of two), the same bits in every lane of a group
template <int N> __device__ __forceinline__ void group_sums(float (&v)[N], int group) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] += dpp_f<DPP_XOR1>(v[i]);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] += dpp_f<DPP_XOR2>(v[i]);
  if (group < 8) return;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] += dpp_f<DPP_MIRROR8>(v[i]);
  if (group < 16) return;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] += dpp_f<DPP_MIRROR16>(v[i]);
  if (group < 32) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
    v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (group < 64) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
    v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
}

// eight channels per lane, four consecutive lanes per block: the block's largest magnitude in each of them
__device__ __forceinline__ unsigned block_amax(const float* v) {
  unsigned m = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) { const unsigned a = abs_bits(v[k]); m = a > m ? a : m; }
  unsigned t = dpp_u<DPP_XOR1>(m);
  m = t > m ? t : m;
  t = dpp_u<DPP_XOR2>(m);
  return t > m ? t : m;
}

// eight values -> eight e4m3 codes and their scale byte
__device__ __forceinline__ u32x2_t micro_pack8(const float* v, unsigned amax, unsigned char& scale) {
  u32x2_t q;
  if (!micro_finite(amax)) {
    scale = MICRO_NAN;
    q[0] = q[1] = 0x7f7f7f7fu;
    return q;
  }
  const int e = micro_exp(amax) - 7;
  const float s = exp2i(-e);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h] * s, v[4 * h + 1] * s, r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2] * s, v[4 * h + 3] * s, r, true);
    q[h] = (unsigned)r;
  }
  scale = (unsigned char)(e + 127);
  return q;
}
// scale byte -> factor: 0 is 2^-127, no normal fp32 number, and 255 NaN
__device__ __forceinline__ float micro_scale(unsigned char s) {
  return __uint_as_float(s == 0 ? 0x00400000u : (s == MICRO_NAN ? 0x7fc00000u : (unsigned)s << 23));
}

__device__ __forceinline__ void micro_unpack8(u32x2_t q, float s, float* v) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)q[h], true);
    v[4 * h] = a[0] * s; v[4 * h + 1] = a[1] * s; v[4 * h + 2] = b[0] * s; v[4 * h + 3] = b[1] * s;
  }
}

// eight consecutive channels of an activation tensor, raw and as fp32
template <int DT> struct raw8 { f32x4_t a, b; };
template <> struct raw8<CSMRI_BF16> { u32x4_t a; };
template <int DT> __device__ __forceinline__ raw8<DT> ldraw8(const void* p, long long idx) {
  raw8<DT> r;
  if constexpr (DT == CSMRI_F32) {
    r.a = *(const f32x4_t*)((const float*)p + idx);
    r.b = *(const f32x4_t*)((const float*)p + idx + 4);
  } else {
    r.a = *(const u32x4_t*)((const unsigned short*)p + idx);
  }
  return r;
}
template <int DT> __device__ __forceinline__ void cvt8(const raw8<DT>& r, float* v) {
  if constexpr (DT == CSMRI_F32) {
#pragma unroll
    for (int k = 0; k < 4; ++k) { v[k] = r.a[k]; v[4 + k] = r.b[k]; }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      v[2 * k] = __uint_as_float(r.a[k] << 16);
      v[2 * k + 1] = __uint_as_float(r.a[k] & 0xffff0000u);
    }
  }
}
template <int DT> __device__ __forceinline__ void st8(void* p, long long idx, const float* v) {
  if constexpr (DT == CSMRI_F32) {
    *(f32x4_t*)((float*)p + idx) = (f32x4_t){v[0], v[1], v[2], v[3]};
    *(f32x4_t*)((float*)p + idx + 4) = (f32x4_t){v[4], v[5], v[6], v[7]};
  } else {
    const u32x2_t a = pack4_bf16((f32x4_t){v[0], v[1], v[2], v[3]}), b = pack4_bf16((f32x4_t){v[4], v[5], v[6], v[7]});
    *(u32x4_t*)((unsigned short*)p + idx) = (u32x4_t){a[0], a[1], b[0], b[1]};
  }
}

// How the streaming kernels walk [rows][slots], a slot being eight channels: a workgroup of 256 threads holds
// 256 / cols rows of cols slots (cols = the row's slots, a multiple of four, at most 256; longer rows continue along
// blockIdx.y), so a thread's slot never changes and the loop over rows has no division.
struct RowWalk { int cols, rows_per_tile; };
static inline RowWalk row_walk(int slots) {
  RowWalk w;
  w.cols = slots < 256 ? slots : 256;
  w.rows_per_tile = 256 / w.cols;
  return w;
}
static inline dim3 row_walk_grid(long long rows, int slots, int unroll) {
  const RowWalk w = row_walk(slots);
  const int gy = (slots + w.cols - 1) / w.cols;
  long long gx = (rows + (long long)w.rows_per_tile * unroll - 1) / ((long long)w.rows_per_tile * unroll);
  const long long cap = 2048 / gy > 0 ? 2048 / gy : 1;       // eight workgroups a CU
  if (gx > cap) gx = cap;
  return dim3((unsigned)(gx < 1 ? 1 : gx), (unsigned)gy);
}

// Do two buffers of fp32 values share an element?  (Sums that add to one place from two threads would lose one another's.)
static inline bool buffers_meet(const float* a, long long na, const float* b, long long nb) {
  return a && b && a < b + nb && b < a + na;
}

// oa[col] (+)= sum over rows of partial[row][col] for col < na, ob[col] likewise for the nb columns behind them, in a fixed
// order (act8.hip; the weight gradient's slabs and the layer norm's affine partials end in it)
int micro_colsum2(const float* partial, int rows, long long row_stride, long long na, float* oa, long long nb, float* ob,
                  int accumulate, hipStream_t st);
