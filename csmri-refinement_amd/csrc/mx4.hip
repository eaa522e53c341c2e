// Microscaled 4-bit operands (micro.h: e2m1 elements, one E8M0 scale per 32 consecutive channels) and the product of a
// 1 x 1 convolution on them:
//
//   y[p][n] = act( sum_c xq[p][c] wq[n][c] + bias[n] ),  xq, wq the values the 4-bit forms stand for
//
// A row of K channels is 64 bytes of codes per 128 channels (two a byte, the even channel in the low half) and one scale
// byte per 32 channels, padded to 16 bytes per 512 channels; padding is code 0, scale 2^0.  The contraction is
// v_mfma_scale_f32_*_f8f6f4, 16x16x128 for few rows and 32x32x64 in the tiles: a lane's operand is 32 channels of one row,
// exactly one block, so its scale rides in the lane next to it.  Products are exact (the elements are multiples of 1/2 up
// to 6); sums across blocks of different scales round to fp32.
//
// Times below: a kernel's own are medians of a kernel trace; where "back to back" is said, launches one behind the other
// without one, which the large products run 10 - 15 % faster.
#include "micro.h"

typedef __attribute__((ext_vector_type(8))) int i32x8_t;

static inline int mx4_code_bytes(int K) { return 64 * ((K + 127) / 128); }
static inline int mx4_scale_bytes(int K) { return 16 * ((K + 511) / 512); }
extern "C" int csmri_mx4_code_bytes(int K) { return K > 0 ? mx4_code_bytes(K) : 0; }
extern "C" int csmri_mx4_scale_bytes(int K) { return K > 0 ? mx4_scale_bytes(K) : 0; }

// eight values -> eight codes; scale: the block's
__device__ __forceinline__ unsigned mx4_pack8(const float* v, float scale) {
  unsigned q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
  return q;
}
// A lane's whole block, 32 consecutive channels -> 16 bytes of codes and the scale byte.  bf16 stays packed: its magnitudes
// order as 16-bit integers, and the conversion takes pairs.
typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
template <int DT> __device__ __forceinline__ u32x4_t mx4_pack_block(const raw8<DT> (&raw)[4], int& scale) {
  unsigned amax;
  if constexpr (DT == CSMRI_BF16) {
    u16x2_t m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, raw[i].a[k] & 0x7fff7fffu));
    amax = (unsigned)(m[0] > m[1] ? m[0] : m[1]) << 16;
  } else {
    amax = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) { amax = max(amax, abs_bits(raw[i].a[k])); amax = max(amax, abs_bits(raw[i].b[k])); }
  }
  const bool fin = micro_finite(amax);
  const int e = fin ? micro_exp(amax) - 2 : 0;
  const float s = exp2i(e);
  u32x4_t q;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == CSMRI_BF16) {
      // (named words: a bit cast of a vector's element takes the vector's first)
      const unsigned w0 = raw[i].a[0], w1 = raw[i].a[1], w2 = raw[i].a[2], w3 = raw[i].a[3];
      unsigned t = 0;
      t = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(t, __builtin_bit_cast(bf16x2_t, w0), s, 0);
      t = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(t, __builtin_bit_cast(bf16x2_t, w1), s, 1);
      t = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(t, __builtin_bit_cast(bf16x2_t, w2), s, 2);
      q[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(t, __builtin_bit_cast(bf16x2_t, w3), s, 3);
    } else {
      float v[8];
      cvt8<DT>(raw[i], v);
      q[i] = mx4_pack8(v, s);
    }
  }
  scale = fin ? e + 127 : MICRO_NAN;
  return q;
}
__device__ __forceinline__ i32x8_t mx4_operand(u32x4_t c) {
  return (i32x8_t){(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
}
__device__ __forceinline__ f32x4_t mx4_mfma(i32x8_t a, int sa, i32x8_t b, int sb, f32x4_t acc) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 0, sa, 0, sb);
}

// ---- quantise / dequantise: one read, one write, bound by HBM (32768 x 1024 bf16: 17 and 15 us for 85 MB) ---------------------------------------------------------
template <int DT>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const void* __restrict__ x, int ps, long long rows, int c8,
                                                           int slots, int sbytes, int cols, int rpt,
                                                           unsigned* __restrict__ q, unsigned char* __restrict__ s) {
  constexpr int U = 4;
  const int slot = blockIdx.y * cols + threadIdx.x % cols, r0 = threadIdx.x / cols;
  const bool live = r0 < rpt && slot < slots, load = live && slot < c8;
  const long long step = (long long)gridDim.x * rpt;
  for (long long row = (long long)blockIdx.x * rpt + r0; row - r0 < rows; row += step * U) {
    raw8<DT> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step;
      raw[u] = raw8<DT>{};
      if (load && rr < rows) raw[u] = ldraw8<DT>(x, rr * ps + slot * 8);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step;
      float v[8];
      cvt8<DT>(raw[u], v);
      const unsigned amax = block_amax(v);
      const bool fin = micro_finite(amax);
      const int e = micro_exp(amax) - 2;
      const unsigned o = fin ? mx4_pack8(v, exp2i(e)) : 0u;
      if (live && rr < rows) {
        q[rr * slots + slot] = o;
        // blocks wholly behind the row's end: scale 2^0
        if ((slot & 3) == 0) s[rr * sbytes + (slot >> 2)] = slot >= c8 ? 127 : (fin ? (unsigned char)(e + 127) : MICRO_NAN);
        if (slot == 0)
          for (int b = slots / 4; b < sbytes; b += 4) *(unsigned*)(s + rr * sbytes + b) = 0x7f7f7f7fu;
      }
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void mx4_dequantize_kernel(const unsigned* __restrict__ q, const unsigned char* __restrict__ s,
                                                             long long rows, int c8, int slots, int sbytes, int cols, int rpt,
                                                             void* __restrict__ out, int ps) {
  constexpr int U = 4;
  const int slot = blockIdx.y * cols + threadIdx.x % cols, r0 = threadIdx.x / cols;
  if (r0 >= rpt || slot >= c8) return;
  const long long step = (long long)gridDim.x * rpt;
  for (long long row = (long long)blockIdx.x * rpt + r0; row < rows; row += step * U) {
    unsigned c[U]; unsigned char sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step < rows ? row + u * step : row;
      c[u] = q[rr * slots + slot];
      sc[u] = s[rr * sbytes + (slot >> 2)];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (row + u * step >= rows) break;
      float v[8];
      // scale 1 here: the factor is applied as an fp32 product, exact
      const float f = micro_scale(sc[u]);
      auto t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 0); v[0] = t[0] * f; v[1] = t[1] * f;
      t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 1); v[2] = t[0] * f; v[3] = t[1] * f;
      t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 2); v[4] = t[0] * f; v[5] = t[1] * f;
      t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 3); v[6] = t[0] * f; v[7] = t[1] * f;
      st8<DT>(out, (row + u * step) * ps + slot * 8, v);
    }
  }
}

#define MX4_MAX_K (1 << 24)    // channels of a row: a tile's 256 rows of codes and scales stay within 32-bit offsets
static bool mx4_shape_ok(long long rows, int K, int ps, int dtype) {
  return rows >= 0 && K > 0 && K % 8 == 0 && K <= MX4_MAX_K && ps >= K && (dtype == CSMRI_F32 || dtype == CSMRI_BF16);
}
static bool mx4_rows_aligned(const void* p, int ps, int dtype) {
  return ((uintptr_t)p & 15) == 0 && ((long long)ps * dtype_size(dtype)) % 16 == 0;
}

extern "C" int csmri_mx4_quantize(int dtype, const void* x, int x_pix_stride, long long rows, int K, void* codes,
                                  uint8_t* scales, void* stream) {
  CSMRI_CHECK_ARG(mx4_shape_ok(rows, K, x_pix_stride, dtype));
  if (rows == 0) return CSMRI_OK;
  CSMRI_CHECK_ARG(x && codes && scales);
  if (!mx4_rows_aligned(x, x_pix_stride, dtype) || (((uintptr_t)codes | (uintptr_t)scales) & 15)) return CSMRI_E_ALIGN;
  const int slots = mx4_code_bytes(K) / 4;
  const RowWalk w = row_walk(slots);
  auto kern = dtype == CSMRI_F32 ? mx4_quantize_kernel<CSMRI_F32> : mx4_quantize_kernel<CSMRI_BF16>;
  hipLaunchKernelGGL(kern, row_walk_grid(rows, slots, 4), dim3(256), 0, (hipStream_t)stream, x, x_pix_stride, rows, K / 8,
                     slots, mx4_scale_bytes(K), w.cols, w.rows_per_tile, (unsigned*)codes, (unsigned char*)scales);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}

extern "C" int csmri_mx4_dequantize(const void* codes, const uint8_t* scales, long long rows, int K, int dtype, void* out,
                                    int out_pix_stride, void* stream) {
  CSMRI_CHECK_ARG(mx4_shape_ok(rows, K, out_pix_stride, dtype));
  if (rows == 0) return CSMRI_OK;
  CSMRI_CHECK_ARG(codes && scales && out);
  if (!mx4_rows_aligned(out, out_pix_stride, dtype) || (((uintptr_t)codes | (uintptr_t)scales) & 15)) return CSMRI_E_ALIGN;
  const int slots = mx4_code_bytes(K) / 4;
  const RowWalk w = row_walk(slots);
  auto kern = dtype == CSMRI_F32 ? mx4_dequantize_kernel<CSMRI_F32> : mx4_dequantize_kernel<CSMRI_BF16>;
  hipLaunchKernelGGL(kern, row_walk_grid(rows, slots, 4), dim3(256), 0, (hipStream_t)stream, (const unsigned*)codes,
                     (const unsigned char*)scales, rows, K / 8, slots, mx4_scale_bytes(K), w.cols, w.rows_per_tile, out,
                     out_pix_stride);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}

// ---- product ------------------------------------------------------------------------------------------------------------
struct MxParams {
  const void* x; int xps;                        // activations to be quantised on the way (few rows), or
  const char* xq; const unsigned char* xs;       // their 4-bit form
  const char* wq; const unsigned char* ws;
  const float* bias; float slope;
  void* out; int out_dt, ops;
  long long M; int N, Npad, K, ksteps, cb, sb;   // ksteps: 128-channel steps; cb, sb: code and scale bytes of a row
  int mtiles, ntiles;
  int splits, schunk; float* slab;               // splits of the channels, schunk steps each; [splits][M][Npad] partial sums
};

// four consecutive outputs n..n+3 of row m
__device__ __forceinline__ void mx4_store(const MxParams& p, long long m, int n, f32x4_t v) {
  if (n >= p.Npad) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const bool ok = n + k < p.N;
    const float y = v[k] + (p.bias && ok ? p.bias[n + k] : 0.f);
    v[k] = ok ? (y > 0.f ? y : y * p.slope) : 0.f;
  }
  store4(p.out, m * p.ops + n, p.out_dt, v);
}

// Few rows (up to 16 MF): bound by the weights' bytes, and for one row by the latency of a single pass over them (1 x 4096
// x 4096: 5.9 us, 4.8 on codes, 8.9 MB; 64 x 4096 x 4096: 12 us).  A workgroup of eight waves owns 16 outputs; the waves split the
// channels, each lane reads its operands straight from memory, and the eight partial tiles are added in wave order.
// QX: a lane quantises its own 32 channels of x, which saves the launch of a quantisation kernel.
template <int MF, int QX>          // QX: -1 = x comes quantised, else the type of x
__global__ __launch_bounds__(512) void mx4_skinny_kernel(const MxParams p) {
  __shared__ float red[8][MF][16][17];
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, r16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, nr = n0 + r16 < p.N ? n0 + r16 : p.N - 1;
  const char* wrow = p.wq + (long long)nr * p.cb + g * 16;
  const unsigned char* wsrow = p.ws + (long long)nr * p.sb + g;
  f32x4_t acc[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) acc[f] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  constexpr int U = MF == 1 ? 4 : 2;               // steps whose loads are in flight together
  for (int kb = wid; kb < p.ksteps; kb += 8 * U) {
    u32x4_t wc[U], xc[U][MF]; int wsc[U], xsc[U][MF];
    raw8<QX < 0 ? CSMRI_BF16 : QX> raw[QX < 0 ? 1 : U][MF][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // a step behind the end: code 0, scale 1
      const int k = kb + 8 * u;
      const bool in = k < p.ksteps;
      wc[u] = (u32x4_t){0, 0, 0, 0}; wsc[u] = 127;
      if (in) { wc[u] = *(const u32x4_t*)(wrow + k * 64); wsc[u] = wsrow[k * 4]; }
#pragma unroll
      for (int f = 0; f < MF; ++f) {
        const long long m = f * 16 + r16;
        xc[u][f] = (u32x4_t){0, 0, 0, 0}; xsc[u][f] = 127;
        if constexpr (QX < 0) {
          if (in && m < p.M) { xc[u][f] = *(const u32x4_t*)(p.xq + m * p.cb + k * 64 + g * 16); xsc[u][f] = p.xs[m * p.sb + k * 4 + g]; }
        } else {
          const int c = k * 128 + g * 32;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            raw[u][f][i] = {};
            if (m < p.M && c + i * 8 < p.K) raw[u][f][i] = ldraw8<QX>(p.x, m * p.xps + c + i * 8);
          }
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < MF; ++f) {
        if constexpr (QX >= 0) xc[u][f] = mx4_pack_block<QX>(raw[u][f], xsc[u][f]);
        acc[f] = mx4_mfma(mx4_operand(wc[u]), wsc[u], mx4_operand(xc[u][f]), xsc[u][f], acc[f]);
      }
  }
  // lane holds outputs n = n0 + 4 g + r of row m = 16 f + r16
#pragma unroll
  for (int f = 0; f < MF; ++f)
#pragma unroll
    for (int r = 0; r < 4; ++r) red[wid][f][r16][4 * g + r] = acc[f][r];
  __syncthreads();
  for (int i = threadIdx.x; i < MF * 64; i += 512) {
    const int m = i >> 2, n4 = (i & 3) * 4;
    if (m >= p.M) continue;
    f32x4_t v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 8; ++w)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] += red[w][m >> 4][m & 15][n4 + k];
    mx4_store(p, m, n0 + n4, v);
  }
}

typedef __attribute__((ext_vector_type(16))) float f32x16_t;

// Many rows: a workgroup of WM x WN waves takes 32 FM WM rows x 32 FN WN outputs.  Codes and scales reach LDS by LDS-DMA,
// 256 channels a stage -- 128 bytes of a row, a cache line -- and two stages: one is read, the next one lands.
// 16384 x 4096 x 4096: 161 us back to back, 3.4 PFLOP/s at the 1.8 GHz that the chip holds under it (187 in a trace of it
// behind its quantisation, 167 on codes); products and fragment reads alone take 98, the loads add 30, the transposed
// stores of bf16 rows 27: time that nothing overlaps, not a bound.  8192^3: 295 us back to back, 3.7 PFLOP/s.  Workgroups that stay and store a tile under the
// next one's products, halves of a workgroup that take turns, and fragments read a quarter of a step ahead took as long.
// The 32 x 32 x 64 form of the matrix instruction, not the 16 x 16 x 128 one: both take the scale operands in an
// instruction slot of their own, which costs the shorter one more of its rate (a loop of nothing else reaches 9.5
// against 6.9 PFLOP/s).
__device__ __forceinline__ int mx_swz(int row) { return (row >> 1) & 7; }     // order of a row's eight 16-byte chunks
typedef __attribute__((address_space(1))) const void* mxg_t;
typedef __attribute__((address_space(3))) void* mxl_t;
// op_sel picks byte U of the scale words
template <int U> __device__ __forceinline__ f32x16_t mx4_mfma32(u32x4_t a, int sa, u32x4_t b, int sb, f32x16_t acc) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(mx4_operand(a), mx4_operand(b), acc, 4, 4, U, sa, U, sb);
}

// A wave's fragments -> out.  acc[i][j] holds outputs 32 i + 8 q + 4 h + (0..3) of row 32 j + r32; they are turned into
// rows of 128 bytes in the wave's own part of LDS, so that a store covers whole lines.
template <int DT, int FM, int FN>
__device__ __forceinline__ void mx4_epilogue(const MxParams& p, long long m0, int n0, const f32x16_t (&acc)[FN][FM], char* img,
                                             const float* bias, int lane) {
  constexpr int NI = DT == CSMRI_F32 ? 1 : 2, CE = DT == CSMRI_F32 ? 4 : 8;     // fragments and outputs per 128 / 16 bytes
  const int r32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int i0 = 0; i0 < FN; i0 += NI) {
#pragma unroll
    for (int i = i0; i < i0 + NI; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const f32x4_t bv = *(const f32x4_t*)(bias + 32 * i + 8 * q + 4 * h);
        const int col = (32 * (i - i0) + 8 * q + 4 * h) * (16 / CE);
#pragma unroll
        for (int j = 0; j < FM; ++j) {
          f32x4_t v;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            v[r] = acc[i][j][4 * q + r] + bv[r];
            v[r] = v[r] > 0.f ? v[r] : v[r] * p.slope;
            if (n0 + 32 * i + 8 * q + 4 * h + r >= p.N) v[r] = 0.f;
          }
          const int row = 32 * j + r32;
          store4(img + row * 128 + (((col >> 4) ^ (row & 7)) << 4) + (col & 15), 0, DT, v);
        }
      }
    const int ch = lane & 7, n = n0 + 32 * i0 + ch * CE;
#pragma unroll
    for (int t = 0; t < FM * 4; ++t) {
      const int row = t * 8 + (lane >> 3);
      const u32x4_t v = *(const u32x4_t*)(img + row * 128 + ((ch ^ (row & 7)) << 4));
      if (m0 + row < p.M && n < p.Npad) *(u32x4_t*)((char*)p.out + ((m0 + row) * p.ops + n) * (16 / CE)) = v;
    }
  }
}

template <int FM, int FN, int WM, int WN, int OCC>
__global__ __launch_bounds__(64 * WM * WN, OCC) void mx4_gemm_kernel(const MxParams p) {
  constexpr int NW = WM * WN, BM = 32 * FM * WM, BN = 32 * FN * WN, STG = (BM + BN) * 128, SCL = (BM + BN) * 16;
  constexpr int NA = BM / (8 * NW), NB = BN / (8 * NW), NS = ((BM + BN) / 64 + NW - 1) / NW;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  char* sscl = smem + 2 * STG;                             // scales: two groups of 512 channels, 16 bytes a row
  float* sbias = (float*)(sscl + 2 * SCL);
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wid / WN, wn = wid % WN, r32 = lane & 31, h = lane >> 5;
  const int tz = xcd_remap(blockIdx.x, p.mtiles * p.ntiles * p.splits), split = tz / (p.mtiles * p.ntiles);
  const int t = tz - split * p.mtiles * p.ntiles;
  // bands of eight row tiles: what runs on an XCD at one time is about square and shares its operands in L2
  // (8192^3 and 16384 x 4096 x 4096 take 3 % longer in row order; smaller ones as long)
  const int band = t / (8 * p.ntiles), r = t - band * 8 * p.ntiles, bm = min(8, p.mtiles - band * 8);
  const int mt = band * 8 + r % bm, nt = r / bm, k0 = split * p.schunk;
  const long long m0 = (long long)mt * BM; const int n0 = nt * BN;
  const int mrows = p.M - m0 < BM ? (int)(p.M - m0) : BM, nrows = p.N - n0 < BN ? p.N - n0 : BN;
  const char* xb = p.xq + m0 * p.cb + k0 * 64; const char* wb = p.wq + (long long)n0 * p.cb + k0 * 64;
  const unsigned char* xsb = p.xs + m0 * p.sb + k0 * 4; const unsigned char* wsb = p.ws + (long long)n0 * p.sb + k0 * 4;
  // rows behind the end read the tile's last row: their results are not stored.  An LDS-DMA instruction fills 1 KiB (eight
  // rows) in lane order, so the swizzle of a row's chunks is applied to the source
  unsigned xo[NA], wo[NB], so[NS];
  const int drow = wid * 8 + (lane >> 3), dch = (lane & 7) ^ mx_swz(drow);       // (j * NW * 8 rows on: the same swizzle)
#pragma unroll
  for (int j = 0; j < NA; ++j) { const int row = j * NW * 8 + drow; xo[j] = (unsigned)(row < mrows ? row : mrows - 1) * p.cb + dch * 16; }
#pragma unroll
  for (int j = 0; j < NB; ++j) { const int row = j * NW * 8 + drow; wo[j] = (unsigned)(row < nrows ? row : nrows - 1) * p.cb + dch * 16; }
#pragma unroll
  for (int j = 0; j < NS; ++j) {
    const int row = (j * NW + wid) * 64 + lane;            // rows of x, then rows of w
    so[j] = row < BM ? (unsigned)(row < mrows ? row : mrows - 1) * p.sb
                     : (unsigned)(row - BM < nrows ? row - BM : nrows - 1) * p.sb;
  }
  const int K = min(p.schunk, p.ksteps - k0);              // (schunk: whole groups of four, at least one in every split)
  auto issue = [&](int st) {
    char* buf = smem + (st & 1) * STG;
    if ((st & 1) == 0) {
      char* sd = sscl + ((st >> 1) & 1) * SCL;
#pragma unroll
      for (int j = 0; j < NS; ++j) {
        const int first = (j * NW + wid) * 64;
        if ((BM + BN) % (64 * NW) == 0 || first < BM + BN) {
          const unsigned char* b = (first < BM ? xsb : wsb) + (st >> 1) * 16;
          __builtin_amdgcn_global_load_lds((mxg_t)(b + so[j]), (mxl_t)(sd + first * 16), 16, 0, 0);
        }
      }
    }
    // where only half of the stage is left, the lanes of the other half read that one again
    const unsigned back = 2 * st + 1 >= K && dch >= 4 ? 64 : 0;
    const char* xk = xb + st * 128; const char* wk = wb + st * 128;
#pragma unroll
    for (int j = 0; j < NA; ++j)
      __builtin_amdgcn_global_load_lds((mxg_t)(xk + (xo[j] - back)), (mxl_t)(buf + (j * NW + wid) * 1024), 16, 0, 0);
#pragma unroll
    for (int j = 0; j < NB; ++j)
      __builtin_amdgcn_global_load_lds((mxg_t)(wk + (wo[j] - back)), (mxl_t)(buf + BM * 128 + (j * NW + wid) * 1024), 16, 0, 0);
  };
  // lane (r32, h) feeds channels 128 u + 64 f + 32 h .. + 31 of its row to the instruction (u, f): chunk 4 u + 2 f + h
  const int foff = r32 * 128 + ((h ^ mx_swz(r32)) << 4);
  const int xoff = wm * FM * 4096 + foff, woff = BM * 128 + wn * FN * 4096 + foff;
  const int xsoff = (wm * FM * 32 + r32) * 16, wsoff = (BM + wn * FN * 32 + r32) * 16;
  const unsigned sel = 0x06040200u + (unsigned)h * 0x01010101u;   // bytes h and 2 + h of two steps' scale words
  f32x16_t acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  u32x4_t xf[FM][2], wf[FN][2]; int xs[FM], ws[FN];
  auto scale_word = [&](const char* a) {
    const u32x2_t v = *(const u32x2_t*)a;
    return (int)__builtin_amdgcn_perm(v[1], v[0], sel);
  };
  auto load = [&](int s) {                                 // s: step of 128 channels
    const char* buf = smem + ((s >> 1) & 1) * STG;
    if ((s & 1) == 0) {                                    // scales of two steps
      const char* sc = sscl + ((s >> 2) & 1) * SCL + (s & 2) * 4;
#pragma unroll
      for (int i = 0; i < FN; ++i) ws[i] = scale_word(sc + wsoff + i * 512);
#pragma unroll
      for (int j = 0; j < FM; ++j) xs[j] = scale_word(sc + xsoff + j * 512);
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      const int flip = (s & 1) * 64 + f * 32;
#pragma unroll
      for (int i = 0; i < FN; ++i) wf[i][f] = *(const u32x4_t*)(buf + ((woff + i * 4096) ^ flip));
#pragma unroll
      for (int j = 0; j < FM; ++j) xf[j][f] = *(const u32x4_t*)(buf + ((xoff + j * 4096) ^ flip));
    }
  };
#define MX_MUL(B) \
    _Pragma("unroll") for (int j = 0; j < FM; ++j) \
    _Pragma("unroll") for (int i = 0; i < FN; ++i) \
      acc[i][j] = mx4_mfma32<B>(wf[i][(B) & 1], ws[i], xf[j][(B) & 1], xs[j], acc[i][j]);
  auto barrier = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  issue(0);
  for (int i = tid; i < BN; i += 64 * NW) sbias[i] = p.bias && p.splits == 1 && n0 + i < p.N ? p.bias[n0 + i] : 0.f;
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  barrier();
#define MX_STEP(U) \
    { \
      if (U == 0 && k + 2 < K) issue((k >> 1) + 1); \
      load(k + U); \
      MX_MUL(2 * U) \
      MX_MUL(2 * U + 1) \
      if (U == 1) { \
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); \
        barrier(); \
      } \
      if (k + U + 1 >= K) break; \
    }
  for (int k = 0;; k += 2) {
    MX_STEP(0)
    MX_STEP(1)
  }
#undef MX_STEP
#undef MX_MUL
  barrier();
  char* img = smem + wid * FM * 4096;
  if (p.splits > 1) {
    MxParams q = p;                                        // a partial sum: no bias, no activation
    q.out = p.slab + split * p.M * p.Npad; q.ops = p.Npad; q.slope = 1.f;
    mx4_epilogue<CSMRI_F32, FM, FN>(q, m0 + wm * FM * 32, n0 + wn * FN * 32, acc, img, sbias + wn * FN * 32, lane);
  } else if (p.out_dt == CSMRI_BF16) mx4_epilogue<CSMRI_BF16, FM, FN>(p, m0 + wm * FM * 32, n0 + wn * FN * 32, acc, img, sbias + wn * FN * 32, lane);
  else mx4_epilogue<CSMRI_F32, FM, FN>(p, m0 + wm * FM * 32, n0 + wn * FN * 32, acc, img, sbias + wn * FN * 32, lane);
}
template <int FM, int FN, int WM, int WN, int OCC> static int mx4_gemm_launch(MxParams& p, hipStream_t st) {
  constexpr int BM = 32 * FM * WM, BN = 32 * FN * WN, LDS = 2 * (BM + BN) * 128 + 2 * (BM + BN) * 16 + BN * 4;
  static_assert(WM * WN * FM * 4096 <= 2 * (BM + BN) * 128, "the output images share the stages' place");
  auto kern = mx4_gemm_kernel<FM, FN, WM, WN, OCC>;
  const long long mt = (p.M + BM - 1) / BM, nt = (p.N + BN - 1) / BN;
  if (mt * nt * p.splits > 0x7fffffff) return CSMRI_E_UNSUPPORTED;
  p.mtiles = (int)mt; p.ntiles = (int)nt;
  CSMRI_SET_MAX_LDS(kern, LDS);
  hipLaunchKernelGGL(kern, dim3((unsigned)(mt * nt * p.splits)), dim3(64 * WM * WN), LDS, st, p);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}

// split sums -> out, four outputs a thread
__global__ __launch_bounds__(256) void mx4_join_kernel(const MxParams p) {
  const int n4 = p.Npad >> 2;
  const long long total = p.M * n4;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long m = i / n4; const int n = (int)(i - m * n4) * 4;
    const float* s = p.slab + m * p.Npad + n;
    f32x4_t v = *(const f32x4_t*)s;
    for (int z = 1; z < p.splits; ++z) v += *(const f32x4_t*)(s + z * p.M * p.Npad);
    mx4_store(p, m, n, v);
  }
}

// Few rows: up to 64, whose fragments fit one wave, as long as the workgroups of 16 outputs make no more than 1024 sets of
// 16 rows -- each of them reads all of x.  Rows x K x outputs, us here and with the tiles: 64 x 4096 x 4096 11 / 13,
// 33 x 4096 x 4096 8 / 11, 32 x 4096 x 8192 13 / 15, 16 x 1024 x 16384 6.1 / 6.5; beyond 64 x 4096 x 8192 20 / 15,
// 32 x 1024 x 16384 9.2 / 6.6.
static bool mx4_few(long long rows, int N) { return rows <= 64 && (rows + 15) / 16 * ((N + 15LL) / 16) <= 1024; }
// Of these up to 16 rows are quantised in the product itself, by every workgroup again: with 512 workgroups or fewer that
// takes less than a launch and a pass of its own (4 x 4096 x 4096: 6.0, 7.2 us; 8 x 4096 x 8192: 10.6, 10.3;
// 4 x 4096 x 16384: 17.0, 15.0).
static bool mx4_packs(long long rows, int N) { return rows <= 16 && N <= 8192; }
// Splits of the channels for the tiled kernel, where its 128 x 128 tiles leave CUs without one.  A group of 512 channels
// takes a workgroup 1.4 us; joining takes 3.5 us and 0.5 us for each MiB of partial sums (512 x 2048 x 1024 in one part
// 9.3 us, in four 12.3; 512 x 8192 x 2048 26 and 21; 128 x 16384 x 4096 in eight parts 18, in one 49): the least
// sum of these, in quarters of a group.
static int mx4_splits(long long rows, int K, int N) {
  if (mx4_few(rows, N)) return 1;
  const long long tiles = ((rows + 127) / 128) * ((N + 127LL) / 128), npad = (N + 7LL) / 8 * 8;
  const int groups = (int)((K + 511LL) / 512);
  if (tiles > 128) return 1;
  const int most = (int)(256 / tiles) < groups ? (int)(256 / tiles) : groups;
  int best = 1; long long least = 4LL * groups;
  for (int s = 2; s <= most; ++s) {
    const int per = (groups + s - 1) / s, n = (groups + per - 1) / per;
    const long long cost = 4LL * per + 10 + ((6 * n * rows * npad) >> 20);
    if (cost < least) { least = cost; best = n; }
  }
  return best;
}
// The 256 x 256 tile reads each operand half as often and has a CU to itself; two of the 128 x 128 ones share one.  At 4096
// channels a round of 256 large tiles takes 40 us, 512 small ones 24 us and 6 us for the first and last, and those need
// not come in whole rounds.  us with large tiles and with small ones, back to back: 16384 x 4096 x 4096 161 / 191, 8192^3
// 294 / 360, 4096^3 42 / 49, 3584 x 4096 x 4096 39 / 45; 2048 x 4096 x 4096 34 / 26, 16384 x 2048 x 1100 41 / 33,
// 131072 x 512 x 128 24 / 17.
static bool mx4_large(long long rows, int N) {
  const long long small = ((rows + 127) / 128) * ((N + 127LL) / 128), big = ((rows + 255) / 256) * ((N + 255LL) / 256);
  return 40 * 512 * ((big + 255) / 256) < 6 * 512 + 24 * small;
}
static size_t mx4_quant_bytes(int x_dtype, long long rows, int K, int N) {
  return x_dtype == CSMRI_MX4 || mx4_packs(rows, N) ? 0 : (size_t)rows * (mx4_code_bytes(K) + mx4_scale_bytes(K));
}
extern "C" size_t csmri_mx4_linear_work_bytes(int x_dtype, long long rows, int K, int N) {
  if (rows <= 0 || K <= 0 || N <= 0) return 0;
  const int s = mx4_splits(rows, K, N);
  return mx4_quant_bytes(x_dtype, rows, K, N) + (s > 1 ? (size_t)s * rows * ((N + 7) / 8 * 8) * sizeof(float) : 0);
}

extern "C" int csmri_mx4_linear(int x_dtype, const void* x, int x_pix_stride, const uint8_t* x_scales, long long rows, int K,
                                const void* w_codes, const uint8_t* w_scales, int N, const float* bias, float slope,
                                void* out, int out_dtype, int out_pix_stride, void* work, void* stream) {
  CSMRI_CHECK_ARG(rows >= 0 && K > 0 && K % 8 == 0 && K <= MX4_MAX_K && N > 0 && N <= 0x7ffffff0 && (out_dtype == CSMRI_F32 || out_dtype == CSMRI_BF16));
  const int npad = (N + 7) / 8 * 8;
  CSMRI_CHECK_ARG(out_pix_stride >= npad && w_codes && w_scales);
  CSMRI_CHECK_ARG(x_dtype == CSMRI_MX4 ? true : mx4_shape_ok(rows, K, x_pix_stride, x_dtype));
  if (rows == 0) return CSMRI_OK;
  CSMRI_CHECK_ARG(x && out && (x_dtype != CSMRI_MX4 || x_scales));
  CSMRI_CHECK_ARG(csmri_mx4_linear_work_bytes(x_dtype, rows, K, N) == 0 || work);
  if ((((uintptr_t)w_codes | (uintptr_t)w_scales | (uintptr_t)work | (uintptr_t)x_scales) & 15) ||
      !mx4_rows_aligned(out, out_pix_stride, out_dtype) ||
      (x_dtype == CSMRI_MX4 ? ((uintptr_t)x & 15) != 0 : !mx4_rows_aligned(x, x_pix_stride, x_dtype))) return CSMRI_E_ALIGN;
  MxParams p = {};
  p.x = x; p.xps = x_pix_stride;
  p.wq = (const char*)w_codes; p.ws = w_scales;
  p.bias = bias; p.slope = slope;
  p.out = out; p.out_dt = out_dtype; p.ops = out_pix_stride;
  p.M = rows; p.N = N; p.Npad = npad; p.K = K;
  p.cb = mx4_code_bytes(K); p.sb = mx4_scale_bytes(K); p.ksteps = p.cb / 64;
  hipStream_t st = (hipStream_t)stream;
  if (x_dtype == CSMRI_MX4) {
    p.xq = (const char*)x; p.xs = x_scales;
  } else if (!mx4_packs(rows, N)) {
    p.xq = (const char*)work; p.xs = (const unsigned char*)work + (size_t)rows * p.cb;
    const int rc = csmri_mx4_quantize(x_dtype, x, x_pix_stride, rows, K, (void*)p.xq, (uint8_t*)p.xs, stream);
    if (rc != CSMRI_OK) return rc;
  }
  if (mx4_few(rows, N)) {
    const dim3 g((npad + 15) / 16), b(512);
    if (!p.xq) {
      if (x_dtype == CSMRI_F32) hipLaunchKernelGGL((mx4_skinny_kernel<1, CSMRI_F32>), g, b, 0, st, p);
      else hipLaunchKernelGGL((mx4_skinny_kernel<1, CSMRI_BF16>), g, b, 0, st, p);
    } else if (rows <= 16) hipLaunchKernelGGL((mx4_skinny_kernel<1, -1>), g, b, 0, st, p);
    else if (rows <= 32) hipLaunchKernelGGL((mx4_skinny_kernel<2, -1>), g, b, 0, st, p);
    else hipLaunchKernelGGL((mx4_skinny_kernel<4, -1>), g, b, 0, st, p);
    CSMRI_LAUNCH_CHECK();
    return CSMRI_OK;
  }
  p.splits = mx4_splits(rows, K, N);
  p.schunk = p.splits > 1 ? 4 * (((K + 511) / 512 + p.splits - 1) / p.splits) : p.ksteps;
  p.slab = (float*)((char*)work + mx4_quant_bytes(x_dtype, rows, K, N));
  const int rc = mx4_large(rows, N) ? mx4_gemm_launch<4, 2, 2, 4, 2>(p, st) : mx4_gemm_launch<2, 2, 2, 2, 2>(p, st);
  if (rc != CSMRI_OK || p.splits == 1) return rc;
  const long long blocks = (rows * (npad / 4) + 255) / 256;
  hipLaunchKernelGGL(mx4_join_kernel, dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st, p);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}
