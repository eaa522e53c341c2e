// Microscaled 4-bit operands (micro.h: e2m1 elements, one E8M0 scale per 32 consecutive channels) and the product of a
// 1 x 1 convolution on them:
//
//   y[p][n] = act( sum_c xq[p][c] wq[n][c] + bias[n] ),  xq, wq the values the 4-bit forms stand for
//
// A row of K channels is 64 bytes of codes per 128 channels (two a byte, the even channel in the low half) and one scale
// byte per 32 channels, padded to 16 bytes per 512 channels; padding is code 0, scale 2^0.  The contraction is
// v_mfma_scale_f32_16x16x128_f8f6f4: a lane's operand is 32 channels of one row, exactly one block, so its scale rides
// in the lane next to it.  Products and sums are exact to fp32 (the elements are multiples of 1/2 up to 6).
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
__device__ __forceinline__ i32x8_t mx4_operand(u32x4_t c) {
  return (i32x8_t){(int)c[0], (int)c[1], (int)c[2], (int)c[3], 0, 0, 0, 0};
}
__device__ __forceinline__ f32x4_t mx4_mfma(i32x8_t a, int sa, i32x8_t b, int sb, f32x4_t acc) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, 4, 0, sa, 0, sb);
}

// ---- quantise / dequantise: one read, one write, bound by HBM ---------------------------------------------------------
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
      // scale 1 here: the factor is applied as an fp32 product, exact, and a NaN scale byte becomes a NaN factor
      const float f = sc[u] == MICRO_NAN ? __uint_as_float(0x7fc00000u) : (sc[u] ? micro_scale(sc[u]) : __uint_as_float(0x00400000u));
      auto t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 0); v[0] = t[0] * f; v[1] = t[1] * f;
      t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 1); v[2] = t[0] * f; v[3] = t[1] * f;
      t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 2); v[4] = t[0] * f; v[5] = t[1] * f;
      t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c[u], 1.f, 3); v[6] = t[0] * f; v[7] = t[1] * f;
      st8<DT>(out, (row + u * step) * ps + slot * 8, v);
    }
  }
}

static bool mx4_shape_ok(long long rows, int K, int ps, int dtype) {
  return rows >= 0 && K > 0 && K % 8 == 0 && ps >= K && (dtype == CSMRI_F32 || dtype == CSMRI_BF16);
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

// Few rows (up to 16 MF): bound by the weights' bytes.  A workgroup of eight waves owns 16 outputs; the waves split the
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
  for (int k = wid; k < p.ksteps; k += 8) {
    const i32x8_t wv = mx4_operand(*(const u32x4_t*)(wrow + k * 64));
    const int wsc = wsrow[k * 4];
#pragma unroll
    for (int f = 0; f < MF; ++f) {
      const long long m = f * 16 + r16;
      u32x4_t xc = {0, 0, 0, 0}; int xsc = 127;
      if constexpr (QX < 0) {
        if (m < p.M) { xc = *(const u32x4_t*)(p.xq + m * p.cb + k * 64 + g * 16); xsc = p.xs[m * p.sb + k * 4 + g]; }
      } else {
        const int c = k * 128 + g * 32;
        float v[4][8];
        unsigned amax = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          raw8<QX> raw = raw8<QX>{};
          if (m < p.M && c + i * 8 < p.K) raw = ldraw8<QX>(p.x, m * p.xps + c + i * 8);
          cvt8<QX>(raw, v[i]);
#pragma unroll
          for (int q = 0; q < 8; ++q) { const unsigned a = abs_bits(v[i][q]); amax = a > amax ? a : amax; }
        }
        const int e = micro_exp(amax) - 2;
        const bool fin = micro_finite(amax);
        const float s = exp2i(fin ? e : 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) xc[i] = mx4_pack8(v[i], s);
        xsc = fin ? e + 127 : MICRO_NAN;
      }
      acc[f] = mx4_mfma(wv, wsc, mx4_operand(xc), xsc, acc[f]);
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

// 128 rows x 128 outputs per workgroup, 4 waves of 64 x 64, both operands through LDS, 128 channels a step
__device__ __forceinline__ int mx_off(int row, int chunk) { return row * 64 + ((chunk ^ ((4 - ((row >> 2) & 3)) & 3)) << 4); }
__global__ __launch_bounds__(256) void mx4_gemm_kernel(const MxParams p) {
  constexpr int BM = 128, BN = 128, IMG = 128 * 64;
  __shared__ __attribute__((aligned(16))) char smem[2 * IMG];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wm = wid >> 1, wn = wid & 1, r16 = lane & 15, g = lane >> 4;
  const int t = xcd_remap(blockIdx.x, p.mtiles * p.ntiles);
  const int mt = t / p.ntiles, nt = t - mt * p.ntiles;
  const long long m0 = (long long)mt * BM; const int n0 = nt * BN;
  // staging: two 16-byte chunks a thread and image; rows behind the end read the last row, their results are not stored
  const char* xsrc[2]; const char* wsrc[2]; int off[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int id = j * 256 + tid, row = id >> 2, ch = id & 3;
    const long long m = m0 + row < p.M ? m0 + row : p.M - 1;
    const int n = n0 + row < p.N ? n0 + row : p.N - 1;
    xsrc[j] = p.xq + m * p.cb + ch * 16;
    wsrc[j] = p.wq + (long long)n * p.cb + ch * 16;
    off[j] = mx_off(row, ch);
  }
  const unsigned char* xsc[4]; const unsigned char* wsc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long m = m0 + wm * 64 + i * 16 + r16;
    const int n = n0 + wn * 64 + i * 16 + r16;
    xsc[i] = p.xs + (m < p.M ? m : p.M - 1) * p.sb + g;
    wsc[i] = p.ws + (long long)(n < p.N ? n : p.N - 1) * p.sb + g;
  }
  f32x4_t acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  for (int k = 0; k < p.ksteps; ++k) {
    u32x4_t xv[2], wv[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) { xv[j] = *(const u32x4_t*)(xsrc[j] + k * 64); wv[j] = *(const u32x4_t*)(wsrc[j] + k * 64); }
    int xs[4], ws[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { xs[i] = xsc[i][k * 4]; ws[i] = wsc[i][k * 4]; }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; ++j) { *(u32x4_t*)(smem + off[j]) = xv[j]; *(u32x4_t*)(smem + IMG + off[j]) = wv[j]; }
    __syncthreads();
    i32x8_t xf[4], wf[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      xf[i] = mx4_operand(*(const u32x4_t*)(smem + mx_off(wm * 64 + i * 16 + r16, g)));
      wf[i] = mx4_operand(*(const u32x4_t*)(smem + IMG + mx_off(wn * 64 + i * 16 + r16, g)));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = mx4_mfma(wf[i], ws[i], xf[j], xs[j], acc[i][j]);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long m = m0 + wm * 64 + j * 16 + r16;
    if (m >= p.M) continue;
#pragma unroll
    for (int i = 0; i < 4; ++i) mx4_store(p, m, n0 + wn * 64 + i * 16 + 4 * g, acc[i][j]);
  }
}

#define MX4_QUANT_ROWS 16      // up to here the product quantises x itself
extern "C" size_t csmri_mx4_linear_work_bytes(int x_dtype, long long rows, int K) {
  if (x_dtype == CSMRI_MX4 || rows <= MX4_QUANT_ROWS || K <= 0) return 0;
  return (size_t)rows * (mx4_code_bytes(K) + mx4_scale_bytes(K));
}

extern "C" int csmri_mx4_linear(int x_dtype, const void* x, int x_pix_stride, const uint8_t* x_scales, long long rows, int K,
                                const void* w_codes, const uint8_t* w_scales, int N, const float* bias, float slope,
                                void* out, int out_dtype, int out_pix_stride, void* work, void* stream) {
  CSMRI_CHECK_ARG(rows >= 0 && K > 0 && K % 8 == 0 && N > 0 && N <= 0x7ffffff0 && (out_dtype == CSMRI_F32 || out_dtype == CSMRI_BF16));
  const int npad = (N + 7) / 8 * 8;
  CSMRI_CHECK_ARG(out_pix_stride >= npad && w_codes && w_scales);
  CSMRI_CHECK_ARG(x_dtype == CSMRI_MX4 ? true : mx4_shape_ok(rows, K, x_pix_stride, x_dtype));
  if (rows == 0) return CSMRI_OK;
  CSMRI_CHECK_ARG(x && out && (x_dtype != CSMRI_MX4 || x_scales));
  CSMRI_CHECK_ARG(csmri_mx4_linear_work_bytes(x_dtype, rows, K) == 0 || work);
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
  } else if (rows > MX4_QUANT_ROWS) {
    p.xq = (const char*)work; p.xs = (const unsigned char*)work + (size_t)rows * p.cb;
    const int rc = csmri_mx4_quantize(x_dtype, x, x_pix_stride, rows, K, (void*)p.xq, (uint8_t*)p.xs, stream);
    if (rc != CSMRI_OK) return rc;
  }
  if (rows <= 64) {
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
  const long long mt = (rows + 127) / 128, nt = (npad + 127) / 128;
  if (mt * nt > 0x7fffffff) return CSMRI_E_UNSUPPORTED;
  p.mtiles = (int)mt; p.ntiles = (int)nt;
  hipLaunchKernelGGL(mx4_gemm_kernel, dim3((unsigned)(mt * nt)), dim3(256), 0, st, p);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}
