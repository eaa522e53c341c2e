// Activations kept for the backward pass in 8 bits (micro.h: e4m3 elements, one power-of-two scale per 32 channels of a
// pixel: 1.03 bytes a channel instead of 2 or 4), and the weight gradient of a 1 x 1 convolution that reads them.
//
// Save and restore are streams: one read, one write, bound by HBM.
#include "micro.h"
#include "wgrad_params.h"

template <int DT>
__global__ __launch_bounds__(256) void act8_save_kernel(const void* __restrict__ x, int ps, long long rows, int c8,
                                                        int blocks, int cols, int rpt, unsigned char* __restrict__ q,
                                                        unsigned char* __restrict__ s) {
  constexpr int U = 4;
  const int slot = blockIdx.y * cols + threadIdx.x % cols, r0 = threadIdx.x / cols;
  const bool live = r0 < rpt && slot < blocks * 4, load = live && slot < c8;
  const long long step = (long long)gridDim.x * rpt;
  for (long long row = (long long)blockIdx.x * rpt + r0; row - r0 < rows; row += step * U) {
    raw8<DT> raw[U];
    // the four lanes of a block share row and liveness, so the shuffles below meet only lanes of the same state
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
      unsigned char sc;
      const u32x2_t o = micro_pack8(v, amax, sc);
      if (load && rr < rows) {
        *(u32x2_t*)(q + rr * c8 * 8 + slot * 8) = o;
        if ((slot & 3) == 0) s[rr * blocks + (slot >> 2)] = sc;
      }
    }
  }
}

template <int DT>
__global__ __launch_bounds__(256) void act8_restore_kernel(const unsigned char* __restrict__ q,
                                                           const unsigned char* __restrict__ s, long long rows, int c8,
                                                           int blocks, int cols, int rpt, void* __restrict__ out, int ps) {
  constexpr int U = 4;
  const int slot = blockIdx.y * cols + threadIdx.x % cols, r0 = threadIdx.x / cols;
  if (r0 >= rpt || slot >= c8) return;
  const long long step = (long long)gridDim.x * rpt;
  for (long long row = (long long)blockIdx.x * rpt + r0; row < rows; row += step * U) {
    u32x2_t c[U]; unsigned char sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step < rows ? row + u * step : row;
      c[u] = *(const u32x2_t*)(q + rr * c8 * 8 + slot * 8);
      sc[u] = s[rr * blocks + (slot >> 2)];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (row + u * step >= rows) break;
      float v[8];
      micro_unpack8(c[u], micro_scale(sc[u]), v);
      st8<DT>(out, (row + u * step) * ps + slot * 8, v);
    }
  }
}

static bool act8_shape_ok(long long npix, int C) { return npix >= 0 && C > 0 && C % 8 == 0; }

extern "C" int csmri_act8_save(int dtype, const void* x, int x_pix_stride, long long npix, int C, void* q8, uint8_t* s8,
                               void* stream) {
  CSMRI_CHECK_ARG(act8_shape_ok(npix, C) && x_pix_stride >= C && (dtype == CSMRI_F32 || dtype == CSMRI_BF16));
  if (npix == 0) return CSMRI_OK;
  CSMRI_CHECK_ARG(x && q8 && s8);
  if (((uintptr_t)x & 15) || ((uintptr_t)q8 & 7) || ((long long)x_pix_stride * dtype_size(dtype)) % 16) return CSMRI_E_ALIGN;
  const int blocks = (C + MICRO_BLOCK - 1) / MICRO_BLOCK;
  const RowWalk w = row_walk(blocks * 4);
  const dim3 grid = row_walk_grid(npix, blocks * 4, 4);
  auto kern = dtype == CSMRI_F32 ? act8_save_kernel<CSMRI_F32> : act8_save_kernel<CSMRI_BF16>;
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, (hipStream_t)stream, x, x_pix_stride, npix, C / 8, blocks, w.cols,
                     w.rows_per_tile, (unsigned char*)q8, (unsigned char*)s8);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}

extern "C" int csmri_act8_restore(const void* q8, const uint8_t* s8, long long npix, int C, int dtype, void* out,
                                  int out_pix_stride, void* stream) {
  CSMRI_CHECK_ARG(act8_shape_ok(npix, C) && out_pix_stride >= C && (dtype == CSMRI_F32 || dtype == CSMRI_BF16));
  if (npix == 0) return CSMRI_OK;
  CSMRI_CHECK_ARG(q8 && s8 && out);
  if (((uintptr_t)out & 15) || ((uintptr_t)q8 & 7) || ((long long)out_pix_stride * dtype_size(dtype)) % 16) return CSMRI_E_ALIGN;
  const int blocks = (C + MICRO_BLOCK - 1) / MICRO_BLOCK;
  const RowWalk w = row_walk(blocks * 4);
  const dim3 grid = row_walk_grid(npix, blocks * 4, 4);
  auto kern = dtype == CSMRI_F32 ? act8_restore_kernel<CSMRI_F32> : act8_restore_kernel<CSMRI_BF16>;
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, (hipStream_t)stream, (const unsigned char*)q8, (const unsigned char*)s8,
                     npix, C / 8, blocks, w.cols, w.rows_per_tile, out, out_pix_stride);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}

// ---- column sums of partial rows ------------------------------------------------------------------------------------
// 16 columns x 64 row lanes per workgroup: the few columns of a narrow layer still spread their rows over 64 loads in
// flight, and a row's 64 bytes are one sector.
__global__ __launch_bounds__(1024) void colsum_rows_kernel(const float* __restrict__ partial, int rows,
                                                           long long row_stride, long long cols,
                                                           float* __restrict__ out, int accumulate) {
  __shared__ float red[64][17];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
  const long long col = (long long)blockIdx.x * 16 + cl;
  float a = 0.f;
  if (col < cols) {
    int r = rl;
    for (; r + 192 < rows; r += 256) {
      float t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) t[u] = partial[(long long)(r + 64 * u) * row_stride + col];
      a += (t[0] + t[1]) + (t[2] + t[3]);
    }
    for (; r < rows; r += 64) a += partial[(long long)r * row_stride + col];
  }
  red[rl][cl] = a;
  __syncthreads();
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    if (rl < o) red[rl][cl] += red[rl + o][cl];
    __syncthreads();
  }
  if (rl == 0 && col < cols) out[col] = (accumulate ? out[col] : 0.f) + red[0][cl];
}
int micro_colsum(const float* partial, int rows, long long row_stride, long long cols, float* out, int accumulate,
                 hipStream_t st) {
  const long long grid = (cols + 15) / 16;
  hipLaunchKernelGGL(colsum_rows_kernel, dim3((unsigned)grid), dim3(1024), 0, st, partial, rows, row_stride, cols, out,
                     accumulate);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}

// ---- weight gradient of a 1 x 1 convolution ---------------------------------------------------------------------------
//   dW[n][c] = sum_p dY[p][n] * Xhat[p][c],  db[n] = sum_p dY[p][n]
// An e4m3 element times its power-of-two scale is a bf16 number exactly, so the kept activations enter
// v_mfma_f32_16x16x32_bf16 without a rounding of their own; an fp32 dY is split into three bf16 parts whose sum is
// exact, three products each.  The sum runs over pixels, the strided direction of both operands: LDS images keep
// [pixel][channel] and ds_read_b64_tr_b16 hands out the pixel-contiguous fragments.
struct A8WParams {
  const char* dy; int dyps;
  const unsigned char* q; const unsigned char* s;
  long long npix, chunk;           // chunk: pixels per split
  int Cout, Cin, Cout_real, Cin_real, ntiles, ctiles, splits;
  float* slab;                     // [splits][Cout_real * Cin_real + Cout_real] when splits > 1
  float* dw; float* db; int accumulate;
};

// three bf16 parts of eight floats: f = h + m + l exactly
__device__ __forceinline__ void split3(const float* f, u32x4_t* o) {
  float h[8], m[8], l[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    h[k] = (float)(__bf16)f[k];
    const float r = f[k] - h[k];
    m[k] = (float)(__bf16)r;
    l[k] = r - m[k];
  }
  const float* part[3] = {h, m, l};
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const u32x2_t a = pack4_bf16((f32x4_t){part[i][0], part[i][1], part[i][2], part[i][3]});
    const u32x2_t b = pack4_bf16((f32x4_t){part[i][4], part[i][5], part[i][6], part[i][7]});
    o[i] = (u32x4_t){a[0], a[1], b[0], b[1]};
  }
}

// BT x BT tile (BT output channels x BT input channels), KP pixels per step, 4 waves in 2 x 2
template <int DT, int BT>
__global__ __launch_bounds__(256) void act8_wgrad_kernel(const A8WParams p) {
  constexpr int KP = 32, CPR = BT / 8, PL = DT == CSMRI_F32 ? 3 : 1;
  constexpr int IMG = KP * BT * 2, NCH = KP * CPR / 256;        // chunks of 8 channels per thread and image
  constexpr int F = BT / 32;
  __shared__ __attribute__((aligned(16))) char smem[IMG * (PL + 1)];
  char* xi = smem + IMG * PL;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, wn = wid >> 1, wc = wid & 1;
  const int tiles = p.ntiles * p.ctiles;
  const int tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
  const int nt = tile / p.ctiles, ct = tile - nt * p.ctiles;
  const int n0 = nt * BT, c0 = ct * BT;
  const long long pb = split * p.chunk, pe = pb + p.chunk < p.npix ? pb + p.chunk : p.npix;
  const int sblocks = (p.Cin + MICRO_BLOCK - 1) / MICRO_BLOCK;

  f32x4_t acc[F][F], accb[F];
#pragma unroll
  for (int i = 0; i < F; ++i) {
    accb[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < F; ++j) acc[i][j] = accb[i];
  }
  const bool want_b = p.db && ct == 0 && wc == 0;
  const bf16x8_t ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};
  // fragment addresses: a 16-lane group reads 4 pixel rows x 16 channels
  const int g = lane >> 4, tr = (lane & 15) >> 2, tc = lane & 3;

  for (long long k0 = pb; k0 < pe; k0 += KP) {
    raw8<DT> dv[NCH]; u32x2_t xv[NCH]; unsigned char sv[NCH];
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int id = j * 256 + tid, row = id / CPR, ch = id % CPR;
      const long long pix = k0 + row;
      const bool ok = pix < pe;
      dv[j] = raw8<DT>{}; xv[j] = (u32x2_t){0, 0}; sv[j] = 0;
      if (ok && n0 + ch * 8 < p.Cout) dv[j] = ldraw8<DT>(p.dy, pix * p.dyps + n0 + ch * 8);
      if (ok && c0 + ch * 8 < p.Cin) {
        xv[j] = *(const u32x2_t*)(p.q + pix * p.Cin + c0 + ch * 8);
        sv[j] = p.s[pix * sblocks + ((c0 + ch * 8) >> 5)];
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NCH; ++j) {
      const int id = j * 256 + tid, row = id / CPR, ch = id % CPR, off = img_off<CPR>(row, ch);
      if constexpr (DT == CSMRI_F32) {
        float f[8]; u32x4_t o[3];
        cvt8<DT>(dv[j], f);
        split3(f, o);
#pragma unroll
        for (int i = 0; i < 3; ++i) *(u32x4_t*)(smem + i * IMG + off) = o[i];
      } else {
        *(u32x4_t*)(smem + off) = dv[j].a;
      }
      float v[8];
      micro_unpack8(xv[j], micro_scale(sv[j]), v);
      st8<CSMRI_BF16>(xi + off, 0, v);
    }
    __syncthreads();
    bf16x8_t xf[F];
    // pixel rows 8 g + (0..3) and 8 g + (4..7) of the step, 16 channels each
    const int lo = 8 * g + tr, hi = lo + 4;
#pragma unroll
    for (int j = 0; j < F; ++j) {
      const int ch = (wc * (BT / 2) + j * 16) / 8 + (tc >> 1), in = (tc & 1) * 8;
      xf[j] = tr_frag(xi, img_off<CPR>(lo, ch) + in, img_off<CPR>(hi, ch) + in);
    }
#pragma unroll
    for (int pl = 0; pl < PL; ++pl)
#pragma unroll
      for (int i = 0; i < F; ++i) {
        const int ch = (wn * (BT / 2) + i * 16) / 8 + (tc >> 1), in = (tc & 1) * 8;
        const bf16x8_t yf = tr_frag(smem + pl * IMG, img_off<CPR>(lo, ch) + in, img_off<CPR>(hi, ch) + in);
#pragma unroll
        for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(yf, xf[j], acc[i][j], 0, 0, 0);
        if (want_b) accb[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(yf, ones, accb[i], 0, 0, 0);
      }
  }
  // lane l holds rows n = 4 g + r, column c = l & 15 of each fragment
  const long long len = (long long)p.Cout_real * p.Cin_real;
  float* dw = p.splits > 1 ? p.slab + split * (len + p.Cout_real) : p.dw;
  float* db = p.splits > 1 ? dw + len : p.db;
  const bool add = p.splits == 1 && p.accumulate;
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + wn * (BT / 2) + i * 16 + 4 * g + r;
      if (n >= p.Cout_real) continue;
#pragma unroll
      for (int j = 0; j < F; ++j) {
        const int c = c0 + wc * (BT / 2) + j * 16 + (lane & 15);
        if (c >= p.Cin_real) continue;
        float* o = dw + (long long)n * p.Cin_real + c;
        *o = acc[i][j][r] + (add ? *o : 0.f);
      }
      if (want_b && (lane & 15) == 0) db[n] = accb[i][r] + (add ? db[n] : 0.f);
    }
}

static int a8w_tile(int Cout, int Cin) { return Cout <= 64 || Cin <= 64 ? 64 : 128; }
extern "C" int csmri_act8_wgrad_splits(long long npix, int Cout, int Cin) {
  if (npix <= 0 || Cout <= 0 || Cin <= 0) return 1;
  const int bt = a8w_tile(Cout, Cin);
  const long long tiles = (long long)cdiv(Cout, bt) * cdiv(Cin, bt);
  long long s = 512 / tiles;                                  // two workgroups a CU
  const long long most = npix / 256;                          // at least eight steps each
  if (s > most) s = most;
  return s < 1 ? 1 : (int)s;
}
extern "C" size_t csmri_act8_wgrad_slab_bytes(int splits, int Cout_real, int Cin_real) {
  return splits > 1 ? (size_t)splits * ((size_t)Cout_real * Cin_real + Cout_real) * sizeof(float) : 0;
}
extern "C" int csmri_act8_wgrad(int dy_dtype, const void* dy, int dy_pix_stride, const void* q8, const uint8_t* s8,
                                long long npix, int Cout, int Cin, int Cout_real, int Cin_real, int splits, float* slab,
                                float* dw, float* db, int accumulate, void* stream) {
  CSMRI_CHECK_ARG(npix >= 0 && Cout > 0 && Cin > 0 && Cout % 8 == 0 && Cin % 8 == 0 && Cout_real > 0 && Cout_real <= Cout &&
                  Cin_real > 0 && Cin_real <= Cin && dy_pix_stride >= Cout && splits >= 1 && dw &&
                  (dy_dtype == CSMRI_F32 || dy_dtype == CSMRI_BF16));
  hipStream_t st = (hipStream_t)stream;
  CSMRI_CHECK_ARG(npix == 0 || (dy && q8 && s8));
  CSMRI_CHECK_ARG(splits == 1 || (slab && splits <= npix));
  if (npix && (((uintptr_t)dy & 15) || ((uintptr_t)q8 & 7) || ((long long)dy_pix_stride * dtype_size(dy_dtype)) % 16)) return CSMRI_E_ALIGN;
  A8WParams p = {};
  p.dy = (const char*)dy; p.dyps = dy_pix_stride;
  p.q = (const unsigned char*)q8; p.s = (const unsigned char*)s8;
  p.npix = npix;
  p.Cout = Cout; p.Cin = Cin; p.Cout_real = Cout_real; p.Cin_real = Cin_real;
  const int bt = a8w_tile(Cout, Cin);
  p.ntiles = cdiv(Cout, bt); p.ctiles = cdiv(Cin, bt);
  p.splits = splits; p.slab = slab; p.dw = dw; p.db = db; p.accumulate = accumulate;
  p.chunk = ((npix + splits - 1) / splits + 31) / 32 * 32;
  const long long grid = (long long)p.ntiles * p.ctiles * splits;
  if (grid > 0x7fffffff) return CSMRI_E_UNSUPPORTED;
  auto kern = dy_dtype == CSMRI_F32 ? (bt == 64 ? act8_wgrad_kernel<CSMRI_F32, 64> : act8_wgrad_kernel<CSMRI_F32, 128>)
                                    : (bt == 64 ? act8_wgrad_kernel<CSMRI_BF16, 64> : act8_wgrad_kernel<CSMRI_BF16, 128>);
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), 0, st, p);
  CSMRI_LAUNCH_CHECK();
  if (splits > 1) {
    const long long len = (long long)Cout_real * Cin_real;
    int rc = micro_colsum(slab, splits, len + Cout_real, len, dw, accumulate, st);
    if (rc == CSMRI_OK && db) rc = micro_colsum(slab + len, splits, len + Cout_real, Cout_real, db, accumulate, st);
    return rc;
  }
  return CSMRI_OK;
}
