// Activations kept for the backward pass in 8 bits (micro.h: e4m3 elements, one power-of-two scale per 32 channels of a
// pixel: 1.03 bytes a channel instead of 2 or 4), and the weight gradient of a 1 x 1 convolution that reads them.
//
// Save and restore are streams: one read, one write, bound by HBM (16384 x 2048 bf16: 18 us for 102 MB; 131072 x 64: 6.1 and
// 6.0 us for 25 MB, a third of it the launch).  A thread keeps its channels and has four rows under way.
#include "micro.h"
#include "wgrad_params.h"
#include <type_traits>

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
// Columns [0, na) go to oa, [na, na + nb) to ob.  Many rows of few columns: 16 columns x 64 row lanes per workgroup, so
// that the loads of a column spread over the lanes, and a row's 64 bytes are one sector.
__global__ __launch_bounds__(1024) void colsum_rows_kernel(const float* __restrict__ partial, int rows, long long row_stride,
                                                           long long na, float* __restrict__ oa, long long nb,
                                                           float* __restrict__ ob, int accumulate) {
  __shared__ float red[64][17];
  const int cl = threadIdx.x & 15, rl = threadIdx.x >> 4;
  const long long col = (long long)blockIdx.x * 16 + cl;
  float a = 0.f;
  if (col < na + nb) {
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
  if (rl == 0 && col < na + nb) {
    float* o = col < na ? oa + col : ob + (col - na);
    *o = (accumulate ? *o : 0.f) + red[0][cl];
  }
}
// Few rows of many columns: a thread per column, its rows' loads in batches of four.
__global__ __launch_bounds__(256) void colsum_cols_kernel(const float* __restrict__ partial, int rows, long long row_stride,
                                                          long long na, float* __restrict__ oa, long long nb,
                                                          float* __restrict__ ob, int accumulate) {
  for (long long col = (long long)blockIdx.x * 256 + threadIdx.x; col < na + nb; col += (long long)gridDim.x * 256) {
    float a = 0.f;
    int r = 0;
    for (; r + 4 <= rows; r += 4) {
      float t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) t[u] = partial[(long long)(r + u) * row_stride + col];
      a += (t[0] + t[1]) + (t[2] + t[3]);
    }
    for (; r < rows; ++r) a += partial[(long long)r * row_stride + col];
    float* o = col < na ? oa + col : ob + (col - na);
    *o = (accumulate ? *o : 0.f) + a;
  }
}
int micro_colsum2(const float* partial, int rows, long long row_stride, long long na, float* oa, long long nb, float* ob,
                  int accumulate, hipStream_t st) {
  const long long cols = na + nb;
  if (rows > 16 && cols <= 65536) {
    hipLaunchKernelGGL(colsum_rows_kernel, dim3((unsigned)((cols + 15) / 16)), dim3(1024), 0, st, partial, rows, row_stride,
                       na, oa, nb, ob, accumulate);
  } else {
    const long long want = (cols + 255) / 256;
    hipLaunchKernelGGL(colsum_cols_kernel, dim3((unsigned)(want < 8192 ? want : 8192)), dim3(256), 0, st, partial, rows,
                       row_stride, na, oa, nb, ob, accumulate);
  }
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}

// ---- weight gradient of a 1 x 1 convolution ---------------------------------------------------------------------------
//   dW[n][c] = sum_p dY[p][n] * Xhat[p][c],  db[n] = sum_p dY[p][n]
// An e4m3 element times its power-of-two scale is a bf16 number exactly, so the kept activations enter
// v_mfma_f32_16x16x32_bf16 without a rounding of their own; an fp32 dY is split into three bf16 parts (split3), three
// products each.  The sum runs over pixels, the strided direction of both operands: LDS images keep
// [pixel][channel] and ds_read_b64_tr_b16 hands out the pixel-contiguous fragments.
struct A8WParams {
  const char* dy; int dyps;
  const unsigned char* q; const unsigned char* s;
  long long npix, chunk;           // chunk: pixels per split
  int Cout, Cin, Cout_real, Cin_real, ntiles, ctiles, splits;
  float* slab;                     // [splits][Cout_real * Cin_real + Cout_real] when splits > 1
  float* dw; float* db; int accumulate;
};

// three bf16 parts of eight floats: f = h + m + l exactly from 2^-103 up (below, the third part is no normal bf16 number any
// more).  The parts are cut off, not rounded: eight bits each are the 24 of an fp32 number, and h never passes bf16's largest
// one.  An infinity or a NaN is its first part, the others are zero.
__device__ __forceinline__ void split3(const float* f, u32x4_t* o) {
  float h[8], m[8], l[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const bool finite = abs_bits(f[k]) < 0x7f800000u;
    h[k] = finite ? __uint_as_float(__float_as_uint(f[k]) & 0xffff0000u) : f[k];
    const float r = finite ? f[k] - h[k] : 0.f;
    m[k] = __uint_as_float(__float_as_uint(r) & 0xffff0000u);
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

// A workgroup of WN x WC waves takes a tile of 16 FN WN output x 16 FC WC input channels over a range of pixels, KP at a
// time.  Both operands pass through registers into one of two LDS stages, the input's codes becoming bf16 on the way, and
// are loaded a step ahead of that.  (LDS-DMA would spare dY the registers, but the compiler lets no transposed read pass a
// pending one; a second set of registers, to load two steps ahead, costs more in occupancy than it hides.)  Bound by the
// matrix unit and the staging beside it: 165 us at 2048 x 2048 channels and 16384 pixels with the launch that adds the
// splits' sums, back to back (830 TFLOP/s; in a kernel trace 188 + 15), where the products alone take 109 at the clock they
// leave the chip, their fragment reads and barriers 20 - 28 more, and the loads and staging the rest.  LDS is not what bounds it: images turned over in
// registers, [channel][pixel], and read 16 bytes at a time halve its reads and took 178.
//
// GK = 2: a second set of waves takes every other step, with stages of its own, and hands its sums over at the end -- the
// occupancy of two workgroups with the partial sums of one, which otherwise cost as much as the small layers' operands.
template <int DT, int FN, int FC, int WN, int WC, int KP, int GK>
__global__ __launch_bounds__(64 * WN * WC * GK, 2) void act8_wgrad_kernel(const A8WParams p) {
  constexpr int NW = WN * WC, NT = 64 * NW, BN = 16 * FN * WN, BC = 16 * FC * WC, CN = BN / 8, CC = BC / 8;
  constexpr int PL = DT == CSMRI_F32 ? 3 : 1, ES = DT == CSMRI_F32 ? 4 : 2;
  constexpr int YIMG = KP * BN * 2, XIMG = KP * BC * 2, STG = PL * YIMG + XIMG;
  constexpr int NY = KP * CN / NT, NX = KP * CC / NT;            // chunks of eight channels a thread and stage
  static_assert(KP * CN % NT == 0 && KP * CC % NT == 0, "whole chunks per thread");
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int tid = threadIdx.x % NT, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wid / WC, wc = wid % WC;
  const int part = __builtin_amdgcn_readfirstlane(threadIdx.x / NT);
  char* stages = smem + part * 2 * STG;
  const int tiles = p.ntiles * p.ctiles;
  // an XCD takes neighbouring tiles of the same pixels, which then meet in its L2
  const int wg = xcd_remap(blockIdx.x, tiles * p.splits), split = wg / tiles, tile = wg - split * tiles;
  const int nt = tile / p.ctiles, ct = tile - nt * p.ctiles;
  const int n0 = nt * BN, c0 = ct * BC;
  const long long pb = split * p.chunk, pe = pb + p.chunk < p.npix ? pb + p.chunk : p.npix;
  const int sblocks = (p.Cin + MICRO_BLOCK - 1) / MICRO_BLOCK;
  const int steps = pe > pb ? (int)((pe - pb + KP - 1) / KP) : 0, mine = (steps + GK - 1) / GK;   // step s of a part: GK s + part

  constexpr int NB = FN / WC;                                     // fragments whose column sums a wave takes
  static_assert(FN % WC == 0, "every wave of a row takes as many");
  f32x4_t acc[FN][FC], accb[NB];
#pragma unroll
  for (int i = 0; i < FN; ++i) {
#pragma unroll
    for (int j = 0; j < FC; ++j) acc[i][j] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int i = 0; i < NB; ++i) accb[i] = (f32x4_t){0.f, 0.f, 0.f, 0.f};

  // chunk j of a thread: row (j NT + tid) / chunks of a row.  Channels behind the end read the first ones (their results are
  // not stored), pixels behind the range its last one, with a dY of zero
  int yrow[NY], yoff[NY], xrow[NX], xoff[NX], ych[NY], xch[NX];
#pragma unroll
  for (int j = 0; j < NY; ++j) {
    const int id = j * NT + tid, ch = id % CN;
    yrow[j] = id / CN; yoff[j] = img_off<CN>(yrow[j], ch); ych[j] = (n0 + ch * 8 < p.Cout ? n0 + ch * 8 : 0) * ES;
  }
#pragma unroll
  for (int j = 0; j < NX; ++j) {
    const int id = j * NT + tid, ch = id % CC;
    xrow[j] = id / CC; xoff[j] = img_off<CC>(xrow[j], ch); xch[j] = c0 + ch * 8 < p.Cin ? c0 + ch * 8 : 0;
  }
  raw8<DT> yv[NY]; u32x2_t xv[NX]; unsigned sv[NX];
  auto left_of = [&](int k) { const long long l = pe - pb - (long long)k * KP; return l < KP ? (int)l : KP; };
  // (behind the last step: the last one again, with a dY of zero)
  auto fetch = [&](int s) {
    const int k = min(s * GK + part, steps - 1);
    const long long pix = pb + (long long)k * KP;
    const char* yb = p.dy + pix * p.dyps * ES;
    const unsigned char* xb = p.q + pix * p.Cin; const unsigned char* sb = p.s + pix * sblocks;
    const int last = left_of(k) - 1;
#pragma unroll
    for (int j = 0; j < NY; ++j) yv[j] = ldraw8<DT>(yb + (unsigned)(min(yrow[j], last) * p.dyps * ES + ych[j]), 0);
#pragma unroll
    for (int j = 0; j < NX; ++j) {
      const int r = min(xrow[j], last);
      xv[j] = *(const u32x2_t*)(xb + (unsigned)(r * p.Cin + xch[j]));
      sv[j] = sb[(unsigned)(r * sblocks + (xch[j] >> 5))];
    }
  };
  auto place = [&](int s) {
    char* yi = stages + (s & 1) * STG; char* xi = yi + PL * YIMG;
    const int left = left_of(s * GK + part);
    if (left < KP) {
#pragma unroll
      for (int j = 0; j < NY; ++j)
        if (yrow[j] >= left) yv[j] = raw8<DT>{};
    }
#pragma unroll
    for (int j = 0; j < NY; ++j) {
      if constexpr (DT == CSMRI_F32) {
        float f[8]; u32x4_t o[3];
        cvt8<DT>(yv[j], f);
        split3(f, o);
#pragma unroll
        for (int i = 0; i < 3; ++i) *(u32x4_t*)(yi + i * YIMG + yoff[j]) = o[i];
      } else {
        *(u32x4_t*)(yi + yoff[j]) = yv[j].a;
      }
    }
#pragma unroll
    for (int j = 0; j < NX; ++j) {
      const float s = __uint_as_float(sv[j] << 23);
      u32x4_t o;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        o[2 * q] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xv[j][q], s, false));
        o[2 * q + 1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(xv[j][q], s, true));
      }
      *(u32x4_t*)(xi + xoff[j]) = o;
    }
  };
  auto barrier = [&]() {                          // (not __syncthreads: that would wait for the loads under way too)
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };
  // fragments: a 16-lane group reads 4 pixel rows x 16 channels; rows 8 g + (0..3) and 8 g + (4..7) of the step
  const int g = lane >> 4, tr = (lane & 15) >> 2, tc = lane & 3, lo = 8 * g + tr, hi = lo + 4;
  const int yc = wn * FN * 2 + (tc >> 1), xc = wc * FC * 2 + (tc >> 1), in = (tc & 1) * 8;
  const bf16x8_t ones = {(__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f, (__bf16)1.f};
  const bool want_b = p.db && ct == 0;
  auto run = [&](auto with_bias) {
    auto multiply = [&](int s) {
      const char* yi = stages + (s & 1) * STG; const char* xi = yi + PL * YIMG;
#pragma unroll
      for (int kk = 0; kk < KP; kk += 32) {
        bf16x8_t xf[FC];
#pragma unroll
        for (int j = 0; j < FC; ++j) xf[j] = tr_frag(xi, img_off<CC>(kk + lo, xc + 2 * j) + in, img_off<CC>(kk + hi, xc + 2 * j) + in);
#pragma unroll
        for (int pl = 0; pl < PL; ++pl)
#pragma unroll
        for (int i = 0; i < FN; ++i) {
          const bf16x8_t yf = tr_frag(yi + pl * YIMG, img_off<CN>(kk + lo, yc + 2 * i) + in, img_off<CN>(kk + hi, yc + 2 * i) + in);
#pragma unroll
          for (int j = 0; j < FC; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(yf, xf[j], acc[i][j], 0, 0, 0);
        }
        if constexpr (decltype(with_bias)::value) {
#pragma unroll
          for (int pl = 0; pl < PL; ++pl)
#pragma unroll
          for (int i = 0; i < NB; ++i) {
            const int c = yc + 2 * (wc * NB + i);
            const bf16x8_t yf = tr_frag(yi + pl * YIMG, img_off<CN>(kk + lo, c) + in, img_off<CN>(kk + hi, c) + in);
            accb[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(yf, ones, accb[i], 0, 0, 0);
          }
        }
      }
    };
    if (steps == 0) return;
    fetch(0);
    place(0);
    fetch(1);
    for (int s = 0; s < mine; ++s) {
      barrier();                                  // stage s is there for everyone; everyone has read stage s - 1
      // half of the waves multiply first, so that staging and products run side by side
      if (wn & 1) { multiply(s); __builtin_amdgcn_sched_barrier(0); }
      place(s + 1);
      fetch(s + 2);
      __builtin_amdgcn_sched_barrier(0);
      if (!(wn & 1)) multiply(s);
    }
  };
  if (want_b) run(std::true_type{});
  else run(std::false_type{});
  if constexpr (GK == 2) {
    static_assert((FN * FC + NB) * NT * 16 <= 4 * STG, "the sums handed over share the stages' place");
    f32x4_t* sums = (f32x4_t*)smem + tid;
    barrier();
    if (part == 1) {
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FC; ++j) sums[(i * FC + j) * NT] = acc[i][j];
#pragma unroll
      for (int i = 0; i < NB; ++i) sums[(FN * FC + i) * NT] = accb[i];
    }
    barrier();
    if (part == 1) return;
#pragma unroll
    for (int i = 0; i < FN; ++i)
#pragma unroll
      for (int j = 0; j < FC; ++j) acc[i][j] += sums[(i * FC + j) * NT];
#pragma unroll
    for (int i = 0; i < NB; ++i) accb[i] += sums[(FN * FC + i) * NT];
  }
  // lane l holds rows n = 4 g + r, column c = l & 15 of each fragment
  const long long len = (long long)p.Cout_real * p.Cin_real;
  float* dw = p.splits > 1 ? p.slab + split * (len + p.Cout_real) : p.dw;
  float* db = p.splits > 1 ? dw + len : p.db;
  const bool add = p.splits == 1 && p.accumulate;
  const int cb = c0 + wc * FC * 16 + (lane & 15);
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = n0 + (wn * FN + i) * 16 + 4 * g + r;
      if (n >= p.Cout_real) continue;
      float* o = dw + (long long)n * p.Cin_real + cb;
      float old[FC];
#pragma unroll
      for (int j = 0; j < FC; ++j) old[j] = add && cb + 16 * j < p.Cin_real ? o[16 * j] : 0.f;
#pragma unroll
      for (int j = 0; j < FC; ++j)
        if (cb + 16 * j < p.Cin_real) o[16 * j] = acc[i][j][r] + old[j];
    }
  if (want_b && (lane & 15) == 0) {
#pragma unroll
    for (int i = 0; i < NB; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = n0 + (wn * FN + wc * NB + i) * 16 + 4 * g + r;
        if (n < p.Cout_real) db[n] = accb[i][r] + (add ? db[n] : 0.f);
      }
  }
}

// Tile: 64 or 128 a side by the channel counts; 256 x 256 (an fp32 dY's three planes do not fit it), which reads LDS a third
// less per product, where that leaves every CU 2304 pixels of a tile or more -- below, its larger partial sums cost as much
// -- and covers no more than a tenth beyond what the smaller tiles do.
// us with it and with 128 x 128, sums included, back to back: 16384 pixels, 2048 to 2048 164 / 176; 32768, 1024 to 2048
// 162 / 181; 16384, 1536 to 1536 109 / 170; 65536, 512 to 1024 100 / 99; 24576, 1024 to 1024 84 / 79; 8192, 2048 to 2048
// 102 / 94.
struct A8WTile { int bn, bc; };
static A8WTile a8w_tile(int dy_dtype, long long npix, int Cout, int Cin) {
  const double big = (double)cdiv(Cout, 256) * cdiv(Cin, 256), small = (double)cdiv(Cout, 128) * cdiv(Cin, 128);
  if (dy_dtype == CSMRI_BF16 && big * npix >= 2304. * 256 && 4 * big <= 1.1 * small) return {256, 256};
  return {Cout <= 64 ? 64 : 128, Cin <= 64 ? 64 : 128};
}
extern "C" int csmri_act8_wgrad_splits(int dy_dtype, long long npix, int Cout, int Cin) {
  if (npix <= 0 || Cout <= 0 || Cin <= 0) return 1;
  const A8WTile t = a8w_tile(dy_dtype, npix, Cout, Cin);
  const long long tiles = (long long)cdiv(Cout, t.bn) * cdiv(Cin, t.bc), len = (long long)(Cout + 1) * Cin * 4;
  const long long most = 256 / tiles < npix / 128 ? 256 / tiles : npix / 128;     // one workgroup of eight waves a CU
  // ns: 128 pixels of a tile; partial sums, written and read, a MiB; the launch that adds them.  Measured, in us, by the
  // number of splits: 4096 pixels, 64 to 128 channels, 1: 37, 8: 14.8, 16 - 32: 13.7; 4096, 512 to 512, 4: 26, 8: 24, 16: 26;
  // 4096, 1024 to 1024, 2: 40, 4: 34, 8: 48; 1024, 1024 to 1024, 1: 23, 2: 25.
  const long long step = (500 + t.bn * t.bc / 1024 * 42) * (dy_dtype == CSMRI_F32 ? 2 : 1);
  long long best = 1, least = step * ((npix + 127) / 128);
  for (long long c = 2; most > 1; c += c & (c - 1) ? c / 3 : c / 2) {      // 2, 3, 4, 6, 8, 12, ... and the most
    const long long s = c < most ? c : most;
    const long long cost = step * (((npix + s - 1) / s + 127) / 128) + 4000 + (600 * s * len >> 20);
    if (cost < least) { least = cost; best = s; }
    if (s == most) break;
  }
  return (int)best;
}
template <int DT, int FN, int FC, int WN, int WC, int KP, int GK> static int a8w_launch(const A8WParams& p, unsigned grid, hipStream_t st) {
  constexpr int BN = 16 * FN * WN, BC = 16 * FC * WC, LDS = GK * 2 * KP * 2 * (BN * (DT == CSMRI_F32 ? 3 : 1) + BC);
  auto kern = act8_wgrad_kernel<DT, FN, FC, WN, WC, KP, GK>;
  CSMRI_SET_MAX_LDS(kern, LDS);
  hipLaunchKernelGGL(kern, dim3(grid), dim3(64 * WN * WC * GK), LDS, st, p);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}
// pixels a step: 64, for fewer barriers, where two stages of that fit LDS twice
template <int DT> static int a8w_dispatch(const A8WTile& t, const A8WParams& p, unsigned grid, hipStream_t st) {
  constexpr int KP = DT == CSMRI_F32 ? 32 : 64;
  if constexpr (DT == CSMRI_BF16) if (t.bn == 256) return a8w_launch<DT, 8, 4, 2, 4, 32, 1>(p, grid, st);
  if (t.bn == 128) return t.bc == 128 ? a8w_launch<DT, 4, 4, 2, 2, KP, 2>(p, grid, st) : a8w_launch<DT, 4, 2, 2, 2, KP, 2>(p, grid, st);
  return t.bc == 128 ? a8w_launch<DT, 2, 4, 2, 2, KP, 2>(p, grid, st) : a8w_launch<DT, 2, 2, 2, 2, KP, 2>(p, grid, st);
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
  CSMRI_CHECK_ARG(!buffers_meet(dw, (long long)Cout_real * Cin_real, db, Cout_real));
  if (npix && (((uintptr_t)dy & 15) || ((uintptr_t)q8 & 7) || ((long long)dy_pix_stride * dtype_size(dy_dtype)) % 16)) return CSMRI_E_ALIGN;
  A8WParams p = {};
  p.dy = (const char*)dy; p.dyps = dy_pix_stride;
  p.q = (const unsigned char*)q8; p.s = (const unsigned char*)s8;
  p.npix = npix;
  p.Cout = Cout; p.Cin = Cin; p.Cout_real = Cout_real; p.Cin_real = Cin_real;
  const A8WTile t = a8w_tile(dy_dtype, npix, Cout, Cin);
  p.ntiles = cdiv(Cout, t.bn); p.ctiles = cdiv(Cin, t.bc);
  p.splits = splits; p.slab = slab; p.dw = dw; p.db = db; p.accumulate = accumulate;
  p.chunk = ((npix + splits - 1) / splits + 63) / 64 * 64;
  const long long grid = (long long)p.ntiles * p.ctiles * splits;
  // offsets inside a step, of 64 pixels (32 of an fp32 dY), are 32 bits
  if (grid > 0x7fffffff || (long long)dy_pix_stride * 4 * 32 > 0x7fffffff || (long long)Cin * 64 > 0x7fffffff) return CSMRI_E_UNSUPPORTED;
  const int rc = dy_dtype == CSMRI_F32 ? a8w_dispatch<CSMRI_F32>(t, p, (unsigned)grid, st)
                                       : a8w_dispatch<CSMRI_BF16>(t, p, (unsigned)grid, st);
  if (rc != CSMRI_OK || splits == 1) return rc;
  const long long len = (long long)Cout_real * Cin_real;
  return micro_colsum2(slab, splits, len + Cout_real, len, dw, db ? Cout_real : 0, db, accumulate, st);
}
