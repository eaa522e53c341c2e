// Layer norm over the channels of each pixel (+ LeakyReLU), forward and backward, NHWC rows.
//
//   m = mean_c x, r = 1 / sqrt(mean_c (x - m)^2 + eps), h = (x - m) r, y = gamma h + beta, z = y > 0 ? y : slope y
//   backward: dy = dz * (y > 0 ? 1 : slope), t = dy gamma,
//             dx = r (t - mean_c t - h mean_c (t h)), dgamma = sum_p dy h, dbeta = sum_p dy
//
// Both passes are bound by HBM: a row is read once into registers, its mean and then its variance around that mean are
// taken from there (no cancellation, whatever the offset of the data), and written once.  A row of up to 64 lanes x
// V vectors of eight channels belongs to one wave -- rows of few channels share a wave -- and a wider one to a
// workgroup.  The backward recomputes m and r from x with the forward's own arithmetic, so nothing but x is kept; where x
// itself was kept in 8 bits (micro.h) the forward's m and r are stored next to it and the backward takes 1.03 bytes a
// channel instead of 2 or 4.  dgamma and dbeta gather in registers over the rows a workgroup walks and leave as one
// partial row per workgroup, summed in fixed order by a second launch: no atomics, the same bits on every run.
#include "micro.h"

struct LNParams {
  const void* x; int xps;
  const unsigned char* q; const unsigned char* s;      // kept input, instead of x (backward) / written beside z (forward)
  unsigned char* qo; unsigned char* so;
  const void* gz; int gps;                             // backward: gradient of z
  const void* z; int zps;                              // backward: output of the forward, for its sign (may be NULL)
  void* out; int ops;                                  // z (forward), dx (backward, may be NULL)
  long long rows;
  int C, C_real, group;                                // lanes per row (a power of two; rows wider than a wave: 256)
  const float* gamma; const float* beta; float* snap;  // forward: parameters and their snapshot
  const float* stats_in; float* stats_out;             // [2][rows] mean, 1 / std
  float eps, slope;
  float* partial;                                      // backward: [gridDim.x][2][C_real], NULL when neither is wanted
};

// sum over the lanes of a row
template <bool WG> __device__ __forceinline__ float row_sum(float a, int group, float* red) {
  if constexpr (WG) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a += __shfl_xor(a, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
  } else {
    for (int o = group >> 1; o > 0; o >>= 1) a += __shfl_xor(a, o);
    return a;
  }
}

// mean and 1 / std of U rows held as V vectors a lane; nv[j]: real channels of vector j
template <bool WG, int V, int U>
__device__ __forceinline__ void row_stats(const float (&x)[U][V][8], const int (&nv)[V], const LNParams& p, float* red,
                                          float (&mean)[U], float (&inv)[U]) {
  const float rc = 1.f / (float)p.C_real;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) a += k < nv[j] ? x[u][j][k] : 0.f;
    mean[u] = a;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) mean[u] = row_sum<WG>(mean[u], p.group, red) * rc;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) { const float d = x[u][j][k] - mean[u]; a += k < nv[j] ? d * d : 0.f; }
    inv[u] = a;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) inv[u] = rsqrtf(row_sum<WG>(inv[u], p.group, red) * rc + p.eps);
}

// the affine step, spelled out so that the forward and the backward's sign test round alike
__device__ __forceinline__ float ln_affine(float h, float g, float b) { return __builtin_fmaf(h, g, b); }

template <int V> __device__ __forceinline__ void ld_affine(const float* p, const int (&c)[V], const int (&nv)[V], float (&o)[V][8]) {
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) o[j][k] = k < nv[j] ? p[c[j] + k] : 0.f;
}

template <int DT, bool WG, int V, int U, bool KEEP>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const LNParams p) {
  __shared__ float red[4];
  const int gl = WG ? threadIdx.x : (threadIdx.x & (p.group - 1));
  const int gpw = WG ? 1 : 256 / p.group, gi = WG ? 0 : threadIdx.x / p.group;
  int c[V], nv[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    c[j] = (j * p.group + gl) * 8;
    const int n = p.C_real - c[j];
    nv[j] = n < 0 ? 0 : (n > 8 ? 8 : n);
  }
  float ga[V][8], be[V][8];
  ld_affine<V>(p.gamma, c, nv, ga);
  ld_affine<V>(p.beta, c, nv, be);
  if (p.snap && blockIdx.x == 0 && gi == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (c[j] < p.C) { st8<CSMRI_F32>(p.snap, c[j], ga[j]); st8<CSMRI_F32>(p.snap, p.C + c[j], be[j]); }
  }
  const int sblocks = (p.C + MICRO_BLOCK - 1) / MICRO_BLOCK;
  const long long step = (long long)gridDim.x * gpw;
  for (long long row = (long long)blockIdx.x * gpw + gi; row - gi < p.rows; row += step * U) {
    raw8<DT> raw[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        raw[u][j] = raw8<DT>{};
        if (c[j] < p.C && row + u * step < p.rows) raw[u][j] = ldraw8<DT>(p.x, (row + u * step) * p.xps + c[j]);
      }
    __builtin_amdgcn_sched_barrier(0);
    float x[U][V][8], mean[U], inv[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) cvt8<DT>(raw[u][j], x[u][j]);
    row_stats<WG, V, U>(x, nv, p, red, mean, inv);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step;
      const bool live = rr < p.rows;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if constexpr (KEEP) {                        // all lanes take part in the block's maximum
          const unsigned amax = block_amax(x[u][j]);
          unsigned char sc;
          const u32x2_t o = micro_pack8(x[u][j], amax, sc);
          if (live && c[j] < p.C) {
            *(u32x2_t*)(p.qo + rr * p.C + c[j]) = o;
            if ((c[j] & (MICRO_BLOCK - 1)) == 0) p.so[rr * sblocks + c[j] / MICRO_BLOCK] = sc;
          }
        }
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float y = ln_affine((x[u][j][k] - mean[u]) * inv[u], ga[j][k], be[j][k]);
          const float z = y > 0.f ? y : y * p.slope;
          o[k] = k < nv[j] ? z : 0.f;
        }
        if (live && c[j] < p.C) st8<DT>(p.out, rr * p.ops + c[j], o);
      }
      if (live && gl == 0 && p.stats_out) { p.stats_out[rr] = mean[u]; p.stats_out[p.rows + rr] = inv[u]; }
    }
  }
}

// KEPT: the input comes as e4m3 codes, with the forward's mean and 1 / std
template <int DT, bool WG, int V, int U, bool KEPT>
__global__ __launch_bounds__(256) void ln_bwd_kernel(const LNParams p) {
  extern __shared__ __attribute__((aligned(16))) float lds[];      // [4] for row_sum, then the affine partials
  float* red = lds;
  const int gl = WG ? threadIdx.x : (threadIdx.x & (p.group - 1));
  const int gpw = WG ? 1 : 256 / p.group, gi = WG ? 0 : threadIdx.x / p.group;
  int c[V], nv[V];
#pragma unroll
  for (int j = 0; j < V; ++j) {
    c[j] = (j * p.group + gl) * 8;
    const int n = p.C_real - c[j];
    nv[j] = n < 0 ? 0 : (n > 8 ? 8 : n);
  }
  float ga[V][8], dg[V][8], db[V][8];
  ld_affine<V>(p.gamma, c, nv, ga);
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) dg[j][k] = db[j][k] = 0.f;
  const int sblocks = (p.C + MICRO_BLOCK - 1) / MICRO_BLOCK;
  const float rc = 1.f / (float)p.C_real;
  const bool gate_z = p.slope != 1.f && p.z, gate_x = p.slope != 1.f && !p.z;
  const long long step = (long long)gridDim.x * gpw;
  for (long long row = (long long)blockIdx.x * gpw + gi; row - gi < p.rows; row += step * U) {
    raw8<DT> rx[U][V], rg[U][V], rz[U][V];
    u32x2_t rq[U][V]; unsigned char rs[U][V];
    float mean[U], inv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step;
      const bool live = rr < p.rows;
      if constexpr (KEPT) { mean[u] = live ? p.stats_in[rr] : 0.f; inv[u] = live ? p.stats_in[p.rows + rr] : 0.f; }
#pragma unroll
      for (int j = 0; j < V; ++j) {
        rg[u][j] = raw8<DT>{};
        if constexpr (KEPT) { rq[u][j] = (u32x2_t){0, 0}; rs[u][j] = 0; } else rx[u][j] = raw8<DT>{};
        if (c[j] < p.C && live) {
          rg[u][j] = ldraw8<DT>(p.gz, rr * p.gps + c[j]);
          if constexpr (KEPT) {
            rq[u][j] = *(const u32x2_t*)(p.q + rr * p.C + c[j]);
            rs[u][j] = p.s[rr * sblocks + c[j] / MICRO_BLOCK];
          } else {
            rx[u][j] = ldraw8<DT>(p.x, rr * p.xps + c[j]);
          }
        }
      }
    }
    if (gate_z) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          rz[u][j] = raw8<DT>{};
          if (c[j] < p.C && row + u * step < p.rows) rz[u][j] = ldraw8<DT>(p.z, (row + u * step) * p.zps + c[j]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    float x[U][V][8];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if constexpr (KEPT) micro_unpack8(rq[u][j], micro_scale(rs[u][j]), x[u][j]);
        else cvt8<DT>(rx[u][j], x[u][j]);
      }
    if constexpr (!KEPT) row_stats<WG, V, U>(x, nv, p, red, mean, inv);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step;
      const bool live = rr < p.rows;
      float t[V][8];
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float g[8];
        cvt8<DT>(rg[u][j], g);
        if (gate_z) {
          float z[8];
          cvt8<DT>(rz[u][j], z);
#pragma unroll
          for (int k = 0; k < 8; ++k) g[k] *= z[k] > 0.f ? 1.f : p.slope;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float h = (x[u][j][k] - mean[u]) * inv[u];
          if (gate_x) g[k] *= ln_affine(h, ga[j][k], k < nv[j] ? p.beta[c[j] + k] : 0.f) > 0.f ? 1.f : p.slope;
          const bool ok = k < nv[j] && live;
          const float hk = ok ? h : 0.f, gk = ok ? g[k] : 0.f;
          x[u][j][k] = hk;
          dg[j][k] += gk * hk;
          db[j][k] += gk;
          t[j][k] = gk * ga[j][k];
          s1 += t[j][k];
          s2 += t[j][k] * hk;
        }
      }
      s1 = row_sum<WG>(s1, p.group, red) * rc;
      s2 = row_sum<WG>(s2, p.group, red) * rc;
      if (p.out && live) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (c[j] >= p.C) continue;
          float o[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = k < nv[j] ? inv[u] * (t[j][k] - s1 - x[u][j][k] * s2) : 0.f;
          st8<DT>(p.out, rr * p.ops + c[j], o);
        }
      }
    }
  }
  if (!p.partial) return;
  float* prow = p.partial + (long long)blockIdx.x * 2 * p.C_real;      // dense: both sums are one launch
  if constexpr (WG) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < nv[j]) { prow[c[j] + k] = dg[j][k]; prow[p.C_real + c[j] + k] = db[j][k]; }
  } else {
    // groups of a wave first, then the four waves in order
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        for (int o = p.group; o < 64; o <<= 1) { dg[j][k] += __shfl_xor(dg[j][k], o); db[j][k] += __shfl_xor(db[j][k], o); }
    float* part = lds + 4;
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63, span = p.group * V * 8;
    for (int w = 0; w < 4; ++w) {
      if (wid == w && lane < p.group) {
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            part[c[j] + k] = (w ? part[c[j] + k] : 0.f) + dg[j][k];
            part[span + c[j] + k] = (w ? part[span + c[j] + k] : 0.f) + db[j][k];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * p.C_real; i += 256) prow[i] = part[i < p.C_real ? i : span + i - p.C_real];
  }
}

#define LN_MAX_C 8192
struct LNShape { bool wg; int group, v; };
// lanes and vectors of a row of C channels: one vector a lane up to a wave's width, then two and four, then a workgroup
static LNShape ln_shape(int C) {
  const int c8 = C / 8;
  LNShape s = {false, 4, 1};                 // four lanes at least: a block of the 8-bit form is four lanes wide
  while (s.group < c8 && s.group < 64) s.group *= 2;
  while (s.group * s.v < c8 && s.v < 4) s.v *= 2;
  if (s.group * s.v < c8) {
    s.wg = true; s.group = 256; s.v = c8 <= 512 ? 2 : 4;
  }
  return s;
}
static bool ln_args_ok(int dtype, long long npix, int C, int C_real) {
  return (dtype == CSMRI_F32 || dtype == CSMRI_BF16) && npix >= 0 && C > 0 && C % 8 == 0 && C_real > 0 && C_real <= C;
}
static bool ln_aligned(const void* p, int ps, int dtype) {
  return ((uintptr_t)p & 15) == 0 && ((long long)ps * dtype_size(dtype)) % 16 == 0;
}
static long long ln_blocks(long long npix, const LNShape& s, int unroll) {
  const long long per = (s.wg ? 1 : 256 / s.group) * unroll;
  return (npix + per - 1) / per;
}

template <int DT, bool KEEP> static int ln_fwd_launch(const LNParams& p, const LNShape& s, hipStream_t st) {
  // rows in flight per lane: four of one vector, two of two, else one
  const int U = s.wg ? 1 : (s.v == 1 ? 4 : (s.v == 2 ? 2 : 1));
  long long blocks = ln_blocks(p.rows, s, U);
  if (blocks > 2048) blocks = 2048;
  const dim3 g((unsigned)blocks), b(256);
  if (s.wg) {
    if (s.v == 2) hipLaunchKernelGGL((ln_fwd_kernel<DT, true, 2, 1, KEEP>), g, b, 0, st, p);
    else hipLaunchKernelGGL((ln_fwd_kernel<DT, true, 4, 1, KEEP>), g, b, 0, st, p);
  } else if (s.v == 1) hipLaunchKernelGGL((ln_fwd_kernel<DT, false, 1, 4, KEEP>), g, b, 0, st, p);
  else if (s.v == 2) hipLaunchKernelGGL((ln_fwd_kernel<DT, false, 2, 2, KEEP>), g, b, 0, st, p);
  else hipLaunchKernelGGL((ln_fwd_kernel<DT, false, 4, 1, KEEP>), g, b, 0, st, p);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}

extern "C" int csmri_ln_fwd(int dtype, const void* x, int x_pix_stride, void* z, int z_pix_stride, long long npix, int C,
                            int C_real, const float* gamma, const float* beta, float eps, float slope,
                            float* affine_snap, float* stats, void* q8, uint8_t* s8, void* stream) {
  CSMRI_CHECK_ARG(ln_args_ok(dtype, npix, C, C_real) && x_pix_stride >= C && z_pix_stride >= C && gamma && beta);
  CSMRI_CHECK_ARG((q8 == NULL) == (s8 == NULL) && (!q8 || stats));
  if (C > LN_MAX_C) return CSMRI_E_UNSUPPORTED;
  CSMRI_CHECK_ARG(npix == 0 || (x && z && x != z));
  if (!ln_aligned(x, x_pix_stride, dtype) || !ln_aligned(z, z_pix_stride, dtype) || ((uintptr_t)affine_snap & 15) ||
      ((uintptr_t)q8 & 7)) return CSMRI_E_ALIGN;
  LNParams p = {};
  p.x = x; p.xps = x_pix_stride; p.out = z; p.ops = z_pix_stride;
  p.rows = npix; p.C = C; p.C_real = C_real;
  p.gamma = gamma; p.beta = beta; p.snap = affine_snap; p.stats_out = stats;
  p.eps = eps; p.slope = slope;
  p.qo = (unsigned char*)q8; p.so = (unsigned char*)s8;
  const LNShape s = ln_shape(C);
  p.group = s.group;
  if (npix == 0) return CSMRI_OK;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == CSMRI_F32) return q8 ? ln_fwd_launch<CSMRI_F32, true>(p, s, st) : ln_fwd_launch<CSMRI_F32, false>(p, s, st);
  return q8 ? ln_fwd_launch<CSMRI_BF16, true>(p, s, st) : ln_fwd_launch<CSMRI_BF16, false>(p, s, st);
}

static int ln_bwd_unroll(const LNShape& s) { return !s.wg && s.v == 1 ? 2 : 1; }
extern "C" int csmri_ln_bwd_rows(long long npix, int C) {
  if (npix <= 0 || C <= 0) return 0;
  const LNShape s = ln_shape(C);
  const long long b = ln_blocks(npix, s, ln_bwd_unroll(s));
  return (int)(b > 1024 ? 1024 : b);
}

template <int DT, bool KEPT> static int ln_bwd_launch(const LNParams& p, const LNShape& s, int blocks, hipStream_t st) {
  const dim3 g(blocks), b(256);
  const size_t lds = (4 + (s.wg ? 0 : 2 * (size_t)s.group * s.v * 8)) * sizeof(float);
  if (s.wg) {
    if (s.v == 2) hipLaunchKernelGGL((ln_bwd_kernel<DT, true, 2, 1, KEPT>), g, b, lds, st, p);
    else hipLaunchKernelGGL((ln_bwd_kernel<DT, true, 4, 1, KEPT>), g, b, lds, st, p);
  } else if (s.v == 1) hipLaunchKernelGGL((ln_bwd_kernel<DT, false, 1, 2, KEPT>), g, b, lds, st, p);
  else if (s.v == 2) hipLaunchKernelGGL((ln_bwd_kernel<DT, false, 2, 1, KEPT>), g, b, lds, st, p);
  else hipLaunchKernelGGL((ln_bwd_kernel<DT, false, 4, 1, KEPT>), g, b, lds, st, p);
  CSMRI_LAUNCH_CHECK();
  return CSMRI_OK;
}

extern "C" int csmri_ln_bwd(int dtype, const void* dz, int dz_pix_stride, const void* x, int x_pix_stride, const void* q8,
                            const uint8_t* s8, const float* stats, const void* z, int z_pix_stride, void* dx,
                            int dx_pix_stride, long long npix, int C, int C_real, const float* affine_snap, float eps,
                            float slope, float* partial, float* dgamma, float* dbeta, int accumulate, void* stream) {
  CSMRI_CHECK_ARG(ln_args_ok(dtype, npix, C, C_real) && dz_pix_stride >= C && (!dx || dx_pix_stride >= C) && affine_snap);
  CSMRI_CHECK_ARG((dgamma == NULL) == (dbeta == NULL) && (!z || z_pix_stride >= C));
  if (C > LN_MAX_C) return CSMRI_E_UNSUPPORTED;
  hipStream_t st = (hipStream_t)stream;
  if (npix == 0) {
    int rc = CSMRI_OK;
    if (dgamma && !accumulate) rc = csmri_fill_f32(dgamma, C_real, 0.f, stream);
    if (rc == CSMRI_OK && dbeta && !accumulate) rc = csmri_fill_f32(dbeta, C_real, 0.f, stream);
    return rc;
  }
  CSMRI_CHECK_ARG(dz && (x != NULL) != (q8 != NULL) && (!q8 || (s8 && stats)) && (!x || x_pix_stride >= C));
  CSMRI_CHECK_ARG(slope == 1.f || x || z);                  // the sign of y is not to be had from rounded inputs
  CSMRI_CHECK_ARG(!dgamma || partial);
  CSMRI_CHECK_ARG(!dx || (dx != dz && dx != x && dx != z));
  if (!ln_aligned(dz, dz_pix_stride, dtype) || (x && !ln_aligned(x, x_pix_stride, dtype)) ||
      (z && !ln_aligned(z, z_pix_stride, dtype)) || (dx && !ln_aligned(dx, dx_pix_stride, dtype)) ||
      ((uintptr_t)q8 & 7) || ((uintptr_t)affine_snap & 15)) return CSMRI_E_ALIGN;
  LNParams p = {};
  p.x = x; p.xps = x_pix_stride;
  p.q = (const unsigned char*)q8; p.s = s8; p.stats_in = stats;
  p.gz = dz; p.gps = dz_pix_stride; p.z = z; p.zps = z_pix_stride;
  p.out = dx; p.ops = dx_pix_stride;
  p.rows = npix; p.C = C; p.C_real = C_real;
  p.gamma = affine_snap; p.beta = affine_snap + C;
  p.eps = eps; p.slope = slope;
  p.partial = dgamma ? partial : NULL;
  const LNShape s = ln_shape(C);
  p.group = s.group;
  const int blocks = csmri_ln_bwd_rows(npix, C);
  int rc;
  if (dtype == CSMRI_F32) rc = q8 ? ln_bwd_launch<CSMRI_F32, true>(p, s, blocks, st) : ln_bwd_launch<CSMRI_F32, false>(p, s, blocks, st);
  else rc = q8 ? ln_bwd_launch<CSMRI_BF16, true>(p, s, blocks, st) : ln_bwd_launch<CSMRI_BF16, false>(p, s, blocks, st);
  if (rc != CSMRI_OK || !dgamma) return rc;
  return micro_colsum2(partial, blocks, 2LL * C_real, C_real, dgamma, C_real, dbeta, accumulate, st);
}
