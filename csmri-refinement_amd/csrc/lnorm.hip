// Layer norm over the channels of each pixel (+ LeakyReLU), forward and backward, NHWC rows.
//
//   m = mean_c x, r = 1 / sqrt(mean_c (x - m)^2 + eps), h = (x - m) r, y = gamma h + beta, z = y > 0 ? y : slope y
//   backward: dy = dz * (y > 0 ? 1 : slope), t = dy gamma,
//             dx = r (t - mean_c t - h mean_c (t h)), dgamma = sum_p dy h, dbeta = sum_p dy
//
// Both passes are bound by HBM: a row is read once into registers, its mean, the deviations' own mean and the variance are
// taken from there (row_stats: what they cost is relative to the deviations, whatever the offset of the data), and written once.  A row of up to 64 lanes x
// V vectors of eight channels belongs to one wave -- rows of few channels share a wave -- and a wider one to a
// workgroup.  The backward recomputes m and r from x with the forward's own arithmetic, so nothing but x is kept; where x
// itself was kept in 8 bits (micro.h) the forward's m and r are stored next to it and the backward takes 1.03 bytes a
// channel instead of 2 or 4.  dgamma and dbeta gather in registers over the rows a workgroup walks and leave as one
// partial row per workgroup, summed in fixed order by a second launch: no atomics, the same bits on every run.
// 8 x 256 x 256 x 32 bf16: 15 and 24 us, 4.6 and 4.1 TB/s, + 4 us for the sums; 8 x 64 x 64 x 1024 with the input kept in
// 8 bits: 41 and 37 us, 4.2 and 4.5 TB/s, + 5 us; 64 fp32 pixels of 100 channels: 3.9 us.  Behind a LeakyReLU the backward
// also needs the sign of y: from x 8 x 256 x 256 x 32 takes 28 us, 8 x 64 x 64 x 1024 78 (41 without: beta is read again for
// every row); from z, of an input kept in 8 bits, 44 (38 without) for 40 % more bytes.
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
  float* dgamma; float* dbeta; int accumulate;         // written at once by a single workgroup, unused otherwise
};

// Sums over the lanes of a row.  A workgroup's four waves meet in one of two places of `red`, taken in turn, so that one
// barrier a sum is enough.
template <bool WG, int N> __device__ __forceinline__ void row_sums(float (&v)[N], int group, float (*red)[4 * 4], int& turn) {
  group_sums(v, WG ? 64 : group);
  if constexpr (WG) {
    static_assert(N <= 4, "places in red");
    float* r = red[turn];
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) r[(threadIdx.x >> 6) * 4 + i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (r[i] + r[4 + i]) + (r[8 + i] + r[12 + i]);
  }
}

// Statistics of U rows held as V vectors a lane; nv[j]: real channels of vector j.  The rounded mean m0 misses the mean by up
// to a few steps of an fp32 number of its size, which a row of nearly equal channels would see as a spread of its own.  So x
// becomes the deviations x - m0 (exact for channels within a factor of two of m0), `corr` their own mean, and
//   mean = m0 + corr,  h = (x - m0 - corr) inv,  variance = mean (x - m0)^2 - corr^2:
// errors are relative to the deviations, not to what the row lies around.  (A negative variance, all rounding, counts as 0.)
// It costs 1 us of a forward and backward of 41 at 8 x 256 x 256 x 32 bf16, with divisions for the products with rc 3.5.
template <bool WG, int V, int U>
__device__ __forceinline__ void row_stats(float (&x)[U][V][8], const int (&nv)[V], const LNParams& p, float (*red)[16],
                                          int& turn, float (&m0)[U], float (&corr)[U], float (&inv)[U]) {
  const float rc = 1.f / (float)p.C_real;       // (rounded too: what it costs m0 is in corr)
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float a = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) a += k < nv[j] ? x[u][j][k] : 0.f;
    m0[u] = a;
  }
  row_sums<WG, U>(m0, p.group, red, turn);
  float s[2 * U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    m0[u] *= rc;
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float d = k < nv[j] ? x[u][j][k] - m0[u] : 0.f;
        x[u][j][k] = d;
        a += d;
        b = __builtin_fmaf(d, d, b);
      }
    s[2 * u] = a; s[2 * u + 1] = b;
  }
  row_sums<WG, 2 * U>(s, p.group, red, turn);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    corr[u] = s[2 * u] * rc;
    const float v = __builtin_fmaf(-corr[u], corr[u], s[2 * u + 1] * rc);
    inv[u] = rsqrtf((v < 0.f ? 0.f : v) + p.eps);
  }
}

// the affine step, spelled out so that the forward and the backward's sign test round alike
__device__ __forceinline__ float ln_affine(float h, float g, float b) { return __builtin_fmaf(h, g, b); }

template <int V> __device__ __forceinline__ void ld_affine(const float* p, const int (&c)[V], const int (&nv)[V], float (&o)[V][8]) {
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) o[j][k] = k < nv[j] ? p[c[j] + k] : 0.f;
}
template <int V> __device__ __forceinline__ void ln_channels(const LNParams& p, int gl, int (&c)[V], int (&nv)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) {
    c[j] = (j * p.group + gl) * 8;
    const int n = p.C_real - c[j];
    nv[j] = n < 0 ? 0 : (n > 8 ? 8 : n);
  }
}

template <int DT, bool WG, int V, int U, bool KEEP>
__global__ __launch_bounds__(256) void ln_fwd_kernel(const LNParams p) {
  __shared__ float red[2][16];
  int turn = 0;
  const int gl = WG ? threadIdx.x : (threadIdx.x & (p.group - 1));
  const int gpw = WG ? 1 : 256 / p.group, gi = WG ? 0 : threadIdx.x / p.group;
  int c[V], nv[V];
  ln_channels<V>(p, gl, c, nv);
  const long long step = (long long)gridDim.x * gpw, first = (long long)blockIdx.x * gpw + gi;
  raw8<DT> raw[U][V];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        raw[u][j] = raw8<DT>{};
        if (c[j] < p.C && row + u * step < p.rows) raw[u][j] = ldraw8<DT>(p.x, (row + u * step) * p.xps + c[j]);
      }
  };
  fetch(first);
  float ga[V][8], be[V][8];
  ld_affine<V>(p.gamma, c, nv, ga);
  ld_affine<V>(p.beta, c, nv, be);
  if (p.snap && blockIdx.x == 0 && gi == 0) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (c[j] < p.C) { st8<CSMRI_F32>(p.snap, c[j], ga[j]); st8<CSMRI_F32>(p.snap, p.C + c[j], be[j]); }
  }
  const int sblocks = (p.C + MICRO_BLOCK - 1) / MICRO_BLOCK;
  const bool act = p.slope != 1.f;
  for (long long row = first; row - gi < p.rows; row += step * U) {
    float x[U][V][8], m0[U], corr[U], inv[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) cvt8<DT>(raw[u][j], x[u][j]);
    fetch(row + step * U);                           // the next rows come in under this one's arithmetic
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (KEEP) {                            // x itself, before it turns into deviations
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const long long rr = row + u * step;
#pragma unroll
        for (int j = 0; j < V; ++j) {                // all lanes take part in the block's maximum
          const unsigned amax = block_amax(x[u][j]);
          unsigned char sc;
          const u32x2_t o = micro_pack8(x[u][j], amax, sc);
          if (rr < p.rows && c[j] < p.C) {
            *(u32x2_t*)(p.qo + rr * p.C + c[j]) = o;
            if ((c[j] & (MICRO_BLOCK - 1)) == 0) p.so[rr * sblocks + c[j] / MICRO_BLOCK] = sc;
          }
        }
      }
    }
    row_stats<WG, V, U>(x, nv, p, red, turn, m0, corr, inv);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step;
      const bool live = rr < p.rows;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = ln_affine((x[u][j][k] - corr[u]) * inv[u], ga[j][k], be[j][k]);
        if (act) {
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = o[k] > 0.f ? o[k] : o[k] * p.slope;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = k < nv[j] ? o[k] : 0.f;
        if (live && c[j] < p.C) st8<DT>(p.out, rr * p.ops + c[j], o);
      }
      if (live && gl == 0 && p.stats_out) { p.stats_out[rr] = m0[u] + corr[u]; p.stats_out[p.rows + rr] = inv[u]; }
    }
  }
}

// KEPT: the input comes as e4m3 codes, with the forward's mean and 1 / std
template <int DT, bool WG, int V, int U, bool KEPT>
__global__ __launch_bounds__(256) void ln_bwd_kernel(const LNParams p) {
  extern __shared__ __attribute__((aligned(16))) float lds[];      // the affine partials of a workgroup
  __shared__ float red[2][16];
  int turn = 0;
  const int gl = WG ? threadIdx.x : (threadIdx.x & (p.group - 1));
  const int gpw = WG ? 1 : 256 / p.group, gi = WG ? 0 : threadIdx.x / p.group;
  int c[V], nv[V];
  ln_channels<V>(p, gl, c, nv);
  const int sblocks = (p.C + MICRO_BLOCK - 1) / MICRO_BLOCK;
  const float rc = 1.f / (float)p.C_real;
  const bool gate_z = p.slope != 1.f && p.z, gate_x = p.slope != 1.f && !p.z;
  const long long step = (long long)gridDim.x * gpw, first = (long long)blockIdx.x * gpw + gi;
  raw8<DT> rx[U][V], rg[U][V];
  u32x2_t rq[U][V]; unsigned char rs[U][V];
  float rm[U], ri[U];
  auto fetch = [&](long long row) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step;
      const bool live = rr < p.rows;
      if constexpr (KEPT) { rm[u] = live ? p.stats_in[rr] : 0.f; ri[u] = live ? p.stats_in[p.rows + rr] : 0.f; }
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
  };
  fetch(first);
  float ga[V][8], dg[V][8], db[V][8];
  ld_affine<V>(p.gamma, c, nv, ga);
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int k = 0; k < 8; ++k) dg[j][k] = db[j][k] = 0.f;
  for (long long row = first; row - gi < p.rows; row += step * U) {
    float x[U][V][8], t[U][V][8], sub[U], inv[U];     // h = (x - sub) inv
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if constexpr (KEPT) micro_unpack8(rq[u][j], micro_scale(rs[u][j]), x[u][j]);
        else cvt8<DT>(rx[u][j], x[u][j]);
        cvt8<DT>(rg[u][j], t[u][j]);
        if constexpr (KEPT) { sub[u] = rm[u]; inv[u] = ri[u]; }
      }
    if (gate_z) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          raw8<DT> rz = raw8<DT>{};
          if (c[j] < p.C && row + u * step < p.rows) rz = ldraw8<DT>(p.z, (row + u * step) * p.zps + c[j]);
          float z[8];
          cvt8<DT>(rz, z);
#pragma unroll
          for (int k = 0; k < 8; ++k) t[u][j][k] *= z[k] > 0.f ? 1.f : p.slope;
        }
    }
    fetch(row + step * U);                           // the next rows come in under this one's arithmetic
    __builtin_amdgcn_sched_barrier(0);
    float m0[U];
    if constexpr (!KEPT) row_stats<WG, V, U>(x, nv, p, red, turn, m0, sub, inv);
    float s[2 * U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool live = row + u * step < p.rows;
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) {
#pragma unroll
        for (int k = 0; k < 8; ++k) x[u][j][k] = (x[u][j][k] - sub[u]) * inv[u];
        if (gate_x) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            t[u][j][k] *= ln_affine(x[u][j][k], ga[j][k], k < nv[j] ? p.beta[c[j] + k] : 0.f) > 0.f ? 1.f : p.slope;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const bool ok = k < nv[j] && live;
          const float h = ok ? x[u][j][k] : 0.f, g = ok ? t[u][j][k] : 0.f;
          x[u][j][k] = h;
          dg[j][k] = __builtin_fmaf(g, h, dg[j][k]);
          db[j][k] += g;
          t[u][j][k] = g * ga[j][k];
          s1 += t[u][j][k];
          s2 = __builtin_fmaf(t[u][j][k], h, s2);
        }
      }
      s[2 * u] = s1; s[2 * u + 1] = s2;
    }
    row_sums<WG, 2 * U>(s, p.group, red, turn);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long rr = row + u * step;
      if (!p.out || rr >= p.rows) continue;
      const float s1 = s[2 * u] * rc, s2 = s[2 * u + 1] * rc;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        if (c[j] >= p.C) continue;
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = k < nv[j] ? inv[u] * (t[u][j][k] - s1 - x[u][j][k] * s2) : 0.f;
        st8<DT>(p.out, rr * p.ops + c[j], o);
      }
    }
  }
  if (!p.partial) return;
  const bool one = gridDim.x == 1;
  auto put = [&](float* o, float v) { *o = (p.accumulate ? *o : 0.f) + v; };
  float* prow = p.partial + (long long)blockIdx.x * 2 * p.C_real;      // dense: both sums are one launch
  if constexpr (WG) {
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (k < nv[j]) {
          if (one) { put(p.dgamma + c[j] + k, dg[j][k]); put(p.dbeta + c[j] + k, db[j][k]); }
          else { prow[c[j] + k] = dg[j][k]; prow[p.C_real + c[j] + k] = db[j][k]; }
        }
  } else {
    // groups of a wave first, then the four waves in order
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
      for (int k = 0; k < 8; ++k)
        for (int o = p.group; o < 64; o <<= 1) { dg[j][k] += __shfl_xor(dg[j][k], o); db[j][k] += __shfl_xor(db[j][k], o); }
    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63, span = p.group * V * 8;
    for (int w = 0; w < 4; ++w) {
      if (wid == w && lane < p.group) {
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            lds[c[j] + k] = (w ? lds[c[j] + k] : 0.f) + dg[j][k];
            lds[span + c[j] + k] = (w ? lds[span + c[j] + k] : 0.f) + db[j][k];
          }
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * p.C_real; i += 256) {
      const float v = lds[i < p.C_real ? i : span + i - p.C_real];
      if (one) put(i < p.C_real ? p.dgamma + i : p.dbeta + i - p.C_real, v);
      else prow[i] = v;
    }
  }
}

#define LN_MAX_C 8192
struct LNShape { bool wg; int group, v; };
// Lanes and vectors of a row of C channels: up to a wave of one vector a lane, then two; from there on a workgroup, of one,
// two and four (four vectors a lane of a wave would keep the backward to one wave a SIMD).
static LNShape ln_shape(int C) {
  const int c8 = C / 8;
  LNShape s = {false, 4, 1};                 // four lanes at least: a block of the 8-bit form is four lanes wide
  while (s.group < c8 && s.group < 64) s.group *= 2;
  if (c8 > 64) s.v = 2;
  if (c8 > 128) { s.wg = true; s.group = 256; s.v = c8 <= 256 ? 1 : (c8 <= 512 ? 2 : 4); }
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

// Rows a lane works on at once (beside those it has under way), and workgroups: about what the registers let reside, which
// then walk the rows.  More of either costs: at 32768 pixels of 1024 bf16 channels kept in 8 bits, forward and backward
// take 41 and 37 us with these, 48 and 47 with 1536 and 1280 workgroups, 54 and 56 with 2048 and 1024 that fetch no row
// ahead.
static int ln_unroll(const LNShape& s) { return s.v == 1 ? 2 : 1; }
#define LN_FWD_BLOCKS 1024
#define LN_BWD_BLOCKS 768

template <int DT, bool KEEP> static int ln_fwd_launch(const LNParams& p, const LNShape& s, hipStream_t st) {
  long long blocks = ln_blocks(p.rows, s, ln_unroll(s));
  if (blocks > LN_FWD_BLOCKS) blocks = LN_FWD_BLOCKS;
  const dim3 g((unsigned)blocks), b(256);
  if (s.wg) {
    if (s.v == 1) hipLaunchKernelGGL((ln_fwd_kernel<DT, true, 1, 2, KEEP>), g, b, 0, st, p);
    else if (s.v == 2) hipLaunchKernelGGL((ln_fwd_kernel<DT, true, 2, 1, KEEP>), g, b, 0, st, p);
    else hipLaunchKernelGGL((ln_fwd_kernel<DT, true, 4, 1, KEEP>), g, b, 0, st, p);
  } else if (s.v == 1) hipLaunchKernelGGL((ln_fwd_kernel<DT, false, 1, 2, KEEP>), g, b, 0, st, p);
  else hipLaunchKernelGGL((ln_fwd_kernel<DT, false, 2, 1, KEEP>), g, b, 0, st, p);
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

extern "C" int csmri_ln_bwd_rows(long long npix, int C) {
  if (npix <= 0 || C <= 0) return 0;
  const LNShape s = ln_shape(C);
  const long long b = ln_blocks(npix, s, ln_unroll(s));
  // What two workgroups would take, one takes in two turns and needs no second launch for the sums: a call on 128 pixels
  // of 64 channels 13.8 us instead of 16.7, 6.9 instead of 7.1 when replayed.  In four turns a replay is slower (256 pixels
  // 9.4, 7.1), and so are two of the widest rows (2 x 8192 19.7, 17.0).
  if (b == 2 && s.v < 4) return 1;
  return (int)(b > LN_BWD_BLOCKS ? LN_BWD_BLOCKS : b);
}

template <int DT, bool KEPT> static int ln_bwd_launch(const LNParams& p, const LNShape& s, int blocks, hipStream_t st) {
  const dim3 g(blocks), b(256);
  const size_t lds = s.wg ? 0 : 2 * (size_t)s.group * s.v * 8 * sizeof(float);
  if (s.wg) {
    if (s.v == 1) hipLaunchKernelGGL((ln_bwd_kernel<DT, true, 1, 2, KEPT>), g, b, lds, st, p);
    else if (s.v == 2) hipLaunchKernelGGL((ln_bwd_kernel<DT, true, 2, 1, KEPT>), g, b, lds, st, p);
    else hipLaunchKernelGGL((ln_bwd_kernel<DT, true, 4, 1, KEPT>), g, b, lds, st, p);
  } else if (s.v == 1) hipLaunchKernelGGL((ln_bwd_kernel<DT, false, 1, 2, KEPT>), g, b, lds, st, p);
  else hipLaunchKernelGGL((ln_bwd_kernel<DT, false, 2, 1, KEPT>), g, b, lds, st, p);
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
    CSMRI_CHECK_ARG(!buffers_meet(dgamma, C_real, dbeta, C_real));
    int rc = CSMRI_OK;
    if (dgamma && !accumulate) rc = csmri_fill_f32(dgamma, C_real, 0.f, stream);
    if (rc == CSMRI_OK && dbeta && !accumulate) rc = csmri_fill_f32(dbeta, C_real, 0.f, stream);
    return rc;
  }
  CSMRI_CHECK_ARG(dz && (x != NULL) != (q8 != NULL) && (!q8 || (s8 && stats)) && (!x || x_pix_stride >= C));
  CSMRI_CHECK_ARG(slope == 1.f || x || z);                  // the sign of y is not to be had from rounded inputs
  CSMRI_CHECK_ARG(slope >= 0.f || !z);                      // nor from z where negative outputs turn positive
  CSMRI_CHECK_ARG(!dgamma || partial);
  CSMRI_CHECK_ARG(!dx || (dx != dz && dx != x && dx != z));
  if (!ln_aligned(dz, dz_pix_stride, dtype) || (x && !ln_aligned(x, x_pix_stride, dtype)) ||
      (z && !ln_aligned(z, z_pix_stride, dtype)) || (dx && !ln_aligned(dx, dx_pix_stride, dtype)) ||
      ((uintptr_t)q8 & 7) || ((uintptr_t)affine_snap & 15)) return CSMRI_E_ALIGN;
  CSMRI_CHECK_ARG(!buffers_meet(dgamma, C_real, dbeta, C_real));
  LNParams p = {};
  p.x = x; p.xps = x_pix_stride;
  p.q = (const unsigned char*)q8; p.s = s8; p.stats_in = stats;
  p.gz = dz; p.gps = dz_pix_stride; p.z = z; p.zps = z_pix_stride;
  p.out = dx; p.ops = dx_pix_stride;
  p.rows = npix; p.C = C; p.C_real = C_real;
  p.gamma = affine_snap; p.beta = affine_snap + C;
  p.eps = eps; p.slope = slope;
  p.partial = dgamma ? partial : NULL;
  p.dgamma = dgamma; p.dbeta = dbeta; p.accumulate = accumulate;
  const LNShape s = ln_shape(C);
  p.group = s.group;
  const int blocks = csmri_ln_bwd_rows(npix, C);
  int rc;
  if (dtype == CSMRI_F32) rc = q8 ? ln_bwd_launch<CSMRI_F32, true>(p, s, blocks, st) : ln_bwd_launch<CSMRI_F32, false>(p, s, blocks, st);
  else rc = q8 ? ln_bwd_launch<CSMRI_BF16, true>(p, s, blocks, st) : ln_bwd_launch<CSMRI_BF16, false>(p, s, blocks, st);
  if (rc != CSMRI_OK || !dgamma || blocks == 1) return rc;
  return micro_colsum2(partial, blocks, 2LL * C_real, C_real, dgamma, C_real, dbeta, accumulate, st);
}
