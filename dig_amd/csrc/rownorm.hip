// dig3d — layer norm over the channels of a row, forward and backward with the reduction of the parameters' gradients.
//
//   mean = sum_c x / C;  r = 1 / sqrt(sum_c (x - mean)^2 / C + eps);  h = (x - mean) r;  y = w h + b
//   gh = w gy;  gx = r (gh - mean_c(gh) - h mean_c(gh h));  gw = sum_rows gy h;  gb = sum_rows gy
//
// Bound: memory.  One read of x and one write of y; in the backward one read of x and gy and one write of gx.  A row stays
// in the registers of its group of threads between the passes over it (mean, centred squares, output), so the variance is
// the centred one, in 32 bits, at the traffic of a single pass.  Groups: 8 to 64 lanes of a wave for the widths that fit
// them (several short rows per wave), 256 or 1024 threads beyond; rows longer than 1024 threads hold are read again.
// The parameters' gradients are summed over the rows of a workgroup in registers, joined through LDS and written as one
// partial row per workgroup; a second kernel adds the partials in a fixed order (no atomics: the same bits every time).
#include "half16.h"

#define RN_TPB 256

// sum over the TPR threads of a row's group, in every one of them.  One-wave groups: lane exchanges; larger ones: LDS.
template <int TPR>
__device__ __forceinline__ float rn_sum(float v, float* sh) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    __syncthreads();                       // the previous sum has been read
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) v += sh[w];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ void rn_sum2(float& a, float& b, float* sh) {
#pragma unroll
  for (int o = (TPR < 64 ? TPR : 64) / 2; o > 0; o >>= 1) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
  if constexpr (TPR > 64) {
    constexpr int NW = TPR / 64;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      sh[threadIdx.x >> 6] = a;
      sh[16 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      a += sh[w];
      b += sh[16 + w];
    }
  }
}

// elements [c, c + N) of a row, zero beyond its end
template <class T, int N>
__device__ __forceinline__ void rn_load(const T* __restrict__ row, int c, int C, float* f) {
  if (c + N <= C) {
    const RowVec<T, N> u = *(const RowVec<T, N>*)(row + c);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = (float)u.v[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = c + i < C ? (float)row[c + i] : 0.f;
  }
}
template <class T, int N>
__device__ __forceinline__ void rn_store(T* __restrict__ row, int c, int C, const float* f) {
  if (c + N <= C) {
    RowVec<T, N> u;
#pragma unroll
    for (int i = 0; i < N; ++i) u.v[i] = to_t<T>(f[i]);
    *(RowVec<T, N>*)(row + c) = u;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (c + i < C) row[c + i] = to_t<T>(f[i]);
  }
}
template <int N>
__device__ __forceinline__ void rn_param(const void* __restrict__ p, int dt, int c, int C, float none, float* f) {
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = p && c + i < C ? load_as(p, dt, c + i) : none;
}

// TPR threads hold a row of at most TPR * NV * N elements; TPR > 64: the whole workgroup is one group
template <class T, int TPR, int NV>
__global__ void __launch_bounds__(TPR > RN_TPB ? TPR : RN_TPB)
    k_rownorm_fwd(const T* __restrict__ x, int64_t ldx, int R, int C, const void* __restrict__ w,
                  const void* __restrict__ b, int wdt, float eps, T* __restrict__ y, float* __restrict__ mean_out,
                  float* __restrict__ rstd_out) {
  constexpr int N = VecLen<T>::n;
  constexpr int TPB = TPR > RN_TPB ? TPR : RN_TPB;
  __shared__ float sh[32];
  const int t = threadIdx.x % TPR;
  const float inv_c = 1.0f / (float)C;
  // a few rows per group, strided by the grid: the parameters are converted once
  float wv[NV][N], bv[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    rn_param<N>(w, wdt, (j * TPR + t) * N, C, 1.f, wv[j]);
    rn_param<N>(b, wdt, (j * TPR + t) * N, C, 0.f, bv[j]);
  }
  const int64_t step = (int64_t)gridDim.x * (TPB / TPR);
  // the bound is uniform over the groups of a workgroup where they meet at a barrier (TPB == TPR: one group)
  for (int64_t r = (int64_t)blockIdx.x * (TPB / TPR) + threadIdx.x / TPR; r < R; r += step) {
    float f[NV][N];
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      rn_load<T, N>(x + r * ldx, (j * TPR + t) * N, C, f[j]);
#pragma unroll
      for (int i = 0; i < N; ++i) s += f[j][i];
    }
    const float m = rn_sum<TPR>(s, sh) * inv_c;
    float q = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = (j * TPR + t) * N + i < C ? f[j][i] - m : 0.f;
        f[j][i] = d;
        q = __fmaf_rn(d, d, q);
      }
    const float rs = 1.0f / sqrtf(rn_sum<TPR>(q, sh) * inv_c + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < N; ++i) f[j][i] = __fmaf_rn(f[j][i] * rs, wv[j][i], bv[j][i]);
      rn_store<T, N>(y + r * C, (j * TPR + t) * N, C, f[j]);
    }
    if (t == 0 && mean_out) {
      mean_out[r] = m;
      rstd_out[r] = rs;
    }
  }
}

// rows longer than a workgroup's registers hold: three passes, the second and third from the caches
template <class T>
__global__ void __launch_bounds__(1024)
    k_rownorm_fwd_long(const T* __restrict__ x, int64_t ldx, int R, int C, const void* __restrict__ w,
                       const void* __restrict__ b, int wdt, float eps, T* __restrict__ y, float* __restrict__ mean_out,
                       float* __restrict__ rstd_out) {
  constexpr int N = VecLen<T>::n;
  __shared__ float sh[32];
  const float inv_c = 1.0f / (float)C;
  for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
    const T* row = x + r * ldx;
    float f[N], g[N], s = 0.f, q = 0.f;
    for (int64_t c = threadIdx.x * N; c < C; c += 1024 * N) {
      rn_load<T, N>(row, (int)c, C, f);
#pragma unroll
      for (int i = 0; i < N; ++i) s += f[i];
    }
    const float m = rn_sum<1024>(s, sh) * inv_c;
    for (int64_t c = threadIdx.x * N; c < C; c += 1024 * N) {
      rn_load<T, N>(row, (int)c, C, f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = c + i < C ? f[i] - m : 0.f;
        q = __fmaf_rn(d, d, q);
      }
    }
    const float rs = 1.0f / sqrtf(rn_sum<1024>(q, sh) * inv_c + eps);
    for (int64_t c = threadIdx.x * N; c < C; c += 1024 * N) {
      rn_load<T, N>(row, (int)c, C, f);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = (f[i] - m) * rs;
      rn_param<N>(w, wdt, (int)c, C, 1.f, g);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] *= g[i];
      rn_param<N>(b, wdt, (int)c, C, 0.f, g);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] += g[i];
      rn_store<T, N>(y + r * C, (int)c, C, f);
    }
    if (threadIdx.x == 0 && mean_out) {
      mean_out[r] = m;
      rstd_out[r] = rs;
    }
  }
}

// part [gridDim.x][2][C]: the workgroup's sums of gy h and gy (null: no parameter takes a gradient)
template <class T, int TPR, int NV>
__global__ void __launch_bounds__(TPR > RN_TPB ? TPR : RN_TPB)
    k_rownorm_bwd(const T* __restrict__ gy, const T* __restrict__ x, int64_t ldx, int R, int C, const void* __restrict__ w,
                  int wdt, const float* __restrict__ mean, const float* __restrict__ rstd, T* __restrict__ gx,
                  float* __restrict__ part) {
  constexpr int N = VecLen<T>::n;
  constexpr int TPB = TPR > RN_TPB ? TPR : RN_TPB;
  constexpr int G = TPB / TPR;               // row groups of the workgroup
  __shared__ float sh[32];
  __shared__ float join[G > 1 ? TPB * N : 1];
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  const float inv_c = 1.0f / (float)C;
  float wv[NV][N], aw[NV][N], ab[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    rn_param<N>(w, wdt, (j * TPR + t) * N, C, 1.f, wv[j]);
#pragma unroll
    for (int i = 0; i < N; ++i) aw[j][i] = ab[j][i] = 0.f;
  }
  const int64_t step = (int64_t)gridDim.x * G;
  for (int64_t r = (int64_t)blockIdx.x * G + grp; r < R; r += step) {
    const float m = mean[r], rs = rstd[r];
    float h[NV][N], g[NV][N], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      rn_load<T, N>(x + r * ldx, (j * TPR + t) * N, C, h[j]);
      rn_load<T, N>(gy + r * C, (j * TPR + t) * N, C, g[j]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float hh = (h[j][i] - m) * rs;  // beyond the row's end g is 0 and nothing of hh is kept
        aw[j][i] = __fmaf_rn(g[j][i], hh, aw[j][i]);
        ab[j][i] += g[j][i];
        const float gh = g[j][i] * wv[j][i];
        s1 += gh;
        s2 = __fmaf_rn(gh, hh, s2);
        h[j][i] = hh;
        g[j][i] = gh;
      }
    rn_sum2<TPR>(s1, s2, sh);
    s1 *= inv_c;
    s2 *= inv_c;
    if (gx) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < N; ++i) g[j][i] = rs * (g[j][i] - s1 - h[j][i] * s2);
        rn_store<T, N>(gx + r * C, (j * TPR + t) * N, C, g[j]);
      }
    }
  }
  if (!part) return;
  float* p = part + (int64_t)blockIdx.x * 2 * C;
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float* a = k == 0 ? aw[j] : ab[j];
      if constexpr (G > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) join[i * TPB + threadIdx.x] = a[i];
        __syncthreads();
        for (int e = threadIdx.x; e < TPR * N; e += TPB) {      // element e % N of lane e / N, over the groups in order
          float s = 0.f;
          for (int q = 0; q < G; ++q) s += join[(e % N) * TPB + q * TPR + e / N];
          const int c = j * TPR * N + e;
          if (c < C) p[(int64_t)k * C + c] = s;
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int c = (j * TPR + t) * N + i;
          if (c < C) p[(int64_t)k * C + c] = a[i];
        }
      }
    }
}

// long rows: the partial row itself is the accumulator (this thread's columns of it are no one else's)
template <class T>
__global__ void __launch_bounds__(1024)
    k_rownorm_bwd_long(const T* __restrict__ gy, const T* __restrict__ x, int64_t ldx, int R, int C,
                       const void* __restrict__ w, int wdt, const float* __restrict__ mean, const float* __restrict__ rstd,
                       T* __restrict__ gx, float* __restrict__ part) {
  constexpr int N = VecLen<T>::n;
  __shared__ float sh[32];
  const float inv_c = 1.0f / (float)C;
  float* p = part ? part + (int64_t)blockIdx.x * 2 * C : nullptr;
  bool first = true;
  for (int64_t r = blockIdx.x; r < R; r += gridDim.x) {
    const float m = mean[r], rs = rstd[r];
    float h[N], g[N], wv[N], s1 = 0.f, s2 = 0.f;
    for (int64_t c = threadIdx.x * N; c < C; c += 1024 * N) {
      rn_load<T, N>(x + r * ldx, (int)c, C, h);
      rn_load<T, N>(gy + r * C, (int)c, C, g);
      rn_param<N>(w, wdt, (int)c, C, 1.f, wv);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float hh = (h[i] - m) * rs, gh = g[i] * wv[i];
        s1 += gh;
        s2 = __fmaf_rn(gh, hh, s2);
        if (p && c + i < C) {
          p[c + i] = first ? g[i] * hh : __fmaf_rn(g[i], hh, p[c + i]);
          p[(int64_t)C + c + i] = first ? g[i] : p[(int64_t)C + c + i] + g[i];
        }
      }
    }
    first = false;
    rn_sum2<1024>(s1, s2, sh);
    s1 *= inv_c;
    s2 *= inv_c;
    if (gx)
      for (int64_t c = threadIdx.x * N; c < C; c += 1024 * N) {
        rn_load<T, N>(x + r * ldx, (int)c, C, h);
        rn_load<T, N>(gy + r * C, (int)c, C, g);
        rn_param<N>(w, wdt, (int)c, C, 1.f, wv);
#pragma unroll
        for (int i = 0; i < N; ++i) g[i] = rs * (g[i] * wv[i] - s1 - (h[i] - m) * rs * s2);
        rn_store<T, N>(gx + r * C, (int)c, C, g);
      }
  }
}

// out[c] = sum_b part[b][c]: 64 slices of the partial rows, each in order, then the slices in order; 16 columns a workgroup
// (64-byte pieces of a row, four of them in flight).  Columns [0, C) go to gw and [C, 2C) to gb (either may be null)
__global__ void __launch_bounds__(1024) k_rownorm_params(const float* __restrict__ part, int nb, int C, void* __restrict__ gw,
                                                          void* __restrict__ gb, int wdt) {
  __shared__ float sh[64][17];
  const int col = threadIdx.x & 15, sl = threadIdx.x >> 4;
  const int64_t c = (int64_t)blockIdx.x * 16 + col, C2 = 2 * (int64_t)C;
  float s = 0.f;
  if (c < C2) {
#pragma unroll 4
    for (int b = sl; b < nb; b += 64) s += part[(int64_t)b * C2 + c];
  }
  sh[sl][col] = s;
  __syncthreads();
  if (sl != 0 || c >= C2) return;
  s = 0.f;
#pragma unroll
  for (int q = 0; q < 64; ++q) s += sh[q][col];
  if (c < C) {
    if (gw) store_as(gw, wdt, c, s);
  } else if (gb) {
    store_as(gb, wdt, c - C, s);
  }
}

// ---- host ------------------------------------------------------------------------------------------------------------------
// the smallest group whose registers hold the row (the backward keeps five values of each element: 16 elements a thread are the
// most that 1024 threads hold)
static inline void rn_pick(int C, int n, int& tpr, int& nv) {
  const int v = (C + n - 1) / n;
  if (v <= 8) { tpr = 8; nv = 1; }
  else if (v <= 16) { tpr = 16; nv = 1; }
  else if (v <= 32) { tpr = 32; nv = 1; }
  else if (v <= 64) { tpr = 64; nv = 1; }
  else if (v <= 128) { tpr = 64; nv = 2; }
  else if (v <= 256) { tpr = 256; nv = 1; }
  else if (v <= 512) { tpr = 256; nv = 2; }
  else if (v <= 1024) { tpr = 1024; nv = 1; }
  else if (v <= 2048) { tpr = 1024; nv = 2; }
  else if (v <= 4096 && n == 4) { tpr = 1024; nv = 4; }
  else { tpr = 0; nv = 0; }
}

// Workgroups per CU, the rows dealt over them: enough bytes in flight, and no more rows at once than the caches and the
// memory's pages like (TB/s, forward / backward):
//   131072 x 1024 bf16 (a wave per row):   2: 3.5 / 3.7   3: 4.8 / 5.0   4: 5.2 / 5.4   6: 4.9 / 4.5   16: 4.1 / 4.4
//   262144 x 256 f32 (a wave per row):     2: 3.2 / 5.2   3: 4.6 / 5.7   4: 5.4 / 5.3   6: 5.3 / 5.0
//   65536 x 2048 bf16 (256 threads, 1):    3: 3.6 / 4.2   4: 4.4 / 4.8   6: 5.3 / 5.1   8: 5.1 / 4.3
//   32768 x 4096 bf16 (256 threads, 2):    2: 3.1 / 3.3   3: 4.5 / 4.5   4: 5.0 / 3.2
//   32768 x 2048 f32 (256 threads, 2):     2: 4.6 / 5.7   3: 5.8 / 5.4   4: 5.3 / 5.1
//   16384 x 8192 bf16 (1024 threads):      1: 3.6 / 4.2   2: 5.0 / 4.1   4: 4.7 / 3.7
// (1024 threads, 16 elements each: 8192 x 8192 f32 4.8 / 4.6 where a row that is read again reaches 2.4 / 1.7; 4096 x 12288 bf16
// 3.3 / 2.5 and 1.3 / 0.6)
static inline int rn_per_cu(int tpr, int nv, bool f32, bool backward) {
  if (tpr <= 64 && tpr) return backward && f32 ? 3 : 4;
  if (tpr == 256 && nv == 1) return backward ? (f32 ? 3 : 5) : 6;
  if (tpr == 256) return backward ? (f32 ? 2 : 3) : (f32 ? 3 : 4);
  return backward && !f32 ? 1 : 2;
}

static inline int64_t rn_groups_per_block(int tpr) { return tpr == 0 || tpr > RN_TPB ? 1 : RN_TPB / tpr; }

template <class T, int TPR, int NV>
static void rn_launch_fwd(const void* x, int64_t ldx, int R, int C, const void* w, const void* b, int wdt, float eps, void* y,
                          float* mean, float* rstd, int grid, hipStream_t st) {
  hipLaunchKernelGGL((k_rownorm_fwd<T, TPR, NV>), dim3(grid), dim3(TPR > RN_TPB ? TPR : RN_TPB), 0, st, (const T*)x, ldx, R, C,
                     w, b, wdt, eps, (T*)y, mean, rstd);
}
template <class T, int TPR, int NV>
static void rn_launch_bwd(const void* gy, const void* x, int64_t ldx, int R, int C, const void* w, int wdt, const float* mean,
                          const float* rstd, void* gx, float* part, int grid, hipStream_t st) {
  hipLaunchKernelGGL((k_rownorm_bwd<T, TPR, NV>), dim3(grid), dim3(TPR > RN_TPB ? TPR : RN_TPB), 0, st, (const T*)gy,
                     (const T*)x, ldx, R, C, w, wdt, mean, rstd, (T*)gx, part);
}

template <class T>
static void rn_fwd(const void* x, int64_t ldx, int R, int C, const void* w, const void* b, int wdt, float eps, void* y,
                   float* mean, float* rstd, hipStream_t st) {
  int tpr, nv;
  rn_pick(C, VecLen<T>::n, tpr, nv);
  const int64_t per = rn_groups_per_block(tpr);
  int64_t g = (R + per - 1) / per;
  const int64_t cap = (int64_t)rn_per_cu(tpr, nv, sizeof(T) == 4, false) * dig3d_num_cus();
  const int grid = (int)(g < cap ? g : cap);
#define RN_CASE(TP, NVV)                                                                                       \
  if (tpr == TP && nv == NVV)                                                                                  \
    return rn_launch_fwd<T, TP, NVV>(x, ldx, R, C, w, b, wdt, eps, y, mean, rstd, grid, st);
  RN_CASE(8, 1) RN_CASE(16, 1) RN_CASE(32, 1) RN_CASE(64, 1) RN_CASE(64, 2)
  RN_CASE(256, 1) RN_CASE(256, 2) RN_CASE(1024, 1) RN_CASE(1024, 2)
  if constexpr (sizeof(T) == 4) { RN_CASE(1024, 4) }
#undef RN_CASE
  hipLaunchKernelGGL((k_rownorm_fwd_long<T>), dim3(grid), dim3(1024), 0, st, (const T*)x, ldx, R, C, w, b, wdt, eps, (T*)y,
                     mean, rstd);
}

template <class T>
static void rn_bwd(const void* gy, const void* x, int64_t ldx, int R, int C, const void* w, int wdt, const float* mean,
                   const float* rstd, void* gx, float* part, int grid, hipStream_t st) {
  int tpr, nv;
  rn_pick(C, VecLen<T>::n, tpr, nv);
#define RN_CASE(TP, NVV)                                                                                       \
  if (tpr == TP && nv == NVV)                                                                                  \
    return rn_launch_bwd<T, TP, NVV>(gy, x, ldx, R, C, w, wdt, mean, rstd, gx, part, grid, st);
  RN_CASE(8, 1) RN_CASE(16, 1) RN_CASE(32, 1) RN_CASE(64, 1) RN_CASE(64, 2)
  RN_CASE(256, 1) RN_CASE(256, 2) RN_CASE(1024, 1) RN_CASE(1024, 2)
  if constexpr (sizeof(T) == 4) { RN_CASE(1024, 4) }
#undef RN_CASE
  hipLaunchKernelGGL((k_rownorm_bwd_long<T>), dim3(grid), dim3(1024), 0, st, (const T*)gy, (const T*)x, ldx, R, C, w, wdt,
                     mean, rstd, (T*)gx, part);
}

extern "C" {

int dig3d_rownorm_bwd_blocks(int R, int C, int dtype) {
  if (R <= 0 || C <= 0 || C >= (1 << 25) || dtype < 0 || dtype > 2) return 0;
  int tpr, nv;
  rn_pick(C, dtype == DT_F32 ? 4 : 8, tpr, nv);
  const int64_t per = rn_groups_per_block(tpr);
  const int64_t g = (R + per - 1) / per;
  const int64_t cap = (int64_t)rn_per_cu(tpr, nv, dtype == DT_F32, true) * dig3d_num_cus();
  return (int)(g < cap ? g : cap);
}

int dig3d_rownorm_fwd(int dtype, const void* x, int64_t ldx, int R, int C, const void* w, const void* b, int wdtype, float eps,
                      void* y, float* mean, float* rstd, void* stream) {
  DIG3D_ENTER();
  if (R < 0 || C <= 0 || C >= (1 << 25) || ldx < C || dtype < 0 || dtype > 2 || wdtype < 0 || wdtype > 2) return DIG3D_ERR_ARG;
  if (R == 0) return DIG3D_OK;
  if (!x || !y || (!mean) != (!rstd)) return DIG3D_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_F32) rn_fwd<float>(x, ldx, R, C, w, b, wdtype, eps, y, mean, rstd, st);
  else if (dtype == DT_BF16) rn_fwd<bf16_t>(x, ldx, R, C, w, b, wdtype, eps, y, mean, rstd, st);
  else rn_fwd<f16_t>(x, ldx, R, C, w, b, wdtype, eps, y, mean, rstd, st);
  DIG3D_CHECK_LAUNCH();
  return DIG3D_OK;
}

int dig3d_rownorm_bwd(int dtype, const void* gy, const void* x, int64_t ldx, int R, int C, const void* w, int wdtype,
                      const float* mean, const float* rstd, void* gx, float* part, int nb, void* gw, void* gb, void* stream) {
  DIG3D_ENTER();
  if (R <= 0 || C <= 0 || C >= (1 << 25) || ldx < C || dtype < 0 || dtype > 2 || wdtype < 0 || wdtype > 2) return DIG3D_ERR_ARG;
  if (!gy || !x || !mean || !rstd || nb != dig3d_rownorm_bwd_blocks(R, C, dtype) || ((gw || gb) && !part))
    return DIG3D_ERR_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DT_F32) rn_bwd<float>(gy, x, ldx, R, C, w, wdtype, mean, rstd, gx, part, nb, st);
  else if (dtype == DT_BF16) rn_bwd<bf16_t>(gy, x, ldx, R, C, w, wdtype, mean, rstd, gx, part, nb, st);
  else rn_bwd<f16_t>(gy, x, ldx, R, C, w, wdtype, mean, rstd, gx, part, nb, st);
  DIG3D_CHECK_LAUNCH();
  if (gw || gb) {
    hipLaunchKernelGGL(k_rownorm_params, dim3((unsigned)((2 * (int64_t)C + 15) / 16)), dim3(1024), 0, st, part, nb, C, gw, gb,
                       wdtype);
    DIG3D_CHECK_LAUNCH();
  }
  return DIG3D_OK;
}

}  // extern "C"
