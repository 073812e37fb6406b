// dig3d — the output head's losses at sizes where launches and copies cost more than the products (head.hip includes this).
//
// One float32 product kernel on 64 x 64 tiles (v_mfma_f32_16x16x4_f32, k steps of 32) that reads x and W where they are: any
// type, width, pitch or alignment, converted on the way into LDS, so there is no copy, no scale and no padding.  e is float32
// and carries the whole incoming gradient.  Two launches forward, three backward (e, then gx and gw in one launch, then the
// sum of gx's k ranges); gb is the column of gw that a column of ones beside x would have.
#pragma once

#define SM_BK 32
#define SM_PITCH 80          // floats per k row of an LDS tile: 4 rows of 16 lanes fall on 64 different banks

struct SmOperand {
  const void* p;
  int dt;                    // type (DT_*); e is DT_F32
  int64_t ld;
  int own, k;                // extents of the own index and of k; beyond them zeros are read
  const float* mask;         // per k row (TR only): rows with 0 are read as zeros, whatever they hold
  int ones;                  // this own index reads as 1 (TR only), -1: none
};

// 8 elements of one row, zeros beyond `left`
__device__ __forceinline__ void sm_row8(const void* p, int dt, int64_t at, int left, float* f) {
  if (left >= 8) {
    if (dt == DT_F32) {
      const RowVec<float, 8> v = *(const RowVec<float, 8>*)((const float*)p + at);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = v.v[i];
    } else if (dt == DT_BF16) {
      const RowVec<bf16_t, 8> v = *(const RowVec<bf16_t, 8>*)((const bf16_t*)p + at);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = (float)v.v[i];
    } else {
      const RowVec<f16_t, 8> v = *(const RowVec<f16_t, 8>*)((const f16_t*)p + at);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = (float)v.v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < left ? load_as(p, dt, at + i) : 0.f;
  }
}

// this thread's 8 elements of a 64 x 32 operand tile: not TR: 8 k of one own index; TR: 8 own indices of one k
template <bool TR>
__device__ __forceinline__ void sm_fetch(const SmOperand& o, int own0, int k0, int tid, float* f) {
  if constexpr (!TR) {
    const int r = own0 + (tid >> 2), k = k0 + (tid & 3) * 8;
    sm_row8(o.p, o.dt, (int64_t)r * o.ld + k, r < o.own ? o.k - k : 0, f);
  } else {
    const int k = k0 + (tid >> 3), c = own0 + (tid & 7) * 8;
    const bool in = k < o.k && (!o.mask || o.mask[k] != 0.f);
    sm_row8(o.p, o.dt, (int64_t)k * o.ld + c, in ? o.own - c : 0, f);
    if (o.ones >= 0 && k < o.k) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = c + i == o.ones ? 1.f : f[i];
    }
  }
}
template <bool TR>
__device__ __forceinline__ void sm_stage(float* lds, int tid, const float* f) {
  if constexpr (!TR) {
    const int r = tid >> 2, k = (tid & 3) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) lds[(k + i) * SM_PITCH + r] = f[i];
  } else {
    float* d = lds + (tid >> 3) * SM_PITCH + (tid & 7) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) d[i] = f[i];
  }
}

// acc[x][y]: out[j, i] = sum over k in [ks, ke) of Q[j, k] P[i, k] for i = i0 + 32 (wave & 1) + 16 x + 4 (lane >> 4) + r,
// j = j0 + 32 (wave >> 1) + 16 y + (lane & 15).  A k step's sum is formed by itself and then added: in one chain of D / 4 additions
// the loss of one row of 1024 is off by 1e-6.
template <bool PT, bool QT>
__device__ __forceinline__ void sm_product(const SmOperand& P, const SmOperand& Q, int i0, int j0, int ks, int ke, float* lds,
                                           f32x4 (&acc)[2][2]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  constexpr int TILE = SM_BK * SM_PITCH;
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int y = 0; y < 2; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
  float fp[8], fq[8];
  if (ks < ke) {
    sm_fetch<PT>(P, i0, ks, tid, fp);
    sm_fetch<QT>(Q, j0, ks, tid, fq);
  }
  int buf = 0;
  for (int k0 = ks; k0 < ke; k0 += SM_BK, buf ^= 1) {
    float* sp = lds + buf * 2 * TILE;
    float* sq = sp + TILE;
    sm_stage<PT>(sp, tid, fp);
    sm_stage<QT>(sq, tid, fq);
    __syncthreads();
    if (k0 + SM_BK < ke) {
      sm_fetch<PT>(P, i0, k0 + SM_BK, tid, fp);
      sm_fetch<QT>(Q, j0, k0 + SM_BK, tid, fq);
    }
    const float* ap = sp + (lane >> 4) * SM_PITCH + (wave & 1) * 32 + (lane & 15);
    const float* aq = sq + (lane >> 4) * SM_PITCH + (wave >> 1) * 32 + (lane & 15);
    f32x4 sum[2][2] = {};
#pragma unroll
    for (int kk = 0; kk < SM_BK; kk += 4) {
      const float p0 = ap[kk * SM_PITCH], p1 = ap[kk * SM_PITCH + 16], q0 = aq[kk * SM_PITCH], q1 = aq[kk * SM_PITCH + 16];
      sum[0][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(p0, q0, sum[0][0], 0, 0, 0);
      sum[0][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(p0, q1, sum[0][1], 0, 0, 0);
      sum[1][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(p1, q0, sum[1][0], 0, 0, 0);
      sum[1][1] = __builtin_amdgcn_mfma_f32_16x16x4f32(p1, q1, sum[1][1], 0, 0, 0);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int y = 0; y < 2; ++y) acc[x][y] += sum[x][y];
  }
}

struct SmArgs {
  SmOperand W, x;            // not TR: rows of classes / of the batch
  const void* bias;
  int dt, N, D, V;
  float inv_tau, f;          // f: tau for the teacher's loss, else 1
  const int64_t* target;
  int64_t ignore;
  const float* live;
  float2* part;              // [N][tiles]
  int tiles;
  float* zt;
  const float *m, *rs, *loss, *g, *count;
  int per_row;
  float* coef;               // [2][N], written by the e kernel: does the row have a loss; the gradient that reaches its logits
  float* E;                  // [N][ldE]
  int64_t ldE;
  void *gx, *gw, *gb;
  float* slots;              // [splits][N][D] partial gx, or null
  int splits, gx_tiles, gw_tiles;
};

template <bool GRAD>
__global__ void __launch_bounds__(256) k_head_small_logits(SmArgs a) {
  __shared__ float lds[4 * SM_BK * SM_PITCH];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int i0 = blockIdx.x * 64, j0 = blockIdx.y * 64;
  f32x4 acc[2][2];
  sm_product<false, false>(a.W, a.x, i0, j0, 0, a.D, lds, acc);
  const int ib = i0 + (wave & 1) * 32 + 4 * (lane >> 4), jb = (wave >> 1) * 32 + (lane & 15);
#pragma unroll
  for (int x = 0; x < 2; ++x)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = ib + x * 16 + r;
      const float b = a.bias && i < a.V ? load_as(a.bias, a.dt, i) : 0.f;
#pragma unroll
      for (int y = 0; y < 2; ++y) acc[x][y][r] = (acc[x][y][r] + b) * a.inv_tau;
    }
  if constexpr (!GRAD) {
    float* sh = lds;                       // [2][64][2]
    __syncthreads();
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int jl = jb + y * 16, j = j0 + jl;
      const int64_t tg = a.target && j < a.N ? a.target[j] : -1;
      float m = -INFINITY, s = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = ib + x * 16 + r;
          if (i < a.V && i == tg) a.zt[j] = acc[x][y][r];
          if (i >= a.V || i == tg) acc[x][y][r] = -INFINITY;
          m = fmaxf(m, acc[x][y][r]);
        }
      m = fmaxf(m, __shfl_xor(m, 16, 64));
      m = fmaxf(m, __shfl_xor(m, 32, 64));
      const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f((acc[x][y][r] - ms) * L2E);
      s += __shfl_xor(s, 16, 64);
      s += __shfl_xor(s, 32, 64);
      if (lane < 16) {
        sh[((wave & 1) * 64 + jl) * 2] = m;
        sh[((wave & 1) * 64 + jl) * 2 + 1] = s;
      }
    }
    __syncthreads();
    const int jl = threadIdx.x;
    if (jl < 64 && j0 + jl < a.N) {
      const float m1 = sh[jl * 2], s1 = sh[jl * 2 + 1], m2 = sh[(64 + jl) * 2], s2 = sh[(64 + jl) * 2 + 1];
      const float m = fmaxf(m1, m2), ms = m == -INFINITY ? 0.f : m;
      a.part[(int64_t)(j0 + jl) * a.tiles + blockIdx.x] =
          make_float2(m, s1 * __builtin_amdgcn_exp2f((m1 - ms) * L2E) + s2 * __builtin_amdgcn_exp2f((m2 - ms) * L2E));
    }
  } else {
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int j = j0 + jb + y * 16;
      if (j >= a.N) continue;
      const float alive = a.target ? (a.target[j] != a.ignore ? 1.f : 0.f) : a.live[j];
      float c = (a.per_row ? a.g[j] : a.g[0] / (a.count ? *a.count : 1.f)) * a.f * alive;
      if (alive == 0.f) c = 0.f;
      if (blockIdx.x == 0 && lane < 16 && (wave & 1) == 0) {
        a.coef[j] = alive;
        a.coef[a.N + j] = c;
      }
      const float m = a.m[j], cp = c * a.rs[j];
      const int64_t tg = a.target ? a.target[j] : -1;
      const float et = a.target ? c * expm1f(-a.loss[j]) : 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = ib + x * 16 + r;
          if (i >= a.V) continue;
          const float p = cp * __builtin_amdgcn_exp2f((acc[x][y][r] - m) * L2E);
          a.E[(int64_t)j * a.ldE + i] = alive == 0.f ? 0.f : i == tg ? et : p;
        }
    }
  }
}

// blocks [0, gx_tiles * splits): gx[n, d] = sum_v e[n, v] W[v, d], a range of v each; the rest: gw[v, d] = sum_n e[n, v] x[n, d]
// and gb[v], the column d = D of it with x[n, D] = 1
__global__ void __launch_bounds__(256) k_head_small_grads(SmArgs a) {
  __shared__ float lds[4 * SM_BK * SM_PITCH];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ir = (wave & 1) * 32 + 4 * (lane >> 4), jr = (wave >> 1) * 32 + (lane & 15);
  f32x4 acc[2][2];
  const int b = blockIdx.x, ngx = a.gx_tiles * a.splits;
  if (b < ngx) {
    const int dt = (a.D + 63) / 64, z = b / a.gx_tiles, t = b % a.gx_tiles;
    const int i0 = (t % dt) * 64, j0 = (t / dt) * 64;
    const int steps = (a.V + SM_BK - 1) / SM_BK;
    const int ks = (int)((int64_t)steps * z / a.splits) * SM_BK, ke = min(a.V, (int)((int64_t)steps * (z + 1) / a.splits) * SM_BK);
    SmOperand P = a.W, Q = {a.E, DT_F32, a.ldE, a.N, a.V, nullptr, -1};
    P.own = a.D;
    P.k = a.V;
    sm_product<true, false>(P, Q, i0, j0, ks, ke, lds, acc);
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int j = j0 + jr + y * 16;
      if (j >= a.N) continue;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = i0 + ir + x * 16 + r;
          if (i >= a.D) continue;
          if (a.slots) a.slots[((int64_t)z * a.N + j) * a.D + i] = acc[x][y][r];
          else store_as(a.gx, a.dt, (int64_t)j * a.D + i, acc[x][y][r]);
        }
    }
  } else {
    const int own = a.D + (a.gb ? 1 : 0), dt = (own + 63) / 64, t = b - ngx;
    const int i0 = (t % dt) * 64, j0 = (t / dt) * 64;
    SmOperand P = a.x, Q = {a.E, DT_F32, a.ldE, a.V, a.N, nullptr, -1};
    P.own = a.D;
    P.k = a.N;
    P.mask = a.coef;
    P.ones = a.gb ? a.D : -1;
    sm_product<true, true>(P, Q, i0, j0, 0, a.N, lds, acc);
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      const int j = j0 + jr + y * 16;
      if (j >= a.V) continue;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = i0 + ir + x * 16 + r;
          if (i < a.D) {
            if (a.gw) store_as(a.gw, a.dt, (int64_t)j * a.D + i, acc[x][y][r]);
          } else if (i == a.D && a.gb) {
            store_as(a.gb, a.dt, j, acc[x][y][r]);
          }
        }
    }
  }
}
