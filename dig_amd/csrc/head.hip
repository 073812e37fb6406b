// dig3d — the trained output head: losses over the classes of logits z = x W^T + bias that are never kept.
//
//   classes:  loss_n = lse(z_n) - z_n[y_n]                                     e_n = c_n (softmax(z_n) - onehot(y_n))
//   teacher:  loss_n = tau^2 sum_k q_k (log q_k - log p_n[i_k]), p = softmax(z / tau)   e_n = c_n (p_n - scatter(q_n))
//   gx = S e W,  gW = S e^T x,  gb = S sum_n e_n          (c_n S: the gradient that reaches row n, |c_n| <= 1)
// (f16: e is kept to 2^-40 of the largest |c|: 11 bits of every entry down to 2^-29 of it, fewer below)
//
// Four products of 2 N V D operations: the logits, the logits again in the backward (the price of not keeping them), e W and
// e^T x.  Bound: the matrix cores.  All four run on ONE product kernel (k_head_gemm): out[j, i] = sum_k Q[j, k] P[i, k], each
// operand either contiguous along k or along its own index, staged through LDS by 16-byte direct loads and read as matrix
// operands (the second kind by the transposing LDS read), so nothing is transposed in memory.  Its epilogues: the softmax
// statistics of a tile of logits (forward), the gradient e of a piece of the vocabulary (backward), or the stored product.
//
// Types.  bf16 / f16: the inputs as they are, sums in f32; e is rounded once to the same type (up to 2^-8 / 2^-11 of each entry,
// at random sign; with few rows e is two such numbers).  f32: every value, of x, W and e alike, is the sum of three bf16
// numbers v = h + m + l, exactly down to 2^-110 (8 bits each, the exponent range of f32: no scale, no entry's bits depend on
// another's), and a product of two is the six products of them that reach 2^-24 of it: h h, h m, m h, m m, h l, l h, with f32
// sums.  What is dropped (m l, l m, l l) is at most 2^-23 of the term.  Six bf16 products take two thirds of the time of one in
// f32 on this chip.  (Two f16 numbers and three products would take half of that again, but their second number runs out of exponents:
// below 2^-18 of the largest value of its tensor an entry loses bits, and the gradient of an unlikely class has no other entries.)
#include <string.h>

#include "half16.h"

#define HD_BK 64           // the k step of the product kernel
#define L2E 1.44269504088896340736f

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));

template <class T>
__device__ __forceinline__ f32x4 hd_mfma(s16x8 a, s16x8 b, f32x4 c);
template <>
__device__ __forceinline__ f32x4 hd_mfma<bf16_t>(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x4 hd_mfma<f16_t>(s16x8 a, s16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// One operand: a matrix of `rows` rows with pitch `ld` (elements, a multiple of 8; base 16-byte aligned); a value of several numbers
// has each `plane` elements behind the one before, in the same row.
//   not TR: row = the operand's own index, columns = k (k extent a multiple of HD_BK inside the pitch)
//   TR:     row = k, columns = the operand's own index (`cols` of them are readable, a multiple of 8)
// Rows beyond the last are read as the last one: for the own index their results are not used, for k the other operand
// holds zeros there.
struct HdOperand {
  const short* p;
  int64_t ld, plane;
  int rows, cols;
};

enum { EPI_STATS = 0, EPI_GRAD = 1, EPI_OUT = 2 };

struct HdArgs {
  HdOperand P, Q;
  int ni, nj;                // extents of the own indices of P and Q
  int ktiles;                // k steps of one product
  int nseg;                  // not F32: Q as one number, or as two (h h, h l)
  int ti, tj;                // tiles along i and j
  int splits, wgs;           // ranges of the k steps, and workgroups to each
  // logits epilogues: i = class v0 + i, j = row
  const void* bias;
  int dt;                    // type of bias / of the stored output
  const float* S;            // the gradients' common factor
  float inv_tau;
  int64_t v0;                // first class of the piece
  const int64_t* target;     // null: no class is kept apart
  float2* part;              // EPI_STATS [nj][ti_all]: (max, sum of exp) of the tile
  int part_ld, part_c0;
  float* zt;                 // EPI_STATS: the target's logit
  const float *m, *rs;       // EPI_GRAD: softmax = exp(z - m) rs
  const float* loss;
  const float* coef;
  int eplanes;               // not F32: e as one number, or as two (its rounding and what that left)
  short* E;                  // EPI_GRAD [rowsE][eplanes][colsE]
  int64_t colsE;
  int rowsE;
  // EPI_OUT
  float* acc;                // f32 partial slots [splits][nj][ni], written or added to
  int add;
  void* out;                 // or the finished result, row pitch ldo
  int64_t ldo;
};

#define HD_FAR 16777216.0f // 2^24: a float32 product below it is off by less than one

#define E_SCALE 32768.0f   // e in f16 (|e| <= 1) is stored times this: small entries stay normal numbers

// what a product with e is multiplied by
template <class T>
__device__ __forceinline__ float hd_factor(const float* S) {
  return __is_same(T, f16_t) ? *S * (1.f / E_SCALE) : *S;
}

// three bf16 numbers whose sum is v; the first alone where v is an infinity or NaN
struct Bf3 {
  bf16_t h, m, l;
};
__device__ __forceinline__ Bf3 hd_split(float v) {
  Bf3 b;
  b.h = (bf16_t)v;
  float r = v - (float)b.h;
  if (!(fabsf(r) <= 3.402823466e38f)) {    // no finite number, or one that rounds to infinity
    const bool fin = fabsf(v) <= 3.402823466e38f;
    b.h = fin ? (bf16_t)copysignf(3.38953139e38f, v) : b.h;
    r = fin ? v - (float)b.h : 0.f;
  }
  b.m = (bf16_t)r;
  b.l = (bf16_t)(r - (float)b.m);
  return b;
}

// LDS of one stage: P tile then Q tile, HD_BK deep
template <int B>
constexpr int hd_tile_shorts() {
  return B * HD_BK;
}

// an address that is the same in every lane, in scalar registers
__device__ __forceinline__ const char* hd_uniform(const char* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const char*)((uint64_t)hi << 32 | lo);
}

// lane l of load `q` of a wave fetches 16 bytes to LDS offset 1024 q + 16 l of its tile.
// not TR: LDS row r holds 8 chunks of 8 k; chunk s of it is source chunk s ^ f(r), f(r) = (r & 3) | (r >> 3 & 1) << 2: the 16
//         rows of either kind of read below (hd_frag) spread over the banks
// TR:     LDS row k holds B / 8 chunks; chunk s of it is source chunk s ^ (2 g(k) mod B / 8), g(k) = (k & 3) | (k >> 3 & 3) << 2
// The lane's byte offsets from the tile's first element are formed once (32 bits: 256 rows of at most HD_MAX_PITCH elements);
// a k step moves the uniform base.
// F32: a step is 32 deep in k and two of the three numbers of a value are staged: the first in the first 4 chunks (not TR) or 32
// rows (TR) of the tile, behind it the second (stage 0) or the third (stage 1).
#define HD_MAX_PITCH (1 << 22)
template <int B, bool TR, bool CLAMP, int NW, bool F32>
struct HdLoad {
  static constexpr int DEEP = F32 ? 32 : HD_BK;
  static constexpr int NL = B * HD_BK * 2 / 1024 / NW;
  static constexpr int CH = B / 8, RPL = TR ? 64 / CH : 8;      // TR: chunks per row, rows per load
  static_assert(NL % 2 == 0 && NW % 2 == 0, "which lanes and loads fetch the later number: see issue");
  uint32_t off[NL];
  __device__ __forceinline__ void init(const HdOperand& o, int own0, int wave, int lane) {
#pragma unroll
    for (int q = 0; q < NL; ++q) {
      const int blk = q * NW + wave;
      if constexpr (!TR) {
        const int r = blk * 8 + (lane >> 3);
        const int ch = (lane & 7) ^ ((r & 3) | (((r >> 3) & 1) << 2));
        off[q] = 2u * ((uint32_t)(min(own0 + r, o.rows - 1) - own0) * (uint32_t)o.ld +
                       (F32 ? (ch & 3) * 8 + (ch >> 2) * (uint32_t)o.plane : ch * 8));
      } else {
        const int k = blk * RPL + lane / CH;
        const int g = (k & 3) | (((k >> 3) & 3) << 2);
        const int ch = (lane % CH) ^ ((2 * g) & (CH - 1));
        off[q] = 2u * ((uint32_t)(k % DEEP) * (uint32_t)o.ld + (k / DEEP) * (uint32_t)o.plane + min(own0 + ch * 8, o.cols - 8));
      }
    }
  }
  // first element of the tile at k step 0, and the distance between k steps (bytes)
  static __device__ __forceinline__ const char* start(const HdOperand& o, int own0) {
    return (const char*)(o.p + (TR ? 0 : (int64_t)own0 * o.ld));
  }
  static __device__ __forceinline__ int64_t advance(const HdOperand& o) { return TR ? 2 * DEEP * o.ld : 2 * DEEP; }
  // The load is written out so that the compiler's own waits do not count it: it has no register result, and the kernel
  // waits for it (vmcnt) before the barrier that hands the stage over.  s_nop: the wait states between a scalar register's
  // writer (M0, or a base that came through a vector instruction) and its reader, which the compiler does not see here.
  __device__ __forceinline__ void issue(const HdOperand& o, const char* base, int k0, uint32_t lds, int wave, int lane, bool third) const {
    // F32 with the third number in the second one's place: not TR, the lanes of chunks 4 to 7 (r >> 3 is blk, whose parity is the
    // wave's); TR, the loads of rows 32 to 63
    const char* at = hd_uniform(base);
    const char* at2 = F32 && TR && third ? hd_uniform(base + 2 * o.plane) : at;
    const uint32_t add = F32 && !TR && third && (((lane >> 2) ^ wave) & 1) ? 2u * (uint32_t)o.plane : 0u;
#pragma unroll
    for (int q = 0; q < NL; ++q) {
      const int blk = q * NW + wave;
      uint32_t v = off[q] + add;
      if constexpr (CLAMP) {               // rows of k beyond the last: the last one again
        const int k = (blk * RPL + lane / CH) % DEEP;
        v -= 2u * (uint32_t)max(0, k - (o.rows - 1 - k0)) * (uint32_t)o.ld;
      }
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(lds + blk * 1024)), "v"(v),
                   "s"(q < NL / 2 ? at : at2)
                   : "memory");
    }
  }
};

// Reading a staged tile (swizzled as above) as matrix operands of 16 own indices each.  hd_at: the lane's LDS address for operand
// 0 of a wave whose own indices start at o0 (a multiple of 32, 8 times a power of two above the operands' range).  hd_frag:
// operand x of half kk (of k, or F32: the kk'th numbers of the stage) from it; x and kk are constants, so it is that address with a few
// bits flipped and an offset in the instruction.
// `pairs`: the logits' products take P's rows in another order, operand x holds rows hd_row(x) + 8 (m >> 2) + (m & 3), m < 16,
// so that a lane's results of operands 2 t and 2 t + 1 are 8 consecutive classes of one row: e is stored 16 bytes at a time
__device__ __forceinline__ constexpr int hd_row(int x) { return (x >> 1) * 32 + (x & 1) * 4; }
template <int B, bool TR, bool pairs>
__device__ __forceinline__ uint32_t hd_at(uint32_t tile, int o0, int lane) {
  const int m = lane & 15;
  if constexpr (TR) {
    const int k = 8 * (lane >> 4) + (m >> 2);
    return tile + k * B * 2 + ((((o0 >> 3) | ((lane & 3) >> 1)) ^ ((2 * (lane >> 2)) & (B / 8 - 1))) << 4) + (lane & 1) * 8;
  } else {
    const int r = o0 + (pairs ? 8 * (m >> 2) + (m & 3) : m), f = pairs ? m & 7 : (m & 3) | (((m >> 3) & 1) << 2);
    return tile + r * HD_BK * 2 + (((lane >> 4) ^ f) << 4);
  }
}
template <int B, bool TR, bool pairs>
__device__ __forceinline__ s16x8 hd_frag(uint32_t at, int x, int kk) {
  if constexpr (TR) {
    typedef __attribute__((address_space(3))) s16x4* lp;
    const uint32_t a = (at ^ (x << 5)) + kk * 32 * B * 2;
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)a);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(a + 4 * B * 2));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
    return *(const __attribute__((address_space(3))) s16x8*)((at ^ (kk << 6)) + (pairs ? hd_row(x) : x * 16) * HD_BK * 2);
  }
}

// n <= 4 consecutive results of a row, from any element address
template <class T>
__device__ __forceinline__ void hd_store4(void* out, int64_t at, f32x4 v, int n) {
  T* o = (T*)out + at;
  if (n == 4) {
    RowVec<T, 4> u;
#pragma unroll
    for (int r = 0; r < 4; ++r) u.v[r] = to_t<T>(v[r]);
    *(RowVec<T, 4>*)o = u;
  } else {
    for (int r = 0; r < n; ++r) o[r] = to_t<T>(v[r]);
  }
}

// a barrier for what passed through LDS; loads and stores of global memory stay in flight
__device__ __forceinline__ void hd_lds_barrier() {
  __builtin_amdgcn_s_waitcnt(0xc07f);      // LDS reads and writes done; vmcnt at its maximum
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// what a finished tile of products becomes (see HdArgs)
template <class T, int BI, int BJ, int WI, int WJ, int EPI, bool F32>
__device__ __forceinline__ void hd_epilogue(const HdArgs& a, f32x4 (&acc)[BI / WI / 16][BJ / WJ / 16], int z, int i0, int j0, int ti,
                                            int wi, int wj, int tid, float* sh) {
  constexpr int NW = WI * WJ, MI = BI / WI / 16, MJ = BJ / WJ / 16;
  const int lane = tid & 63, wave = tid >> 6;
  const int q4 = 4 * (lane >> 4), l15 = lane & 15;
  if constexpr (EPI == EPI_OUT) {
    const float s = a.out ? hd_factor<T>(a.S) : 1.f;
#pragma unroll
    for (int y = 0; y < MJ; ++y) {
      const int j = j0 + wj + y * 16 + l15;
      if (j >= a.nj) continue;
#pragma unroll
      for (int x = 0; x < MI; ++x) {
        const int i = i0 + wi + x * 16 + q4;
        const int left = min(4, a.ni - i);
        if (left <= 0) continue;
        f32x4 v = acc[x][y];
        if (a.out) {
          v *= s;
          if (a.dt == DT_F32) hd_store4<float>(a.out, (int64_t)j * a.ldo + i, v, left);
          else if (a.dt == DT_BF16) hd_store4<bf16_t>(a.out, (int64_t)j * a.ldo + i, v, left);
          else hd_store4<f16_t>(a.out, (int64_t)j * a.ldo + i, v, left);
        } else {
          const int64_t at = ((int64_t)z * a.nj + j) * a.ni + i;
          if (a.add) {
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] += r < left ? a.acc[at + r] : 0.f;
          }
          hd_store4<float>(a.acc, at, v, left);
        }
      }
    }
  } else {
    // z = u acc: the product in units of 1 / tau; with a bias, acc becomes z and u one.
    // exp(z - m) = 2^(z k - m k) in one fused step, off by the rounding of the product m k alone, which is the same factor in
    // all of a row and is taken out of its sum.  That rounding is below one only for |m k| < HD_FAR: beyond (a tile whose classes are
    // all masked by a bias of -1e10, or of the type's lowest value) 2^rounding leaves the range, and the difference is formed
    // first.  Classes beyond the last and targets are looked for only where a tile can hold them: 128 results a lane are 128
    // times whatever one costs.
    float u = a.inv_tau;
    if (a.bias) {
#pragma unroll
      for (int x = 0; x < MI; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = i0 + wi + hd_row(x) + 2 * q4 + r;
          const float b = i < a.ni ? load_as(a.bias, a.dt, a.v0 + i) * a.inv_tau : 0.f;
#pragma unroll
          for (int y = 0; y < MJ; ++y) acc[x][y][r] = __fmaf_rn(acc[x][y][r], u, b);
        }
      u = 1.f;
    }
    const bool edge = i0 + BI > a.ni;                            // of the workgroup
    const int first = i0 + wi + 2 * q4, last = a.ni - first;     // this lane's results are classes first + hd_row(x) + r
    auto target_at = [&](int j) -> int {                         // the place of row j's target among them, or -1
      if (!a.target || j >= a.nj) return -1;
      const int64_t t = a.target[j] - a.v0;
      return t >= first && t < a.ni && t < first + 16 * MI ? (int)t - first : -1;
    };
    if constexpr (EPI == EPI_STATS) {
      // (max, sum of exp) over this tile's classes without the target, per row; a row's classes lie in the 4 lane groups of
      // WI waves.  sh: [WI][BJ][2]
#pragma unroll
      for (int y = 0; y < MJ; ++y) {
        const int jl = wj + y * 16 + l15, j = j0 + jl;
        if (edge) {
#pragma unroll
          for (int x = 0; x < MI; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[x][y][r] = hd_row(x) + r >= last ? -INFINITY : acc[x][y][r];
        }
        const int tl = target_at(j);
        if (__any(tl >= 0)) {
          float z = 0.f;
#pragma unroll
          for (int x = 0; x < MI; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              z = tl == hd_row(x) + r ? acc[x][y][r] : z;
              acc[x][y][r] = tl == hd_row(x) + r ? -INFINITY : acc[x][y][r];
            }
          if (tl >= 0 && (tl & 31) < 8) a.zt[j] = z * u;
        }
        float m = -INFINITY, s = 0.f;
#pragma unroll
        for (int x = 0; x < MI; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r) m = fmaxf(m, acc[x][y][r]);
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        const float ms = m == -INFINITY ? 0.f : m, k = u * L2E, mk = ms * k;
        const bool far = !(fabsf(mk) < HD_FAR);                   // the same in a row's four lanes, and no matter of other rows
        if (far) {
#pragma unroll
          for (int x = 0; x < MI; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f((acc[x][y][r] - ms) * k);
        } else {
#pragma unroll
          for (int x = 0; x < MI; ++x)
#pragma unroll
            for (int r = 0; r < 4; ++r) s += __builtin_amdgcn_exp2f(__fmaf_rn(acc[x][y][r], k, -mk));
        }
        s += __shfl_xor(s, 16, 64);
        s += __shfl_xor(s, 32, 64);
        if (!far) s *= __builtin_amdgcn_exp2f(-__fmaf_rn(ms, k, -mk));
        if (lane < 16) {
          sh[((wave % WI) * BJ + jl) * 2] = m * u;
          sh[((wave % WI) * BJ + jl) * 2 + 1] = s;
        }
      }
      hd_lds_barrier();
      for (int jl = tid; jl < BJ; jl += NW * 64) {
        const int j = j0 + jl;
        if (j >= a.nj) continue;
        float m = sh[jl * 2], s = sh[jl * 2 + 1];
        for (int w = 1; w < WI; ++w) {
          const float m2 = sh[(w * BJ + jl) * 2], s2 = sh[(w * BJ + jl) * 2 + 1];
          const float mm = fmaxf(m, m2), ms = mm == -INFINITY ? 0.f : mm;
          s = s * __builtin_amdgcn_exp2f((m - ms) * L2E) + s2 * __builtin_amdgcn_exp2f((m2 - ms) * L2E);
          m = mm;
        }
        a.part[(int64_t)j * a.part_ld + a.part_c0 + ti] = make_float2(m, s);
      }
    } else {
      // e = c (exp(z - m) rs - [target]); zeros in the padding that the next products read, and in rows without a loss
      const float k = u * L2E;
#pragma unroll
      for (int y = 0; y < MJ; ++y) {
        const int j = j0 + wj + y * 16 + l15;
        const bool in = j < a.nj;
        const float keep = __is_same(T, f16_t) ? E_SCALE : 1.f;
        const float c = in ? a.coef[j] * keep : 0.f;
        // exp(z - m) with m = r u + (what the quotient left): 2^(acc k - r k), and what r k left, as in the statistics
        float mk = INFINITY, cp = 0.f, m = 0.f;                  // no loss: exp(0 - inf) = 0, whatever W and the bias hold
        bool far = false;
        if (c == 0.f) {
#pragma unroll
          for (int x = 0; x < MI; ++x) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
        } else {
          m = a.m[j];
          const float r = m / u;
          mk = r * k;
          far = !(fabsf(mk) < HD_FAR);
          cp = c * a.rs[j] * (far ? 1.f : __builtin_amdgcn_exp2f(-__fmaf_rn(r, k, -mk) - __fmaf_rn(-r, u, m) * L2E));
        }
        float ky = k;
        if (far) {                                               // the exponents themselves take the products' place
          ky = 1.f;
          mk = 0.f;
#pragma unroll
          for (int x = 0; x < MI; ++x)
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[x][y][q] = __fmaf_rn(acc[x][y][q], u, -m) * L2E;
        }
        const int tl = target_at(j);
        const bool any = __any(tl >= 0);
        // p - 1 of the target: what the other classes hold, not a difference near 1
        const float et = tl >= 0 && c != 0.f ? c * expm1f(-a.loss[j]) : 0.f;
        if (j >= a.rowsE) continue;
        short* row = a.E + (int64_t)j * (F32 ? 3 : a.eplanes) * a.colsE + first;
#pragma unroll
        for (int x = 0; x < MI; x += 2) {
          float e[8];
#pragma unroll
          for (int r = 0; r < 8; ++r)
            e[r] = cp * __builtin_amdgcn_exp2f(__fmaf_rn(acc[x + (r >> 2)][y][r & 3], ky, -mk));
          if (any) {
#pragma unroll
            for (int r = 0; r < 8; ++r) e[r] = tl == hd_row(x) + r ? et : e[r];
          }
          if (edge) {
            if (first + hd_row(x) >= a.colsE) continue;
#pragma unroll
            for (int r = 0; r < 8; ++r) e[r] = hd_row(x) + r >= last ? 0.f : e[r];
          }
          struct alignas(16) { T t[8]; } h, l;
          if constexpr (F32) {
            decltype(h) m;
#pragma unroll
            for (int r = 0; r < 8; ++r) {
              h.t[r] = to_t<T>(e[r]);                            // |e| <= 1, or no finite number in all three
              const float d = e[r] - (float)h.t[r];
              m.t[r] = to_t<T>(d);
              l.t[r] = to_t<T>(d - (float)m.t[r]);
            }
            *(decltype(h)*)(row + hd_row(x)) = h;
            *(decltype(h)*)(row + a.colsE + hd_row(x)) = m;
            *(decltype(h)*)(row + 2 * a.colsE + hd_row(x)) = l;
            continue;
          }
#pragma unroll
          for (int r = 0; r < 8; ++r) h.t[r] = to_t<T>(e[r]);
          *(decltype(h)*)(row + hd_row(x)) = h;
          if (a.eplanes > 1) {
#pragma unroll
            for (int r = 0; r < 8; ++r) l.t[r] = to_t<T>(e[r] - (float)h.t[r]);
            *(decltype(l)*)(row + a.colsE + hd_row(x)) = l;
          }
        }
      }
    }
  }
}

// out[j, i] = sum_k Q[j, k] P[i, k] on tiles of BI x BJ, WI x WJ waves; the lanes of a matrix result hold 4 consecutive i of
// one j, so rows of the output are written in pieces of 4.
//
// A workgroup walks its tiles as one sequence of k steps.  Two stages are in LDS; a step is four phases (two halves of k, two
// of the wave's i).  F32: 32 of k are two steps, one over the first and second numbers (h h, h m, m h, m m: eight phases), one
// over the first and third (h l, l h: four), so that what is loaded and read from LDS for four multiplies for six.  The
// operands of a phase are read while the phase before it multiplies.  The barrier that ends a step stands before its last
// phase, whose operands are in registers by then: the loads of the step after the next and the
// first reads of the next one are issued under that phase's products.  The sequence runs on into the next tile, so a
// tile's first loads are under way during the last steps and the epilogue of the tile before it.  Behind the last tile the
// loads fetch that tile's first steps again, into stages that are read no more.
// Measured (bf16, 4096 x 2048 x 65536): see hd_shape.  What bounds it: the latency of loads that miss the L2 (one step of
// 64 KB in flight per CU) and the clock, which this load holds near 2.0 GHz.
template <class T, int BI, int BJ, int WI, int WJ, bool PT, bool QT, int EPI, bool F32>
__global__ void __launch_bounds__(WI* WJ * 64, BI == 64 ? 4 : 2) k_head_gemm(HdArgs a) {
  constexpr int NW = WI * WJ, MI = BI / WI / 16, MJ = BJ / WJ / 16, HX = MI / 2;
  constexpr int SZ = hd_tile_shorts<BI>() + hd_tile_shorts<BJ>();
  __shared__ __attribute__((aligned(1024))) short sm[2 * SZ];
  __shared__ float sh[EPI == EPI_STATS ? WI * BJ * 2 : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // An XCD takes a contiguous range of tiles, ordered in bands of 4 tiles along j, so that the tiles in flight on one L2
  // share operand panels along both indices; of split products it takes whole ranges of k, all of whose tiles share panels
  const int n = a.ti * a.tj, xcd = (int)blockIdx.x & 7, slot = (int)blockIdx.x >> 3;
  int id, end, stride, z = 0;
  if (a.splits == 1) {
    const int per = (n + 7) >> 3;
    id = xcd * per + slot;
    end = min(n, (xcd + 1) * per);
    stride = (int)gridDim.x >> 3;
  } else {
    const int w = xcd * ((int)gridDim.x >> 3) + slot;
    z = w / a.wgs;
    id = z < a.splits ? w - z * a.wgs : n;
    end = n;
    stride = a.wgs;
  }
  if (id >= end) return;
  auto place = [&](int t, int& ti, int& tj) __attribute__((always_inline)) {
    const int band = t / (4 * a.ti), bw = min(4, a.tj - band * 4), rem = t - band * 4 * a.ti;
    tj = band * 4 + rem % bw;
    ti = rem / bw;
  };
  const int wi = (wave % WI) * (BI / WI), wj = (wave / WI) * (BJ / WJ);
  const int nseg = F32 ? 1 : a.nseg, total = a.ktiles * nseg;
  const int t0 = (int)((int64_t)total * z / a.splits), t1 = (int)((int64_t)total * (z + 1) / a.splits);

  // only W is read along k where it lies, with rows beyond its last (PT && !QT); e and the copied x are whole k steps
  using LP = HdLoad<BI, PT, PT && !QT, NW, F32>;
  using LQ = HdLoad<BJ, QT, false, NW, F32>;
  LP lp;
  LQ lq;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) short*)sm;
  // The next load: its tile, how many of the tile's are left, the step of k and in it the number of Q's values (a step is read
  // again while the L2 has it), and the operands' bases.  Stages alternate by constants in the code, so an odd count of
  // steps gets one more that repeats the last load and multiplies nothing (F32: two steps to a k, so never).
  const int steps = F32 ? 2 * (t1 - t0) : t1 - t0, pad = F32 ? 0 : steps & 1;
  const int first_k = t0 / nseg, first_seg = t0 - first_k * nseg;
  const int64_t pq = 2 * a.Q.plane, dp = LP::advance(a.P), dq = LQ::advance(a.Q) - (nseg == 2 ? pq : 0);
  int lid = id, left, seg, lk, li0, lj0;
  const char *bp, *bq;
  auto base = [&]() __attribute__((always_inline)) {
    bp = LP::start(a.P, li0) + lk * dp;
    bq = LQ::start(a.Q, lj0) + lk * LQ::advance(a.Q) + (seg == 1 ? pq : 0);
  };
  auto aim = [&]() __attribute__((always_inline)) {
    int ti, tj;
    place(lid, ti, tj);
    li0 = ti * BI;
    lj0 = tj * BJ;
    lp.init(a.P, li0, wave, lane);
    lq.init(a.Q, lj0, wave, lane);
  };
  auto rewind = [&]() __attribute__((always_inline)) {
    left = steps + pad;
    seg = first_seg;
    lk = first_k;
    base();
  };
  auto issue = [&](int stage) __attribute__((always_inline)) {
    lp.issue(a.P, bp, lk * LP::DEEP, lds0 + stage * (SZ * 2), wave, lane, stage == 1);
    lq.issue(a.Q, bq, lk * LQ::DEEP, lds0 + stage * (SZ * 2) + hd_tile_shorts<BI>() * 2, wave, lane, stage == 1);
    if (--left == 0) {
      if (lid + stride < end) {
        lid += stride;
        aim();
      }
      rewind();
    } else if constexpr (F32) {
      if (stage == 1) {
        ++lk;
        bp += dp;
        bq += dq;
      }
    } else if (left > pad) {
      if (++seg == nseg) {
        seg = 0;
        ++lk;
        bp += dp;
        bq += dq;
      } else {
        bq += pq;
      }
    }
  };
  s16x8 fp[2][HX], fq[2][MJ];
  f32x4 acc[MI][MJ];
  // half `kk` of the tiles' depth (F32: the first or the later numbers) of half `hx` of the wave's P, and of its Q, into a buffer each
  // F32: the addresses are formed anew from one register each time.  Kept per operand and stage they would not fit beside both
  // numbers' operands (the empty asm keeps the compiler from doing so), and a spilled one is a load that waits for the tiles'
  // loads (two thirds more time).  Single numbers have the registers, and lose 3 % without them.
  constexpr bool pairs = EPI != EPI_OUT;
  const uint32_t ap = hd_at<BI, PT, pairs>(lds0, wi, lane), aq = hd_at<BJ, QT, false>(lds0 + hd_tile_shorts<BI>() * 2, wj, lane);
  auto read_p = [&](int stage, int kk, int hx) __attribute__((always_inline)) {
    uint32_t at = ap + stage * (SZ * 2);
    if constexpr (F32) asm volatile("" : "+v"(at));
#pragma unroll
    for (int x = 0; x < HX; ++x) fp[hx][x] = hd_frag<BI, PT, pairs>(at, hx * HX + x, kk);
  };
  auto read_q = [&](int stage, int kk, int buf) __attribute__((always_inline)) {
    uint32_t at = aq + stage * (SZ * 2);
    if constexpr (F32) asm volatile("" : "+v"(at));
#pragma unroll
    for (int y = 0; y < MJ; ++y) fq[buf][y] = hd_frag<BJ, QT, false>(at, y, kk);
  };
  auto mul = [&](int hx, int buf) __attribute__((always_inline)) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int x = 0; x < HX; ++x)
#pragma unroll
      for (int y = 0; y < MJ; ++y) acc[hx * HX + x][y] = hd_mfma<T>(fp[hx][x], fq[buf][y], acc[hx * HX + x][y]);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
  };
  // A step's products but for the last group, mul(1, 1), whose operands are read: on `stage`, whose first half of P and of Q is in
  // registers (fp[0], fq[0]).
  auto multiply = [&](int stage) __attribute__((always_inline)) {
    read_p(stage, 0, 1);
    if constexpr (F32) {
      if (stage == 0) {                    // h and m of both
        read_q(0, 1, 1);
        mul(0, 0);                         // h h
        mul(1, 0);
        mul(0, 1);                         // h m
        read_p(0, 1, 0);
        mul(1, 1);
        read_p(0, 1, 1);
        mul(0, 0);                         // m h
        mul(0, 1);                         // m m
        mul(1, 0);
      } else {                             // h and l of both, Q's l read first
        read_q(1, 0, 1);
        mul(0, 0);                         // h l
        read_p(1, 1, 0);
        mul(1, 0);
        read_p(1, 1, 1);
        mul(0, 1);                         // l h
      }
    } else {
      mul(0, 0);
      read_q(stage, 1, 1);
      read_p(stage, 1, 0);
      mul(1, 0);
      read_p(stage, 1, 1);
      mul(0, 1);
    }
  };
  // this wave's loads have landed and its LDS reads are done, and every other wave's
  auto meet = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(7 << 4);
    hd_lds_barrier();
  };
  aim();
  rewind();
  issue(0);
  issue(1);
  meet();
  for (; id < end; id += stride) {
    int ti, tj;
    place(id, ti, tj);
#pragma unroll
    for (int x = 0; x < MI; ++x)
#pragma unroll
      for (int y = 0; y < MJ; ++y) acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Tiles of 64 are for few rows, whose losses nothing averages: their sums are added up every eight steps (1 x 1024 x 32768 in
    // bf16: the loss is off by 1.4e-7 of itself, in one chain by 6e-7).  The larger ones have no registers for a second sum.
    f32x4 sum[BI == 64 ? MI : 1][BI == 64 ? MJ : 1] = {};
    auto collect = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int x = 0; x < MI; ++x)
#pragma unroll
        for (int y = 0; y < MJ; ++y) {
          sum[x][y] += acc[x][y];
          acc[x][y] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    read_q(0, 0, 0);
    read_p(0, 0, 0);
    for (int t = 0; t < steps; t += 2) {
      multiply(0);
      meet();                              // the next step has arrived; this one has been read by all
      issue(0);
      read_q(1, F32 ? 1 : 0, 0);
      read_p(1, 0, 0);
      mul(1, 1);
      // not of an odd count's last step, whose partner is only waited for (F32 has none; without the branch the compiler keeps
      // both steps' addresses and spills 13 to 31 registers, with it at most 7)
      const bool more = t + 1 < steps;
      if (more) multiply(1);
      meet();
      issue(1);
      if (t + 2 < steps) {                 // across the epilogue the registers are the result's
        read_q(0, 0, 0);
        read_p(0, 0, 0);
      }
      if (more) mul(1, 1);
      if constexpr (BI == 64) {
        if ((t & 7) == 6) collect();
      }
    }
    if constexpr (BI == 64) {
      collect();
#pragma unroll
      for (int x = 0; x < MI; ++x)
#pragma unroll
        for (int y = 0; y < MJ; ++y) acc[x][y] = sum[x][y];
    }
    hd_epilogue<T, BI, BJ, WI, WJ, EPI, F32>(a, acc, z, ti * BI, tj * BJ, ti, wi, wj, tid, sh);
  }
  __builtin_amdgcn_s_waitcnt(0);           // nothing is in flight into LDS when it is given back
  __builtin_amdgcn_s_barrier();
}

#include "head_small.h"

// ---- kernels around the products ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ float hd_wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
// the maximum over a workgroup of NW waves, in every thread
template <int NW>
__device__ __forceinline__ float hd_block_max(float m, float* sh) {
  m = hd_wave_max(m);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
  m = 0.f;
#pragma unroll
  for (int w = 0; w < NW; ++w) m = fmaxf(m, sh[w]);
  return m;
}
__device__ __forceinline__ float hd_finite_max(float m, float v) {
  v = fabsf(v);
  return v <= 3.402823466e38f ? fmaxf(m, v) : m;
}
// live is NaN for a row that lists a class that does not exist
__device__ __forceinline__ bool hd_has(int64_t n, const int64_t* target, int64_t ignore, const float* live) {
  return target ? target[n] != ignore : live[n] != 0.f;
}

// What stands before the products, in one launch: the rows' coefficients (backward), and the copies of x and of a piece of W
// where they are not read in place.
struct HdPack {
  const void* src;
  int dt;
  int64_t ld, R;
  int D;
  short* out;                // [orows][numbers][ocols]
  int64_t orows;
  int ocols, blocks;
};
struct HdPrep {
  HdPack x, w;
  int masked;                // rows of x without a loss are copied as zeros
  float* S;
  int coef_blocks;           // HD_COEF rows each
  const float *g, *gm;       // per_row: the rows' gradients and, beyond HD_COEF rows, their partial maxima
  int ngm, per_row;
  const float* count;
  float f;                   // tau for the teacher's loss, else 1
  const int64_t* target;
  int64_t ignore;
  const float* live;
  int N;
  float* coef;
};
#define HD_COEF 2048

// coef[n] (|.| <= 1, 0 for a row without a loss) and the scalar S with coef[n] S = the gradient of row n's logits' loss:
// reductions: coef = 1 or 0, S = g f / count (no finite number: coef takes it);  none: S = a power of two over max |g f|
__device__ __forceinline__ void hd_coef(const HdPrep& a, int b, float* sh) {
  float S = 1.f, all = 1.f;
  if (a.per_row) {
    float m = 0.f;
    if (a.gm) {
      for (int i = threadIdx.x; i < a.ngm; i += 256) m = fmaxf(m, a.gm[i]);
    } else {
      for (int n = threadIdx.x; n < a.N; n += 256)
        if (hd_has(n, a.target, a.ignore, a.live)) m = hd_finite_max(m, a.g[n] * a.f);
    }
    m = hd_block_max<4>(m, sh);
    if (m > 0.f) {
      int e;
      frexpf(m, &e);
      S = ldexpf(1.f, min(max(e, -100), 100));
    }
  } else {
    S = a.g[0] * a.f / (a.count ? *a.count : 1.f);
    if (!(fabsf(S) <= 3.402823466e38f)) {  // the rows', not a factor of everything
      all = S;
      S = 1.f;
    }
  }
  const int end = min(a.N, (b + 1) * HD_COEF);
  for (int n = b * HD_COEF + threadIdx.x; n < end; n += 256)       // a NaN of live is the gradient's too
    a.coef[n] = hd_has(n, a.target, a.ignore, a.live) ? (a.per_row ? a.g[n] * a.f / S : all) * (a.live ? a.live[n] : 1.f) : 0.f;
  if (b == 0 && threadIdx.x == 0) *a.S = S;
}

// out <- rows [0, R) of src (type dt, pitch ld, D columns), zeros elsewhere and in masked rows (their contents, whatever they
// are, take no part in any sum).  f32: three numbers.
__device__ __forceinline__ void hd_pack(const HdPrep& a, const HdPack& j, int b, bool masked) {
  const int oc8 = j.ocols >> 3;
  const int64_t pitch = j.dt == DT_F32 ? 3 * (int64_t)j.ocols : j.ocols;
  const int64_t n = j.orows * oc8;
  for (int64_t u = (int64_t)b * 256 + threadIdx.x; u < n; u += (int64_t)j.blocks * 256) {
    const int64_t r = u / oc8;
    const int c = (int)(u - r * oc8) * 8;
    const bool live = r < j.R && (!masked || hd_has(r, a.target, a.ignore, a.live));
    const int left = live ? min(8, j.D - c) : 0;
    s16x8 h = {0, 0, 0, 0, 0, 0, 0, 0}, m = h, l = h;
    if (j.dt == DT_F32) {
      float f[8];
      const float* p = (const float*)j.src + r * j.ld + c;
      if (left == 8) {
        const RowVec<float, 8> v = *(const RowVec<float, 8>*)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = v.v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = i < left ? p[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const Bf3 n = hd_split(f[i]);
        h[i] = __builtin_bit_cast(short, n.h);
        m[i] = __builtin_bit_cast(short, n.m);
        l[i] = __builtin_bit_cast(short, n.l);
      }
      *(s16x8*)(j.out + r * pitch + j.ocols + c) = m;
      *(s16x8*)(j.out + r * pitch + 2 * j.ocols + c) = l;
    } else {
      const short* p = (const short*)j.src + r * j.ld + c;
      if (left == 8) {
        const RowVec<short, 8> v = *(const RowVec<short, 8>*)p;
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = v.v[i];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = i < left ? p[i] : (short)0;
      }
    }
    *(s16x8*)(j.out + r * pitch + c) = h;
  }
}

__global__ void __launch_bounds__(256) k_head_prep(HdPrep a) {
  __shared__ float sh[4];
  const int b = blockIdx.x, bx = b - a.coef_blocks, bw = bx - a.x.blocks;
  if (bx < 0) hd_coef(a, b, sh);
  else if (bw < 0) hd_pack(a, a.x, bx, a.masked);
  else hd_pack(a, a.w, bw, false);
}

__device__ __forceinline__ float hd_wave_sum(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// the tiles' statistics of one row joined by G lanes (result in their first, `lane` 0): softmax = exp(z - mo) rs, the maximum and the sum
// apart (their lse, rounded at its own size, would shift every probability of the row); with a target the row's loss, 0
// where it is `ignore`, NaN where it is no class or where no class has a finite logit
template <int G>
__device__ __forceinline__ void hd_join_row(const float2* __restrict__ p, int tiles, int64_t V, bool with_target, int64_t tg,
                                            int64_t ignore, const float* zt, int lane, float& mo, float& rs, float& loss) {
  float m = -INFINITY, s = 0.f;
  for (int t = lane; t < tiles; t += G) m = fmaxf(m, p[t].x);
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float ms = m == -INFINITY ? 0.f : m;
  for (int t = lane; t < tiles; t += G) s += p[t].y * __builtin_amdgcn_exp2f((p[t].x - ms) * L2E);
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  mo = loss = 0.f;
  rs = 1.f;
  if (!with_target) {
    mo = m;
    rs = 1.f / s;
    return;
  }
  if (tg == ignore) return;
  if (tg < 0 || tg >= V) {
    mo = rs = loss = NAN;
    return;
  }
  // s exp(m) over the other classes, z the target's logit.  The loss from the others' share, not from a difference of
  // two near numbers, where the target holds almost everything
  const float z = *zt;
  const float M = fmaxf(m, z), Ms = M == -INFINITY ? 0.f : M;
  // no other class is left (s = 0, their maximum -inf): their share is 0, not 0 times exp(0 - z), which overflows below z = -88
  const float so = s == 0.f ? 0.f : s * expf(ms - Ms), st = expf(z - Ms);
  mo = M;
  rs = 1.f / (so + st);
  loss = z >= m ? log1pf(so) : (Ms - z) + logf(so + st);
  if (!(so + st > 0.f)) loss = NAN;        // no class is left, or one is infinite: 0 / 0 and infinity / infinity
}

// G lanes per row
template <int G>
__global__ void __launch_bounds__(256) k_head_join(const float2* __restrict__ part, int tiles, int N, int64_t V,
                                                    const int64_t* __restrict__ target, int64_t ignore,
                                                    const float* __restrict__ zt, float* __restrict__ mo,
                                                    float* __restrict__ rs, float* __restrict__ loss,
                                                    float* __restrict__ rows_out) {
  const int lane = threadIdx.x % G;
  const int64_t n = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (n >= N) return;                      // G lanes together
  float m, r, v;
  hd_join_row<G>(part + n * tiles, tiles, V, true, target[n], ignore, zt + n, lane, m, r, v);
  if (lane == 0) {
    mo[n] = m;
    rs[n] = r;
    loss[n] = v;
    if (rows_out) rows_out[n] = v;
  }
}

// out = sum or mean of the rows' losses, count = how many rows have one (at least 1; one that is NaN is a row like others): a
// fixed tree of additions over the 1024 threads of a workgroup
__device__ __forceinline__ void hd_total(float s, float c, int mean, float* out, float* count, float* sh) {
  s = hd_wave_sum(s);
  c = hd_wave_sum(c);
  if ((threadIdx.x & 63) == 0) {
    sh[threadIdx.x >> 6] = s;
    sh[16 + (threadIdx.x >> 6)] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = c = 0.f;
    for (int w = 0; w < 16; ++w) {
      s += sh[w];
      c += sh[16 + w];
    }
    if (!count) {                          // one of several partial sums
      out[0] = s;
      out[1] = c;
      return;
    }
    c = fmaxf(c, 1.f);
    *out = mean ? s / c : s;
    *count = c;
  }
}
// HD_TOTAL rows a workgroup; with more than one of them the sums (mid) are joined by a launch more.  `pairs`: N of those sums
#define HD_TOTAL 8192
__global__ void __launch_bounds__(1024) k_head_total(const float* __restrict__ loss, const int64_t* __restrict__ target,
                                                      int64_t ignore, const float* __restrict__ live, const float2* __restrict__ pairs,
                                                      int N, int mean, float* __restrict__ out, float* __restrict__ count) {
  __shared__ float sh[32];
  float s = 0.f, c = 0.f;
  const int end = min(N, (int)(blockIdx.x + 1) * HD_TOTAL);
  for (int n = blockIdx.x * HD_TOTAL + threadIdx.x; n < end; n += 1024) {
    s += pairs ? pairs[n].x : loss[n];
    c += pairs ? pairs[n].y : hd_has(n, target, ignore, live) ? 1.f : 0.f;
  }
  hd_total(s, c, mean, out + (count ? 0 : 2 * blockIdx.x), count, sh);
}
// few rows: the join and the total in one workgroup
__global__ void __launch_bounds__(1024) k_head_join_total(const float2* __restrict__ part, int tiles, int N, int64_t V,
                                                           const int64_t* __restrict__ target, int64_t ignore,
                                                           const float* __restrict__ zt, float* __restrict__ mo,
                                                           float* __restrict__ rs, float* __restrict__ loss, int mean,
                                                           float* __restrict__ out,
                                                           float* __restrict__ count) {
  __shared__ float sh[32];
  const int lane = threadIdx.x & 63;
  float s = 0.f, c = 0.f;
  for (int n = threadIdx.x >> 6; n < N; n += 16) {
    float m, r, v;
    hd_join_row<64>(part + (int64_t)n * tiles, tiles, V, true, target[n], ignore, zt + n, lane, m, r, v);
    if (lane == 0) {
      mo[n] = m;
      rs[n] = r;
      loss[n] = v;
      s += v;
      c += target[n] != ignore ? 1.f : 0.f;
    }
  }
  hd_total(s, c, mean, out, count, sh);
}

#define TC_MAX 2048          // a teacher's entries per row (12 bytes of LDS each)

// sum / maximum over the WPR waves of a row, in every one of its threads (`sh`: its WPR floats)
template <int WPR, bool MAX>
__device__ __forceinline__ float hd_row_reduce(float v, float* sh, int wave, int lane) {
  v = MAX ? hd_wave_max(v) : hd_wave_sum(v);
  if constexpr (WPR == 1) return __shfl(v, 0, 64);
  if (lane == 0) sh[wave] = v;
  __syncthreads();
  v = sh[0];
#pragma unroll
  for (int w = 1; w < WPR; ++w) v = MAX ? fmaxf(v, sh[w]) : v + sh[w];
  __syncthreads();
  return v;
}

// teacher: WPR waves per row, the first of which joins the row's statistics.  q [N, K]: the softmax over the row's listed
// classes of t / tau, summed over the entries of the same class, -1 for an absent entry (negative index, or logit -inf);
// z [N, K]: the student's own logits / tau there; loss[n]; live[n] = 1, 0 without entries, NaN with an index that is no
// class.  (t - max) / tau is kept finite, so that a listed logit of the type's lowest value is not an absent entry at any
// tau.  A wave forms four logits at a time: the row of x and four rows of W in 16-byte pieces (N K D elements of W are
// gathered: bound by the caches).
template <class T, int WPR>
__global__ void __launch_bounds__(256) k_head_teacher(const T* __restrict__ x, const T* __restrict__ w, const void* __restrict__ bias,
                                                       int dt, int64_t ldx, int64_t ldw, int D, int64_t V,
                                                       const int64_t* __restrict__ index, const void* __restrict__ tl, int tdt, int K,
                                                       float inv_tau, float tau, const float2* __restrict__ stats, int tiles, int N,
                                                       float* __restrict__ mo, float* __restrict__ rs, float* __restrict__ q,
                                                       float* __restrict__ z, float* __restrict__ loss, float* __restrict__ live,
                                                       float* __restrict__ rows_out) {
  constexpr int N8 = VecLen<T>::n, RPB = 4 / WPR, TPR = 64 * WPR;
  extern __shared__ float dyn[];           // per row: t, then (t - max) / tau [K], q [K], index [K] (-1: absent, V: no class)
  __shared__ float shared[4], own[RPB][2];
  const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) % WPR, slot = (threadIdx.x >> 6) / WPR, tid = wave * 64 + lane;
  const int64_t n = (int64_t)blockIdx.x * RPB + slot;
  if (WPR == 1 && n >= N) return;          // one wave to a row: nothing to meet at
  float *st = dyn + slot * 3 * K, *sq = st + K, *sh = shared + slot * WPR;
  int* si = (int*)(sq + K);
  if (wave == 0) {
    float jm, jr, jl;
    hd_join_row<64>(stats + n * tiles, tiles, V, false, 0, 0, nullptr, lane, jm, jr, jl);
    if (lane == 0) {
      mo[n] = own[slot][0] = jm;
      rs[n] = own[slot][1] = jr;
    }
  }
  float m = -INFINITY;
  for (int k = tid; k < K; k += TPR) {
    const int64_t v = index[n * K + k];
    const float t = v < 0 ? -INFINITY : load_as(tl, tdt, n * K + k);
    si[k] = t == -INFINITY ? -1 : (int)(v < V ? v : V);
    st[k] = t;
    m = fmaxf(m, t);
  }
  m = hd_row_reduce<WPR, true>(m, sh, wave, lane);
  const float ms = m == -INFINITY ? 0.f : m;
  float s = 0.f;
  for (int k = tid; k < K; k += TPR) {
    float d = (st[k] - ms) * inv_tau;
    d = d < -3.402823466e38f ? -3.402823466e38f : d;             // a NaN stays one
    st[k] = d;
    if (si[k] >= 0) s += expf(d);
  }
  s = hd_row_reduce<WPR, false>(s, sh, wave, lane);
  const bool any = s > 0.f || s != s;      // a NaN among the listed logits is not an empty row
  const float ls = any ? logf(s) : 0.f;
  for (int k = tid; k < K; k += TPR) sq[k] = si[k] < 0 ? 0.f : expf(st[k] - ls);
  if constexpr (WPR > 1) __syncthreads();
  else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const float sm = own[slot][0], sl = logf(own[slot][1]);         // the student's log softmax is z - sm + sl
  const T* xr = x + n * ldx;
  float part = 0.f;
  for (int k0 = wave * 4; k0 < K; k0 += 4 * WPR) {
    const T* row[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int v = k0 + e < K ? si[k0 + e] : 0;
      row[e] = w + (int64_t)(v >= 0 && v < V ? v : 0) * ldw;     // what is not there reads class 0, and is not used
    }
    float d[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = lane * N8; c < D; c += 64 * N8) {
      if (c + N8 <= D) {
        const RowVec<T, N8> xv = *(const RowVec<T, N8>*)(xr + c);
        RowVec<T, N8> wv[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) wv[e] = *(const RowVec<T, N8>*)(row[e] + c);
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int i = 0; i < N8; ++i) d[e] = __fmaf_rn((float)xv.v[i], (float)wv[e].v[i], d[e]);
      } else {
        for (int i = c; i < D; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) d[e] = __fmaf_rn((float)xr[i], (float)row[e][i], d[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float dot = hd_wave_sum(d[e]);
      const int k = k0 + e;
      if (lane != 0 || k >= K) continue;
      const int v = si[k];
      float zk = 0.f;
      if (any && v >= 0) {
        zk = v < V ? (bias ? dot + load_as(bias, dt, v) : dot) * inv_tau : NAN;     // no such class: the row says so
        if (sq[k] != 0.f || v >= V) part += sq[k] * (st[k] - ls - (zk - sm + sl));   // 0 log 0 = 0, also where p is 0
      }
      z[n * K + k] = zk;
    }
  }
  // entries of the same class add up: 4 entries a thread at a time against every other (4096 rows of 2048: 5.7 ms, one at a time 8.1)
  for (int k0 = tid; k0 < K; k0 += 4 * TPR) {
    int v[4];
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = k0 + j * TPR < K ? si[k0 + j * TPR] : -1;
    for (int e = 0; e < K; ++e) {
      const int o = si[e];
      const float w1 = sq[e];
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[j] += o == v[j] ? w1 : 0.f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k0 + j * TPR < K) q[n * K + k0 + j * TPR] = v[j] < 0 ? -1.f : sum[j];
  }
  part = hd_row_reduce<WPR, false>(lane == 0 ? part : 0.f, sh, wave, lane);
  if (tid == 0) {
    const float v = tau * tau * part;
    loss[n] = any ? v : 0.f;
    live[n] = !any ? 0.f : v == v ? 1.f : v;
    if (rows_out) rows_out[n] = any ? v : 0.f;
  }
}

// gm[block] = the largest finite |g f| of HD_TOTAL rows' losses
__global__ void __launch_bounds__(1024) k_head_gmax(const float* __restrict__ g, float f, const int64_t* __restrict__ target,
                                                     int64_t ignore, const float* __restrict__ live, int N, float* __restrict__ gm) {
  __shared__ float sh[16];
  float m = 0.f;
  const int end = min(N, (int)(blockIdx.x + 1) * HD_TOTAL);
  for (int n = blockIdx.x * HD_TOTAL + threadIdx.x; n < end; n += 1024)
    if (hd_has(n, target, ignore, live)) m = hd_finite_max(m, g[n] * f);
  m = hd_block_max<16>(m, sh);
  if (threadIdx.x == 0) gm[blockIdx.x] = m;
}

// teacher: the listed classes of this piece get e = c (softmax_k - q_k), from the entry's own logit, over what the
// product's epilogue wrote there.  Entries of the same class hold the same q and z and write the same value.
template <class T>
__global__ void __launch_bounds__(256) k_head_teacher_grad(const int64_t* __restrict__ index, const float* __restrict__ q,
                                                            const float* __restrict__ z, const float* __restrict__ mo,
                                                            const float* __restrict__ rs, const float* __restrict__ coef, int64_t N, int K, int64_t v0,
                                                            int64_t nv, int planes, void* __restrict__ E,
                                                            int64_t colsE) {
  const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (u >= N * K) return;
  const int64_t n = u / K;
  const float qk = q[u], c = coef[n];
  const int64_t v = index[u];
  if (v < v0 || v >= v0 + nv || c == 0.f || qk < 0.f) return;
  const float e = c * (__builtin_amdgcn_exp2f((z[u] - mo[n]) * L2E) * rs[n] - qk);
  T* o = (T*)E + n * planes * colsE + (v - v0);
  if constexpr (sizeof(T) == 4) {
    *o = e;
  } else {
    float s = __is_same(T, f16_t) ? e * E_SCALE : e;
    for (int q = 0; q < planes; ++q) {     // its rounding, and that of what it left
      const T h = to_t<T>(s);
      o[q * colsE] = h;
      s -= (float)h;
    }
  }
}

#define HD_SLICE 128
// column sums of e over slices of HD_SLICE rows: part[slice][colsE].  32 lanes across 256 columns (16 bytes each), 8 row lanes
template <class T>
__global__ void __launch_bounds__(256) k_head_colsum(const short* __restrict__ E, int64_t colsE, int planes, int rows,
                                                      float* __restrict__ part) {
  __shared__ float sh[8][32 * 8 + 4];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.y * 256 + cl * 8;
  float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (c < colsE) {                           // a multiple of 64: a lane's 8 columns are all there
    const int r0 = blockIdx.x * HD_SLICE, r1 = min(rows, r0 + HD_SLICE);
    for (int p = 0; p < planes; ++p) {
#pragma unroll 4
      for (int r = r0 + rl; r < r1; r += 8) {
        struct alignas(16) { T t[8]; } v = *(const decltype(v)*)(E + ((int64_t)r * planes + p) * colsE + c);
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] += (float)v.t[i];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) sh[rl][cl * 8 + i] = s[i];
  __syncthreads();
  const int64_t o = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (o < colsE) {
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < 8; ++q) v += sh[q][threadIdx.x];
    part[(int64_t)blockIdx.x * colsE + o] = v;
  }
}

// out[at0 + i] = factor * sum_s part[s][i] over `slots` partials: in order, or `many` (see hd_sums) by 16 lanes of 16 results, each
// lane every 16th partial, and the lanes in order.  Up to three such sums in one launch.
struct HdSum {
  const float* part;
  int slots;
  int64_t stride, n;
  void* out;
  int64_t at0;
  int many, blocks;
};
struct HdSums {
  HdSum j[3];
  int dt;
  const float* S;            // the factor's (hd_factor); null: factors of 1
};
template <class T>
__global__ void __launch_bounds__(256) k_head_sum(HdSums a) {
  __shared__ float sh[16][17];
  int b = blockIdx.x, k = 0;
  while (k < 2 && b >= a.j[k].blocks) b -= a.j[k++].blocks;
  const HdSum& j = a.j[k];
  const float f = a.S ? hd_factor<T>(a.S) : 1.f;
  if (j.many) {
    const int col = threadIdx.x & 15, sl = threadIdx.x >> 4;
    const int64_t i = (int64_t)b * 16 + col;
    float s = 0.f;
    if (i < j.n) {
#pragma unroll 8
      for (int q = sl; q < j.slots; q += 16) s += j.part[(int64_t)q * j.stride + i];
    }
    sh[sl][col] = s;
    __syncthreads();
    if (sl != 0 || i >= j.n) return;
    s = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) s += sh[q][col];
    store_as(j.out, a.dt, j.at0 + i, s * f);
  } else {
    for (int64_t i = (int64_t)b * 256 + threadIdx.x; i < j.n; i += (int64_t)j.blocks * 256) {
      float s = j.part[i];
#pragma unroll 8
      for (int q = 1; q < j.slots; ++q) s += j.part[(int64_t)q * j.stride + i];
      store_as(j.out, a.dt, j.at0 + i, s * f);
    }
  }
}

// ---- host: tile shapes, pieces and workspace ---------------------------------------------------------------------------------
struct HdShape {
  int b, splits;             // tile edge 64 / 128 / 256
};

// The tile edge and the number of k ranges with the smallest estimated time.  The estimate is fitted to measured launches of
// the product kernel (bf16; us of one k step of 64 with c tiles on a CU, and us of a tile's epilogue that its neighbours do
// not hide):   64: 0.5 alone, 1.1 with five on the CU;   128: 0.8 alone, 1.2 with two;   256: 1.9 (one to a CU)
// us with tiles of 64 / 128 / 256 (and k ranges):
//   logits' statistics, 4096 x 2048 x 65536: 1985 / 1076 / 945 (1.16 PFLOP/s; on another card 892, a library's plain product: 904)
//   8192 x 128 x 65536: 424 / 287 / 231    2048 x 256 x 32768: 82 / 55 / 45    64 x 1024 x 16384: 12 / 15 / 29
//   their gradient e, 4096 x 2048 x 65536: 2372 / 1219 / 1014    2048 x 256 x 32768: 94 / 67 / 55
//   e W, 4096 x 2048 x 65536: 2325 (1) / 1063 (1) / 946 (2)    2048 x 256 x 32768: 57 (16) / 39 (16) / 43 (32)
//   1024 x 128 x 65536: 34 (32) / 32 (32) / 40 (64)    e^T x, 4096 x 2048 x 65536: 2452 / 1214 / 989    2048 x 256 x 32768: 56 / 41 / 61
// F32, 32 of k with six products: 2.4 times a step's time.  us with tiles of 64 / 128 / 256:
//   statistics, 4096 x 1024 x 32000: 2985 / 1469 / 1200 (1.34 PFLOP/s of bf16 products, the copies included)   2048 x 256 x 32768:
//   315 / 205 / 188   1024 x 128 x 65536: 186 / 126 / 117   512 x 512 x 4096: 41 / 48 / 88.  What the estimate takes is within 2 % of
//   the best of every tile and count of ranges tried, in all three products of seven sizes.
// A split product writes its partial results and a second launch adds them (bytes at 4 TB/s and 4 us).
static HdShape hd_shape(int64_t ni, int64_t nj, int64_t ksteps, bool f32, int max_splits) {
  const int cus = dig3d_num_cus();
  HdShape best = {64, 1};
  double tb = 1e30;
  for (int e = 0; e < 3; ++e) {
    const int edge = 64 << e, occ = e == 0 ? 5 : e == 1 ? 2 : 1;
    const int64_t tiles = ((ni + edge - 1) / edge) * ((nj + edge - 1) / edge);
    // powers of two, and the counts that fill the chip once or twice
    for (int q = 0; q < 9; ++q) {
      const int64_t fill = (int64_t)cus * occ * (q - 6) / tiles;
      const int s = q < 7 ? 1 << q : (int)(fill < max_splits ? fill : max_splits);
      if (s < 1 || s > max_splits || (s > 1 && (ksteps / s < 4 || (double)s * ni * nj * 4 > 512e6))) continue;
      const int64_t items = tiles * s, c0 = (items + cus - 1) / cus;
      const int c = (int)(c0 < occ ? c0 : occ);
      const int64_t rounds = (items + (int64_t)cus * c - 1) / ((int64_t)cus * c);
      const double step = (f32 ? 2.4 : 1.0) * (e == 0 ? 0.35 + 0.15 * c : e == 1 ? 0.42 + 0.38 * c : 1.9);
      const double fixed = e == 0 ? 2.0 + 0.5 * c : e == 1 ? 1.5 + 0.8 * c : 6.0;
      double t = (double)rounds * (fixed + (double)((ksteps + s - 1) / s) * step);
      if (s > 1) t += 4.0 + (double)s * ni * nj * 8 / 4e6;
      if (t < tb) {
        tb = t;
        best = {edge, s};
      }
    }
  }
  return best;
}

static inline int64_t up64(int64_t v) { return (v + 63) & ~63ll; }
static inline int64_t al256(int64_t v) { return (v + 255) & ~255ll; }

struct HdPlan {
  bool small;                // head_small.h
  int Dp, eplanes;           // eplanes: numbers of an entry of e
  bool f32;                  // every value is three numbers
  bool dx, dw;               // x / W are read where they are
  int64_t Np, vp, np, ldE;
  HdShape lg, gx, gw;
  int tiles_all;
  // byte offsets into the workspace
  int64_t o_x, o_w, o_part, o_zt, o_coef, o_S, o_E, o_gx, o_gw, o_col, total;
};

// 16-bit rows are used in place when their pitch keeps 16-byte loads aligned and D is whole k steps
static bool hd_direct(int dt, const void* p, int64_t ld, int D) {
  return dt != DT_F32 && D % HD_BK == 0 && ld % 8 == 0 && ld <= HD_MAX_PITCH && ((uintptr_t)p & 15) == 0;
}

// e of one piece, per plane; a piece also bounds the packed part of W.  ms with gradients by pieces of 64 / 128 / 256 / 512 MiB:
// 4096 x 2048 x 131072 bf16 7.71 / 7.40 / 7.43 / 7.32   8192 x 128 x 65536 bf16 1.65 / 1.30 / 1.37 / 1.38: the last-level cache
// returns nothing for it.  A piece is 256 classes at least, whatever its rows take.
#define HD_PIECE_BYTES (512ll << 20)

// Float32 products in place (head_small.h) where copies and launches are what the general path costs, or where few float32 rows meet
// a W that it would copy, at one and a half times its size, before the first product.  us of a replayed graph in place / general, with
// gradients (losses alone).  A training call is five launches in place and eight to ten otherwise, which a host that
// launches them one by one pays with some 15 us: the border is where the GPU loses that much.
//   f32: 32 x 128 x 1195: 38 / 49 (19 / 22)   128 x 128 x 1195: 42 / 52   512 x 128 x 1195: 65 / 57 (19 / 23)   1024 x 128 x 1195: 98 / 66
//        512 x 128 x 4096: 80 / 70 (22 / 25)   256 x 128 x 16384: 91 / 89 (28 / 32)   200 x 256 x 2048: 68 / 63   64 x 256 x 1024: 52 / 58 (26 / 27)
//        64 x 256 x 32768: 112 / 131 (43 / 55)   128 x 512 x 1024: 76 / 73 (32 / 30)   128 x 512 x 2048: 85 / 78   256 x 512 x 1024: 86 / 79
//        8 x 1024 x 1024: 110 / 93 (54 / 39)   64 x 512 x 16384: 115 / 123 (41 / 51)   1 x 1024 x 8192: 133 / 126 (55 / 50)
//        64 x 1024 x 8192: 149 / 142 (57 / 58)   16 x 1024 x 16384: 156 / 211 (54 / 65)   64 x 2048 x 32768: 507 / 796 (139 / 271)
//   16-bit rows read in place by both: 32 x 128 x 1195: 40 / 37   128 x 64 x 300: 38 / 35   32 x 128 x 8192: 43 / 37   512 x 128 x 256: 62 / 38
//   16-bit rows that the general path copies (odd widths or addresses): 32 x 127 x 8192: 47 / 44   14 x 40 x 67126: 66 / 66
//        64 x 127 x 32768: 95 / 77   128 x 127 x 4096: 57 / 43   16 x 255 x 8192: 58 / 48   10 x 214 x 105058: 215 / 142
// A wave joins a row's V / 64 statistics: up to 2^20 classes.
static bool hd_small(bool f32, bool copies, int64_t N, int64_t D, int64_t V) {
  const double work = (double)N * D * V;
  if (V > 1048576) return false;
  if (f32)
    return (N <= 512 && D <= 128 && work <= 268435456.0) || (N <= 128 && D <= 512 && work <= 134217728.0) ||
           (N <= 64 && (D <= 256 || V >= 16384));
  if (N > 128 || D > (copies ? 256 : 128)) return false;
  return work <= (!copies || D > 128 ? 33554432.0 : N <= 64 ? 268435456.0 : 67108864.0);
}

// k steps of a product over `k` values, one operand of `q` numbers each
static int64_t hd_steps(const HdPlan& p, int64_t k, int q) { return p.f32 ? (k + 31) / 32 : (k + 63) / 64 * q; }

// needs: bit 0 gx, bit 1 gw, bit 2 gb; backward = 0: the forward's plan
static HdPlan hd_plan(int dt, int64_t N, int D, int64_t V, bool dx, bool dw, int backward, int needs) {
  HdPlan p;
  memset(&p, 0, sizeof p);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t o = at;
    at += al256(bytes);
    return o;
  };
  p.small = hd_small(dt == DT_F32, !(dx && dw), N, D, V);
  if (p.small) {
    p.vp = V;
    p.np = 1;
    p.ldE = (V + 3) & ~3ll;
    p.tiles_all = (int)((V + 63) / 64);
    if (!backward) {
      p.o_part = take(N * p.tiles_all * 8);
      p.o_zt = take(N * 4);
    } else {
      p.o_coef = take(2 * N * 4);
      p.o_E = take(N * p.ldE * 4);
      p.gx = {64, 1};
      if (needs & 1) {       // about two workgroups per CU, at least four k steps each
        const int64_t tiles = ((D + 63) / 64) * ((N + 63) / 64), steps = (V + SM_BK - 1) / SM_BK;
        while (p.gx.splits < 512 && tiles * p.gx.splits < 2 * dig3d_num_cus() && steps / (2 * p.gx.splits) >= 2) p.gx.splits *= 2;
        if (p.gx.splits > 1) p.o_gx = take(p.gx.splits * N * D * 4);
      }
    }
    p.total = at;
    return p;
  }
  p.f32 = dt == DT_F32;
  const int planes = p.f32 ? 3 : 1;
  // One rounding of e is lost among the roundings of the gradients where many rows add up (2^1/2 of the error of their own);
  // in a few rows it is a common factor of a whole row of gw.  There W is what the products wait for, and e is two numbers;
  // also where the second product costs no more than launches do (512 x 512 x 8192: 15 us of 190)
  p.eplanes = p.f32 ? 3 : N <= 128 || (double)N * D * V <= 2147483648.0 ? 2 : 1;
  p.Dp = (int)up64(D);
  p.dx = dx && !backward;    // the backward masks rows while it copies x (N D elements: nothing beside its products)
  p.dw = dw;
  p.Np = up64(N);
  int64_t most = V;
  if (backward) most = min(most, min(HD_PIECE_BYTES / (p.Np * 2), (int64_t)HD_MAX_PITCH / p.eplanes - 1024));
  if (!p.dw) most = min(most, HD_PIECE_BYTES / ((int64_t)p.Dp * 2 * planes));
  if (most < V) most = max((int64_t)256, most & ~255ll);
  p.np = (V + most - 1) / most;
  p.vp = p.np == 1 ? V : ((V + p.np - 1) / p.np + 255) & ~255ll;
  p.np = (V + p.vp - 1) / p.vp;
  p.ldE = up64(p.vp);
  if (p.ldE * p.eplanes % 1024 == 0) p.ldE += 64;      // rows of e a multiple of 2 KB apart fall on few channels of the caches
  p.lg = hd_shape(p.vp, N, hd_steps(p, p.Dp, 1), p.f32, 1);
  if (!p.dx) p.o_x = take(p.Np * p.Dp * 2 * planes);
  if (!p.dw) p.o_w = take(min(p.vp, V) * p.Dp * 2 * planes);
  if (!backward) {
    p.tiles_all = 0;
    for (int64_t v0 = 0; v0 < V; v0 += p.vp) p.tiles_all += (int)((min(p.vp, V - v0) + p.lg.b - 1) / p.lg.b);
    p.o_part = take(N * p.tiles_all * 8);
    p.o_zt = take(N * 4);
  } else {
    p.o_coef = take(N * 4);
    p.o_S = take(4 + (N + HD_TOTAL - 1) / HD_TOTAL * 4);
    p.o_E = take(p.Np * p.ldE * 2 * p.eplanes);
    if (needs & 1) {
      p.gx = hd_shape(D, N, hd_steps(p, p.vp, p.eplanes), p.f32, 512);
      if (p.np > 1 || p.gx.splits > 1) p.o_gx = take((int64_t)p.gx.splits * N * D * 4);
    }
    if (needs & 2) {
      p.gw = hd_shape(D, p.vp, hd_steps(p, N, p.eplanes), p.f32, 512);
      if (p.gw.splits > 1) p.o_gw = take((int64_t)p.gw.splits * p.vp * D * 4);
    }
    if (needs & 4) p.o_col = take((N + HD_SLICE - 1) / HD_SLICE * p.ldE * 4);
  }
  p.total = at;
  return p;
}

template <class T, bool PT, bool QT, int EPI, bool F32>
static void hd_launch(const HdArgs& a, int b, const dim3& grid, hipStream_t st) {
  if (b == 256) hipLaunchKernelGGL((k_head_gemm<T, 256, 256, 2, 4, PT, QT, EPI, F32>), grid, dim3(512), 0, st, a);
  else if (b == 128) hipLaunchKernelGGL((k_head_gemm<T, 128, 128, 2, 2, PT, QT, EPI, F32>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_head_gemm<T, 64, 64, 2, 2, PT, QT, EPI, F32>), grid, dim3(256), 0, st, a);
}
template <class T, bool PT, bool QT, int EPI>
static void hd_gemm(const HdArgs& a0, const HdShape& sh, bool f32, hipStream_t st) {
  HdArgs a = a0;
  a.ti = (a.ni + sh.b - 1) / sh.b;
  a.tj = (a.nj + sh.b - 1) / sh.b;
  a.splits = sh.splits;
  // as many workgroups as run at once; each walks its tiles
  const int most = dig3d_num_cus() * (sh.b == 256 ? 1 : sh.b == 128 ? 2 : 5);
  a.wgs = min(a.ti * a.tj, max(1, most / sh.splits));
  const dim3 grid((unsigned)(sh.splits == 1 ? min(dig3d_xcd_grid(a.ti * a.tj), (most + 7) & ~7) : (a.wgs * sh.splits + 7) & ~7));
  if constexpr (__is_same(T, bf16_t)) {
    if (f32) return hd_launch<T, PT, QT, EPI, true>(a, sh.b, grid, st);
  }
  hd_launch<T, PT, QT, EPI, false>(a, sh.b, grid, st);
}

static inline unsigned hd_grid(int64_t items, int per) {
  const int64_t b = (items + per - 1) / per, cap = 16ll * dig3d_num_cus();
  return (unsigned)(b < 1 ? 1 : b < cap ? b : cap);
}

// one of a launch's sums.  us in order / by 16 lanes:  2140 results of 64 partials 6.0 / 4.0, 32768 of 16: 5.4 / 4.8; 574 of 32 in
// order 4.1, of 512 by 16 lanes 4.0
static void hd_add_sum(HdSums& a, const float* part, int slots, int64_t stride, int64_t n, void* out, int64_t at0) {
  int k = 0;
  while (a.j[k].blocks) ++k;
  const bool many = slots >= 16 && n <= 65536;
  a.j[k] = {part, slots, stride, n, out, at0, many, many ? (int)((n + 15) / 16) : (int)hd_grid(n, 256)};
}
template <class T>
static int hd_sums(const HdSums& a, hipStream_t st) {
  const int blocks = a.j[0].blocks + a.j[1].blocks + a.j[2].blocks;
  if (!blocks) return DIG3D_OK;
  hipLaunchKernelGGL((k_head_sum<T>), dim3(blocks), dim3(256), 0, st, a);
  DIG3D_CHECK_LAUNCH();
  return DIG3D_OK;
}

static HdPack hd_pack_job(const void* src, int dt, int64_t ld, int64_t R, int D, void* out, int64_t orows, int ocols) {
  return {src, dt, ld, R, D, (short*)out, orows, ocols, (int)hd_grid(orows * (ocols >> 3), 256)};
}
static int hd_prep(const HdPrep& a, hipStream_t st) {
  const int blocks = a.coef_blocks + a.x.blocks + a.w.blocks;
  if (!blocks) return DIG3D_OK;
  hipLaunchKernelGGL(k_head_prep, dim3(blocks), dim3(256), 0, st, a);
  DIG3D_CHECK_LAUNCH();
  return DIG3D_OK;
}

static bool hd_bad(int dt, int N, int D, int V, int64_t ldx, int64_t ldw) {
  // tile counts and the launches' threads (256 a row) stay inside 32 bits
  return dt < 0 || dt > 2 || N <= 0 || D <= 0 || V <= 0 || ldx < D || ldw < D ||
         ((int64_t)N + 63) / 64 * (((int64_t)V + 63) / 64) > (1ll << 30) || N >= (1 << 24) || V > (1 << 28) || D > (1 << 20);
}

static const short* at_bytes(const void* p, int64_t o) { return (const short*)((const char*)p + o); }

// everything the entries share
struct HdCall {
  int dt;
  const void *x, *w, *bias;
  int64_t ldx, ldw;
  int N, D, V;
  const int64_t* target;
  int64_t ignore;
  const int64_t* index;
  const void* teacher;
  int tdt, K;
  float tau;
  int reduction;             // 0 one loss per row, 1 mean, 2 sum
  // kept from the forward for the backward (float[HD_KEEP + 4 N + 2 N K])
  float *count, *m, *rs, *loss, *live, *q, *z;
  hipStream_t st;
};
#define HD_KEEP 8

static void hd_keep(HdCall& c, float* keep) {
  c.count = keep;
  c.m = keep + HD_KEEP;
  c.rs = c.m + c.N;
  c.loss = c.rs + c.N;
  c.live = c.loss + c.N;
  c.q = c.live + c.N;
  c.z = c.q + (int64_t)c.N * c.K;
}

static SmArgs sm_args(const HdCall& c, const HdPlan& p, char* ws) {
  SmArgs a;
  memset(&a, 0, sizeof a);
  a.W = {c.w, c.dt, c.ldw, c.V, c.D, nullptr, -1};
  a.x = {c.x, c.dt, c.ldx, c.N, c.D, nullptr, -1};
  a.bias = c.bias;
  a.dt = c.dt;
  a.N = c.N;
  a.D = c.D;
  a.V = c.V;
  a.inv_tau = 1.0f / c.tau;
  a.f = c.index ? c.tau : 1.f;
  a.target = c.target;
  a.ignore = c.ignore;
  a.live = c.live;
  a.part = (float2*)(ws + p.o_part);
  a.tiles = p.tiles_all;
  a.zt = (float*)(ws + p.o_zt);
  a.m = c.m;
  a.rs = c.rs;
  a.loss = c.loss;
  return a;
}

// the logits' statistics into a.part / a.zt
template <class T>
static int hd_stats(const HdCall& c, const HdPlan& p, char* ws) {
  HdArgs a;
  memset(&a, 0, sizeof a);
  HdPrep prep;
  memset(&prep, 0, sizeof prep);
  const int nums = p.f32 ? 3 : 1;          // numbers of a value
  if (p.dx) a.Q = {(const short*)c.x, c.ldx, 0, c.N, c.D};
  else {
    prep.x = hd_pack_job(c.x, c.dt, c.ldx, c.N, c.D, ws + p.o_x, p.Np, p.Dp);
    a.Q = {at_bytes(ws, p.o_x), (int64_t)p.Dp * nums, p.Dp, c.N, p.Dp};
  }
  a.nj = c.N;
  a.ktiles = (int)hd_steps(p, p.Dp, 1);
  a.nseg = 1;
  a.bias = c.bias;
  a.dt = c.dt;
  a.inv_tau = 1.0f / c.tau;
  a.target = c.target;
  a.part = (float2*)(ws + p.o_part);
  a.part_ld = p.tiles_all;
  a.zt = (float*)(ws + p.o_zt);
  const int esz = c.dt == DT_F32 ? 4 : 2;
  for (int64_t v0 = 0; v0 < c.V; v0 += p.vp) {
    const int nv = (int)min(p.vp, c.V - v0);
    const char* wp = (const char*)c.w + v0 * c.ldw * esz;
    if (p.dw) a.P = {(const short*)wp, c.ldw, 0, nv, c.D};
    else {
      prep.w = hd_pack_job(wp, c.dt, c.ldw, nv, c.D, ws + p.o_w, nv, p.Dp);
      a.P = {at_bytes(ws, p.o_w), (int64_t)p.Dp * nums, p.Dp, nv, p.Dp};
    }
    const int rc = hd_prep(prep, c.st);
    if (rc != DIG3D_OK) return rc;
    prep.x.blocks = 0;                     // once
    a.ni = nv;
    a.v0 = v0;
    a.part_c0 = (int)(v0 / p.lg.b);
    hd_gemm<T, false, false, EPI_STATS>(a, p.lg, p.f32, c.st);
    DIG3D_CHECK_LAUNCH();
  }
  return DIG3D_OK;
}

static int hd_fwd(const HdCall& c, const HdPlan& p, char* ws, float* out) {
  float2* part = (float2*)(ws + p.o_part);
  float* zt = (float*)(ws + p.o_zt);
  if (p.small) {
    hipLaunchKernelGGL((k_head_small_logits<false>), dim3((unsigned)p.tiles_all, (unsigned)((c.N + 63) / 64)), dim3(256), 0, c.st,
                       sm_args(c, p, ws));
    DIG3D_CHECK_LAUNCH();
  } else {
    const int rc = c.dt == DT_F16 ? hd_stats<f16_t>(c, p, ws) : hd_stats<bf16_t>(c, p, ws);
    if (rc != DIG3D_OK) return rc;
  }
  // 64 rows: one workgroup joins them in the time of one more launch (2 us each)
  if (c.target && c.reduction && c.N <= 64) {
    hipLaunchKernelGGL(k_head_join_total, dim3(1), dim3(1024), 0, c.st, part, p.tiles_all, c.N, (int64_t)c.V, c.target, c.ignore, zt,
                       c.m, c.rs, c.loss, c.reduction == 1, out, c.count);
    DIG3D_CHECK_LAUNCH();
    return DIG3D_OK;
  }
  float* rows_out = c.reduction ? nullptr : out;
  if (!c.index) {
    // as many lanes as tiles, several rows of few classes a wave (1000000 x 64 x 16: 24 us, a wave each 284)
#define JOIN_GO(G)                                                                                                                          \
  hipLaunchKernelGGL((k_head_join<G>), dim3((unsigned)(((int64_t)c.N * G + 255) / 256)), dim3(256), 0, c.st, part, p.tiles_all, c.N,         \
                     (int64_t)c.V, c.target, c.ignore, zt, c.m, c.rs, c.loss, rows_out)
    if (p.tiles_all <= 4) JOIN_GO(4);
    else if (p.tiles_all <= 16) JOIN_GO(16);
    else JOIN_GO(64);
#undef JOIN_GO
    DIG3D_CHECK_LAUNCH();
  } else {
    // One wave to a row where there are many rows and the rows of W are short, four otherwise.  us of the forward, one / four:
    // 5000 x 256 x 1000 float32 with 8, 16, 64 entries 59 / 72, 63 / 74, 90 / 102, bfloat16 29 / 38, 34 / 40, 64 / 68;
    // 4096 x 1024 x 32000 with 64: 1394 / 1360, bfloat16 335 / 310; 64 x 128 x 1195 with 16: 28 / 22, bfloat16 29 / 23
    const int wpr = c.K <= 4 || (c.K <= 64 && c.N >= 2048 && c.D <= 512) ? 1 : 4, rpb = 4 / wpr;
    const dim3 g((unsigned)((c.N + rpb - 1) / rpb)), b(256);
    const size_t lds = (size_t)c.K * 12 * rpb;
    const float it = 1.0f / c.tau;
#define TC_GO(T, WPR)                                                                                                                   \
  hipLaunchKernelGGL((k_head_teacher<T, WPR>), g, b, lds, c.st, (const T*)c.x, (const T*)c.w, c.bias, c.dt, c.ldx, c.ldw, c.D,           \
                     (int64_t)c.V, c.index, c.teacher, c.tdt, c.K, it, c.tau, part, p.tiles_all, c.N, c.m, c.rs, c.q, c.z, c.loss,      \
                     c.live, rows_out)
    if (c.dt == DT_F32) { if (wpr == 1) TC_GO(float, 1); else TC_GO(float, 4); }
    else if (c.dt == DT_BF16) { if (wpr == 1) TC_GO(bf16_t, 1); else TC_GO(bf16_t, 4); }
    else { if (wpr == 1) TC_GO(f16_t, 1); else TC_GO(f16_t, 4); }
#undef TC_GO
    DIG3D_CHECK_LAUNCH();
  }
  if (c.reduction) {
    const int blocks = (c.N + HD_TOTAL - 1) / HD_TOTAL;
    float* mid = (float*)part;             // the tiles' statistics have been joined
    hipLaunchKernelGGL(k_head_total, dim3(blocks), dim3(1024), 0, c.st, c.loss, c.target, c.ignore, c.live, (const float2*)nullptr, c.N,
                       c.reduction == 1, blocks > 1 ? mid : out, blocks > 1 ? (float*)nullptr : c.count);
    DIG3D_CHECK_LAUNCH();
    if (blocks > 1) {
      hipLaunchKernelGGL(k_head_total, dim3(1), dim3(1024), 0, c.st, (const float*)nullptr, (const int64_t*)nullptr, (int64_t)0,
                         (const float*)nullptr, (const float2*)mid, blocks, c.reduction == 1, out, c.count);
      DIG3D_CHECK_LAUNCH();
    }
  }
  return DIG3D_OK;
}

template <class T>
static int hd_teacher_grad(const HdCall& c, const float* coef, int64_t v0, int64_t nv, int planes, void* E, int64_t colsE) {
  hipLaunchKernelGGL((k_head_teacher_grad<T>), dim3((unsigned)(((int64_t)c.N * c.K + 255) / 256)), dim3(256), 0, c.st, c.index, c.q,
                     c.z, c.m, c.rs, coef, (int64_t)c.N, c.K, v0, nv, planes, E, colsE);
  DIG3D_CHECK_LAUNCH();
  return DIG3D_OK;
}

static int hd_bwd_small(const HdCall& c, const HdPlan& p, const float* g, void* gx, void* gw, void* gb, char* ws) {
  SmArgs a = sm_args(c, p, ws);
  a.g = g;
  a.count = c.reduction == 1 ? c.count : nullptr;
  a.per_row = c.reduction == 0;
  a.coef = (float*)(ws + p.o_coef);
  a.E = (float*)(ws + p.o_E);
  a.ldE = p.ldE;
  hipLaunchKernelGGL((k_head_small_logits<true>), dim3((unsigned)p.tiles_all, (unsigned)((c.N + 63) / 64)), dim3(256), 0, c.st, a);
  DIG3D_CHECK_LAUNCH();
  if (c.index) {
    const int rc = hd_teacher_grad<float>(c, a.coef + c.N, 0, c.V, 1, a.E, a.ldE);
    if (rc != DIG3D_OK) return rc;
  }
  a.gx = gx;
  a.gw = gw;
  a.gb = gb;
  a.splits = p.gx.splits;
  a.slots = gx && p.gx.splits > 1 ? (float*)(ws + p.o_gx) : nullptr;
  a.gx_tiles = gx ? ((c.D + 63) / 64) * ((c.N + 63) / 64) : 0;
  a.gw_tiles = gw || gb ? ((c.D + (gb ? 1 : 0) + 63) / 64) * ((c.V + 63) / 64) : 0;
  hipLaunchKernelGGL(k_head_small_grads, dim3((unsigned)(a.gx_tiles * a.splits + a.gw_tiles)), dim3(256), 0, c.st, a);
  DIG3D_CHECK_LAUNCH();
  if (a.slots) {
    const int64_t n = (int64_t)c.N * c.D;
    HdSums sums;
    memset(&sums, 0, sizeof sums);
    sums.dt = c.dt;
    hd_add_sum(sums, a.slots, p.gx.splits, n, n, gx, 0);
    return hd_sums<bf16_t>(sums, c.st);
  }
  return DIG3D_OK;
}

template <class T>
static int hd_bwd(const HdCall& c, const HdPlan& p, const float* g, void* gx, void* gw, void* gb, char* ws) {
  float* S = (float*)(ws + p.o_S);         // what the forward kept is read only: several backward passes may use it
  const int nums = p.f32 ? 3 : 1;          // numbers of a value
  HdPrep prep;
  memset(&prep, 0, sizeof prep);
  prep.x = hd_pack_job(c.x, c.dt, c.ldx, c.N, c.D, ws + p.o_x, p.Np, p.Dp);
  prep.masked = 1;
  prep.S = S;
  prep.coef_blocks = (c.N + HD_COEF - 1) / HD_COEF;
  prep.g = g;
  prep.per_row = c.reduction == 0;
  prep.count = c.reduction == 1 ? c.count : nullptr;
  prep.f = c.index ? c.tau : 1.f;
  prep.target = c.target;
  prep.ignore = c.ignore;
  prep.live = c.index ? c.live : nullptr;
  prep.N = c.N;
  prep.coef = (float*)(ws + p.o_coef);
  if (prep.per_row && prep.coef_blocks > 1) {
    float* gm = S + 1;
    prep.gm = gm;
    prep.ngm = (c.N + HD_TOTAL - 1) / HD_TOTAL;
    hipLaunchKernelGGL(k_head_gmax, dim3(prep.ngm), dim3(1024), 0, c.st, g, prep.f, c.target, c.ignore, prep.live, c.N, gm);
    DIG3D_CHECK_LAUNCH();
  }
  short* E = (short*)(ws + p.o_E);
  const HdOperand x = {at_bytes(ws, p.o_x), (int64_t)p.Dp * nums, p.Dp, (int)p.Np, p.Dp};
  const HdOperand e = {E, p.ldE * p.eplanes, p.ldE, (int)p.Np, (int)p.ldE};
  const int esz = c.dt == DT_F32 ? 4 : 2;
  const bool gx_slots = gx && (p.np > 1 || p.gx.splits > 1);
  for (int64_t v0 = 0; v0 < c.V; v0 += p.vp) {
    const int nv = (int)min(p.vp, c.V - v0);
    const char* wsrc = (const char*)c.w + v0 * c.ldw * esz;
    HdOperand W;
    if (p.dw) W = {(const short*)wsrc, c.ldw, 0, nv, c.D};
    else {
      prep.w = hd_pack_job(wsrc, c.dt, c.ldw, nv, c.D, ws + p.o_w, nv, p.Dp);
      W = {at_bytes(ws, p.o_w), (int64_t)p.Dp * nums, p.Dp, nv, p.Dp};
    }
    const int rc = hd_prep(prep, c.st);
    if (rc != DIG3D_OK) return rc;
    prep.x.blocks = prep.coef_blocks = 0;  // once
    HdSums sums;
    memset(&sums, 0, sizeof sums);
    sums.dt = c.dt;
    sums.S = S;
    HdArgs a;
    memset(&a, 0, sizeof a);
    a.P = W;
    a.Q = x;
    a.ni = nv;
    a.nj = c.N;
    a.ktiles = (int)hd_steps(p, p.Dp, 1);
    a.nseg = 1;
    a.bias = c.bias;
    a.dt = c.dt;
    a.inv_tau = 1.0f / c.tau;
    a.v0 = v0;
    a.target = c.target;
    a.m = c.m;
    a.rs = c.rs;
    a.loss = c.loss;
    a.coef = prep.coef;
    a.eplanes = p.eplanes;
    a.E = E;
    a.colsE = p.ldE;
    a.rowsE = (int)p.Np;
    hd_gemm<T, false, false, EPI_GRAD>(a, p.lg, p.f32, c.st);
    DIG3D_CHECK_LAUNCH();
    if (c.index) {
      const int rc = hd_teacher_grad<T>(c, prep.coef, v0, nv, p.eplanes, E, p.ldE);
      if (rc != DIG3D_OK) return rc;
    }
    HdArgs o;
    memset(&o, 0, sizeof o);
    o.nseg = p.f32 ? 1 : p.eplanes;
    o.S = S;
    o.dt = c.dt;
    if (gx) {                              // gx[n, d] += sum_v e[n, v] W[v, d]
      o.P = W;
      o.Q = e;
      o.ni = c.D;
      o.nj = c.N;
      o.ktiles = (int)hd_steps(p, nv, 1);  // no step starts beyond W's last row
      o.acc = gx_slots ? (float*)(ws + p.o_gx) : nullptr;
      o.add = v0 > 0;
      o.out = gx_slots ? nullptr : gx;
      o.ldo = c.D;
      hd_gemm<T, true, false, EPI_OUT>(o, p.gx, p.f32, c.st);
      DIG3D_CHECK_LAUNCH();
    }
    if (gw) {                              // gw[v, d] = sum_n e[n, v] x[n, d]
      const bool slots = p.gw.splits > 1;
      o.P = x;
      o.Q = e;
      o.ni = c.D;
      o.nj = nv;
      o.ktiles = (int)hd_steps(p, c.N, 1);
      o.acc = slots ? (float*)(ws + p.o_gw) : nullptr;
      o.add = 0;
      o.out = slots ? nullptr : (char*)gw + v0 * c.D * esz;
      o.ldo = c.D;
      hd_gemm<T, true, true, EPI_OUT>(o, p.gw, p.f32, c.st);
      DIG3D_CHECK_LAUNCH();
      if (slots) hd_add_sum(sums, (const float*)(ws + p.o_gw), p.gw.splits, (int64_t)nv * c.D, (int64_t)nv * c.D, gw, v0 * c.D);
    }
    if (gb) {
      float* part = (float*)(ws + p.o_col);
      const int slices = (c.N + HD_SLICE - 1) / HD_SLICE;
      hipLaunchKernelGGL((k_head_colsum<T>), dim3((unsigned)slices, (unsigned)((p.ldE + 255) / 256)), dim3(256), 0, c.st, E, p.ldE,
                         p.eplanes, c.N, part);
      DIG3D_CHECK_LAUNCH();
      hd_add_sum(sums, part, slices, p.ldE, nv, gb, v0);
    }
    if (gx_slots && v0 + p.vp >= c.V)
      hd_add_sum(sums, (const float*)(ws + p.o_gx), p.gx.splits, (int64_t)c.N * c.D, (int64_t)c.N * c.D, gx, 0);
    const int rs = hd_sums<T>(sums, c.st);
    if (rs != DIG3D_OK) return rs;
  }
  return DIG3D_OK;
}

// the arguments that both entries take; false: refused
static bool hd_call(HdCall& c, int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                    const int64_t* target, int64_t ignore, const int64_t* index, const void* teacher, int tdtype, int K, float tau,
                    int N, int D, int V, int reduction, float* keep, void* stream) {
  if (hd_bad(dtype, N, D, V, ldx, ldw) || !x || !w || !keep || reduction < 0 || reduction > 2 || !(tau > 0.f)) return false;
  if ((!target) == (!index) || (target && (K != 0 || tau != 1.f))) return false;
  if (index && (!teacher || tdtype < 0 || tdtype > 2 || K <= 0 || K > TC_MAX || (int64_t)N * K > (1ll << 31))) return false;
  c = {dtype, x, w, bias, ldx, ldw, N, D, V, target, ignore, index, teacher, tdtype, K, tau, reduction};
  c.st = (hipStream_t)stream;
  hd_keep(c, keep);
  return true;
}

extern "C" {

int dig3d_head_ws_kib(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, int N, int D, int V, int backward, int needs) {
  if (hd_bad(dtype, N, D, V, ldx, ldw)) return DIG3D_ERR_ARG;
  const HdPlan p = hd_plan(dtype, N, D, V, hd_direct(dtype, x, ldx, D), hd_direct(dtype, w, ldw, D), backward, needs);
  const int64_t kib = (p.total + 1023) / 1024;
  return kib > 2147483647ll ? DIG3D_ERR_ARG : (int)kib;
}

int dig3d_head_fwd(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const int64_t* target,
                   int64_t ignore_index, const int64_t* index, const void* teacher, int tdtype, int K, float tau, int N, int D, int V,
                   int reduction, float* keep, float* out, void* ws, int ws_kib, void* stream) {
  DIG3D_ENTER();
  HdCall c;
  if (!hd_call(c, dtype, x, ldx, w, ldw, bias, target, ignore_index, index, teacher, tdtype, K, tau, N, D, V, reduction, keep, stream) ||
      !out)
    return DIG3D_ERR_ARG;
  const HdPlan p = hd_plan(dtype, N, D, V, hd_direct(dtype, x, ldx, D), hd_direct(dtype, w, ldw, D), 0, 0);
  if (p.total > (int64_t)ws_kib * 1024 || !ws) return DIG3D_ERR_ARG;
  return hd_fwd(c, p, (char*)ws, out);
}

int dig3d_head_bwd(int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const int64_t* target,
                   int64_t ignore_index, const int64_t* index, const void* teacher, int tdtype, int K, float tau, int N, int D, int V,
                   int reduction, const float* keep, const float* g, void* gx, void* gw, void* gb, void* ws, int ws_kib, void* stream) {
  DIG3D_ENTER();
  HdCall c;
  if (!hd_call(c, dtype, x, ldx, w, ldw, bias, target, ignore_index, index, teacher, tdtype, K, tau, N, D, V, reduction,
               const_cast<float*>(keep), stream) || !g)
    return DIG3D_ERR_ARG;
  const int needs = (gx ? 1 : 0) | (gw ? 2 : 0) | (gb ? 4 : 0);
  if (!needs) return DIG3D_OK;
  const HdPlan p = hd_plan(dtype, N, D, V, hd_direct(dtype, x, ldx, D), hd_direct(dtype, w, ldw, D), 1, needs);
  if (p.total > (int64_t)ws_kib * 1024 || !ws) return DIG3D_ERR_ARG;
  if (p.small) return hd_bwd_small(c, p, g, gx, gw, gb, (char*)ws);
  return dtype == DT_F16 ? hd_bwd<f16_t>(c, p, g, gx, gw, gb, (char*)ws) : hd_bwd<bf16_t>(c, p, g, gx, gw, gb, (char*)ws);
}

}  // extern "C"
