// One layer of a network of any shape:  y = act(x W^T + b) + residual,  and its three gradient products
//   zbar = ybar act'(z),   xbar = zbar W,   Wbar = zbar^T x,   bbar = sum_rows zbar.
// float32, float16 and bfloat16 tensors; sums, bias, activation and residual in float32, one rounding to the tensor's type.
//
// All three products are  out[i, j] = sum_r A(i, r) B(j, r)  (nrh_layers.h) on one tiled kernel: a workgroup of four waves owns a
// (64 NI) x (64 NJ) tile of the output and walks the reduction in steps of BK.  An operand's next step travels through registers
// (global loads issued before the products of the current one) into LDS rows of BK values of the reduction, whatever its layout in
// memory - reduction contiguous (ROWS) or tile axis contiguous (COLS: the 8 x V block a thread loads is transposed by indexing its
// registers).  act' is applied on the way: zbar is never stored.
//   * 16-bit types: v_mfma_f32_32x32x16_{f16,bf16}.  zbar = ybar act' is rounded to the type once, as every operand of a 16-bit
//     product is; for NONE and RELU it is exact.
//   * float32: x = x0 + x1 + x2 in three bfloat16 (each the rounded rest of the one before: 24 bits), and the six products x_a w_b
//     with a + b <= 2 on v_mfma_f32_32x32x16_bf16.  What is left out is below 2^-25 of |x w|, under float32's own rounding; six
//     passes at the bf16 rate are 2.6 times the rate of v_mfma_f32_32x32x2_f32.  bfloat16 has float32's exponent range, so nothing
//     is scaled.  Infinities, NaN and values that round up to infinity make the parts NaN: a tile whose sums are not all finite is
//     computed again with v_mfma_f32_32x32x2_f32, so its results are those of float32 arithmetic.
// The MFMA's A role is played by the j operand: a lane then holds 16 values of ONE output row.  Its LDS rows are stored permuted (row
// j = 16 h + 4 q + s of a block of 32 at 8 q + 4 h + s), which makes those 16 values consecutive columns.
// LDS rows are padded by 16 B: 16 lanes reading the same 16-byte column of 16 rows meet 16 different bank groups.
// A small output with a long reduction (every weight gradient) is split over the reduction; float32 partial tiles are joined in a
// fixed order by reduce_kernel, so results do not depend on the order of execution.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "nrh_layers.h"

namespace nrhlin {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef long long ll;

enum Src { ROWS = 0, COLS = 1 };

template <typename T> struct Ty;
template <> struct Ty<float> { static constexpr int BK = 32, PLANES = 3; typedef __bf16 L; typedef bf16x8 L8; };
template <> struct Ty<_Float16> { static constexpr int BK = 64, PLANES = 1; typedef _Float16 L; typedef f16x8 L8; };
template <> struct Ty<__bf16> { static constexpr int BK = 64, PLANES = 1; typedef __bf16 L; typedef bf16x8 L8; };

struct Args {
  const void *ip, *iq, *jp;        // A operand, its act' factor (or null), B operand
  ll ild, iqld, jld;
  ll I, J, R;
  int ivec, iqvec, jvec, ovec;     // rows start on vector boundaries: vector loads / stores allowed
  int mask;                        // the factor is a mask (RELU)
  int TI, TJ, S;                   // tiles, splits of the reduction
  ll chunk;                        // reduction per split, a multiple of BK
  void* out;
  ll ldo;
  const void *bias, *res;
  ll ldr;
  void* dact;
  int act;
  float beta;
  float *part, *part_bias;         // S > 1: [S][I][J] and [S][I] float32
  void* bias_bar;
};

// ---- activation ------------------------------------------------------------------------------------------------------------
// act(z) and act'(z); every exponential has a non-positive argument, so none overflows, and NaN passes through
__device__ __forceinline__ float act_eval(int act, float beta, float z, float& d) {
  if (act == NONE) { d = 1.0f; return z; }
  if (act == RELU) { d = z > 0.0f ? 1.0f : 0.0f; return z < 0.0f ? 0.0f : z; }
  if (act == SOFTPLUS) {
    const float e = expf(-fabsf(beta * z));
    const float s = 1.0f / (1.0f + e);
    d = z > 0.0f ? s : e * s;
    return (z < 0.0f ? 0.0f : z) + log1pf(e) / beta;
  }
  if (act == GELU) {
    const float phi = 0.5f * erfcf(-0.70710678118654752f * z);      // erfc: no cancellation for negative z
    d = phi + z * (0.3989422804014327f * expf(-0.5f * z * z));
    return z * phi;
  }
  const float e = expf(-fabsf(z));
  const float r = 1.0f / (1.0f + e);
  const float s = z < 0.0f ? e * r : r, c = z < 0.0f ? r : e * r;   // sigmoid(z), sigmoid(-z)
  if (act == SIGMOID) { d = s * c; return z != z ? z : s; }
  d = s * (1.0f + z * c);
  return z * s;
}

// ---- staging -----------------------------------------------------------------------------------------------------------------
// One operand's step of the reduction: ROWN tile rows x BK values, held as NC groups of 8 consecutive reduction values per thread.
template <typename T, int SRC, int ROWN> struct Stage {
  static constexpr int BK = Ty<T>::BK, CH = BK / 8, NC = ROWN * CH / 256;
  T v[NC][8];

  static __device__ __forceinline__ int row(int tid, int u) {
    if (SRC == ROWS) return (tid + 256 * u) / CH;
    return CH == 4 ? (tid >> 2) * NC + u : ((tid >> 2) & 31) * NC + u;
  }
  static __device__ __forceinline__ int col(int tid, int u) {
    if (SRC == ROWS) return (tid + 256 * u) % CH;
    return CH == 4 ? (tid & 3) : (tid & 3) + 4 * (tid >> 7);
  }
  // tile rows a0 .. of n, reduction r0 .. of rn; rows past n repeat the last one (never stored), reduction past rn is zero
  __device__ __forceinline__ void load(const T* __restrict__ p, ll ld, ll a0, ll n, ll r0, ll rn, bool vec, int tid) {
    if (SRC == ROWS) {
#pragma unroll
      for (int u = 0; u < NC; ++u) {
        ll a = a0 + row(tid, u);
        a = a < n ? a : n - 1;
        const ll r = r0 + 8 * col(tid, u);
        const T* q = p + a * ld + r;
        if (vec && r + 8 <= rn) {
          if (sizeof(T) == 4) {
            const f32x4 x = *(const f32x4*)q, y = *(const f32x4*)((const float*)q + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) { v[u][e] = (T)x[e]; v[u][4 + e] = (T)y[e]; }
          } else {
            const typename Ty<T>::L8 x = *(const typename Ty<T>::L8*)q;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[u][e] = (T)x[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[u][e] = r + e < rn ? q[e] : (T)0.0f;
        }
      }
    } else {
      const ll a = a0 + row(tid, 0);
      const ll r = r0 + 8 * col(tid, 0);
      typedef T V __attribute__((ext_vector_type(NC > 1 ? NC : 2)));
      if (NC > 1 && vec && a + NC <= n) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (r + e < rn) {
            const V x = *(const V*)(p + (r + e) * ld + a);
#pragma unroll
            for (int u = 0; u < NC; ++u) v[u][e] = x[u];
          } else {
#pragma unroll
            for (int u = 0; u < NC; ++u) v[u][e] = (T)0.0f;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int u = 0; u < NC; ++u) {
            const ll au = a + u < n ? a + u : n - 1;
            v[u][e] = r + e < rn ? p[(r + e) * ld + au] : (T)0.0f;
          }
      }
    }
  }
};

// x -> three bfloat16 parts (PLANES = 3) or itself
template <typename T> __device__ __forceinline__ void put8(const float* x, char* dst, int plane_bytes);
template <> __device__ __forceinline__ void put8<float>(const float* x, char* dst, int plane_bytes) {
  bf16x8 p0, p1, p2;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    p0[e] = (__bf16)x[e];
    const float r1 = x[e] - (float)p0[e];
    p1[e] = (__bf16)r1;
    p2[e] = (__bf16)(r1 - (float)p1[e]);
  }
  *(bf16x8*)dst = p0;
  *(bf16x8*)(dst + plane_bytes) = p1;
  *(bf16x8*)(dst + 2 * plane_bytes) = p2;
}
template <> __device__ __forceinline__ void put8<_Float16>(const float* x, char* dst, int) {
  f16x8 p;
#pragma unroll
  for (int e = 0; e < 8; ++e) p[e] = (_Float16)x[e];
  *(f16x8*)dst = p;
}
template <> __device__ __forceinline__ void put8<__bf16>(const float* x, char* dst, int) {
  bf16x8 p;
#pragma unroll
  for (int e = 0; e < 8; ++e) p[e] = (__bf16)x[e];
  *(bf16x8*)dst = p;
}

__device__ __forceinline__ int perm32(int j) {      // column 16 h + 4 q + s of a block of 32 -> MFMA row 8 q + 4 h + s
  return (j & ~31) | (((j >> 2) & 3) << 3) | (((j >> 4) & 1) << 2) | (j & 3);
}

__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

template <typename T> __device__ __forceinline__ float times_act(float y, T q, int mask) {
  return mask ? ((float)q > 0.0f ? y : 0.0f) : y * (float)q;
}

// bias, activation, residual of one output element; returns y and leaves act' in d
template <typename T>
__device__ __forceinline__ float finish(const Args& a, ll i, ll j, float z, float& d) {
  if (a.bias) z += (float)((const T*)a.bias)[j];
  float y = act_eval(a.act, a.beta, z, d);
  if (a.res) y += (float)((const T*)a.res)[i * a.ldr + j];
  return y;
}

template <typename T, int OP, int NI, int NJ>
__global__ __launch_bounds__(256, 2) void tile_kernel(const Args a) {
  constexpr int SI = OP == BACK_WEIGHT ? COLS : ROWS, SJ = OP == FORWARD ? ROWS : COLS;
  constexpr int BK = Ty<T>::BK, PL = Ty<T>::PLANES, BI = 64 * NI, BJ = 64 * NJ;
  constexpr int PITCH = BK * 2 + 16, PLANE = (BI + BJ) * PITCH;
  constexpr int EPITCH = 32 * NJ + 4, EPI = 4 * 32 * EPITCH * 4;
  constexpr int EXACT = PL == 3 ? (BI + BJ) * (BK + 1) * 4 : 0;
  constexpr int LDS = PL * PLANE > EPI ? (PL * PLANE > EXACT ? PL * PLANE : EXACT) : (EPI > EXACT ? EPI : EXACT);
  typedef typename Ty<T>::L8 L8;
  __shared__ __align__(16) char lds[LDS];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // consecutive tiles (same A rows) go to one XCD: workgroups are dealt to the 8 XCDs in turn, and each has its own L2
  const unsigned total = gridDim.x, per = total / 8, rem = total % 8, xcd = blockIdx.x % 8;
  unsigned t = xcd * per + (xcd < rem ? xcd : rem) + blockIdx.x / 8;
  const int tj = t % a.TJ;
  t /= a.TJ;
  const int ti = t % a.TI, s = t / a.TI;
  const ll i0 = (ll)ti * BI, j0 = (ll)tj * BJ;
  const ll rbeg = s * a.chunk, rend = rbeg + a.chunk < a.R ? rbeg + a.chunk : a.R;

  const T* ip = (const T*)a.ip;
  const T* iq = (const T*)a.iq;
  const T* jp = (const T*)a.jp;
  Stage<T, SI, BI> si, sq;
  Stage<T, SJ, BJ> sj;
  const bool scaled = OP != FORWARD && iq != nullptr;
  const bool sums = OP == BACK_WEIGHT && a.bias_bar && tj == 0;
  float bs[Stage<T, SI, BI>::NC] = {};

  const int wi = wave >> 1, wj = wave & 1;
  f32x16 acc[NI][NJ] = {};
  auto fill = [&](ll r) {
    si.load(ip, a.ild, i0, a.I, r, rend, a.ivec, tid);
    if (scaled) sq.load(iq, a.iqld, i0, a.I, r, rend, a.iqvec, tid);
    sj.load(jp, a.jld, j0, a.J, r, rend, a.jvec, tid);
  };
  fill(rbeg);
  for (ll r = rbeg; r < rend; r += BK) {
    __syncthreads();
#pragma unroll
    for (int u = 0; u < si.NC; ++u) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = scaled ? times_act((float)si.v[u][e], sq.v[u][e], a.mask) : (float)si.v[u][e];
      if (sums) {
#pragma unroll
        for (int e = 0; e < 8; ++e) bs[u] += x[e];
      }
      put8<T>(x, lds + si.row(tid, u) * PITCH + si.col(tid, u) * 16, PLANE);
    }
#pragma unroll
    for (int u = 0; u < sj.NC; ++u) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)sj.v[u][e];
      put8<T>(x, lds + (BI + perm32(sj.row(tid, u))) * PITCH + sj.col(tid, u) * 16, PLANE);
    }
    __syncthreads();
    if (r + BK < rend) fill(r + BK);
#pragma unroll
    for (int kk = 0; kk < BK / 16; ++kk) {
      L8 fi[NI][PL], fj[NJ][PL];
      const int off = (2 * kk + (lane >> 5)) * 16;
#pragma unroll
      for (int p = 0; p < PL; ++p) {
#pragma unroll
        for (int b = 0; b < NI; ++b) fi[b][p] = *(const L8*)(lds + p * PLANE + ((wi * NI + b) * 32 + (lane & 31)) * PITCH + off);
#pragma unroll
        for (int b = 0; b < NJ; ++b) fj[b][p] = *(const L8*)(lds + p * PLANE + (BI + (wj * NJ + b) * 32 + (lane & 31)) * PITCH + off);
      }
#pragma unroll
      for (int sum = PL - 1; sum >= 0; --sum)          // the small products first
#pragma unroll
        for (int p = sum; p >= 0; --p)
#pragma unroll
          for (int bi = 0; bi < NI; ++bi)
#pragma unroll
            for (int bj = 0; bj < NJ; ++bj) acc[bi][bj] = mfma(fj[bj][p], fi[bi][sum - p], acc[bi][bj]);
    }
  }

  if (PL == 3) {
    int bad = 0;
#pragma unroll
    for (int bi = 0; bi < NI; ++bi)
#pragma unroll
      for (int bj = 0; bj < NJ; ++bj)
#pragma unroll
        for (int e = 0; e < 16; ++e) bad |= !(fabsf(acc[bi][bj][e]) < __builtin_huge_valf());
    if (__syncthreads_or(bad)) {                       // float32 products: rows of BK + 1 floats, two values of the reduction per MFMA
      float* fl = (float*)lds;
#pragma unroll
      for (int bi = 0; bi < NI; ++bi)
#pragma unroll
        for (int bj = 0; bj < NJ; ++bj) acc[bi][bj] = f32x16{};
      for (ll r = rbeg; r < rend; r += BK) {
        __syncthreads();
        for (int q = tid; q < (BI + BJ) * BK; q += 256) {
          const int rr = q % BK, row = q / BK;
          const ll rg = r + rr;
          float x = 0.0f;
          if (rg < rend) {
            if (row < BI) {
              ll i = i0 + row;
              i = i < a.I ? i : a.I - 1;
              x = (float)ip[SI == ROWS ? i * a.ild + rg : rg * a.ild + i];
              if (scaled) x = times_act(x, iq[SI == ROWS ? i * a.iqld + rg : rg * a.iqld + i], a.mask);
            } else {
              ll j = j0 + row - BI;
              j = j < a.J ? j : a.J - 1;
              x = (float)jp[SJ == ROWS ? j * a.jld + rg : rg * a.jld + j];
            }
          }
          fl[(row < BI ? row : BI + perm32(row - BI)) * (BK + 1) + rr] = x;
        }
        __syncthreads();
        for (int kk = 0; kk < BK; kk += 2) {
          float fi[NI], fj[NJ];
#pragma unroll
          for (int b = 0; b < NI; ++b) fi[b] = fl[((wi * NI + b) * 32 + (lane & 31)) * (BK + 1) + kk + (lane >> 5)];
#pragma unroll
          for (int b = 0; b < NJ; ++b) fj[b] = fl[(BI + (wj * NJ + b) * 32 + (lane & 31)) * (BK + 1) + kk + (lane >> 5)];
#pragma unroll
          for (int bi = 0; bi < NI; ++bi)
#pragma unroll
            for (int bj = 0; bj < NJ; ++bj) acc[bi][bj] = __builtin_amdgcn_mfma_f32_32x32x2f32(fj[bj], fi[bi], acc[bi][bj], 0, 0, 0);
        }
      }
    }
  }

  // the tile leaves through LDS, 32 rows of a wave at a time: a lane then finishes 4 consecutive columns and rows are stored whole
  float* ep = (float*)lds + wave * 32 * EPITCH;
  T* out = (T*)a.out;
#pragma unroll
  for (int bi = 0; bi < NI; ++bi) {
    __syncthreads();
#pragma unroll
    for (int bj = 0; bj < NJ; ++bj)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = acc[bi][bj][4 * q + e];
        *(f32x4*)(ep + (lane & 31) * EPITCH + bj * 32 + 16 * (lane >> 5) + 4 * q) = x;
      }
    __syncthreads();
    constexpr int LPR = 8 * NJ;                        // lanes per row
    for (int it = 0; it < 32 * LPR / 64; ++it) {
      const int row = it * (64 / LPR) + lane / LPR, cc = 4 * (lane % LPR);
      const ll i = i0 + (wi * NI + bi) * 32 + row, j = j0 + wj * NJ * 32 + cc;
      if (i >= a.I || j >= a.J) continue;
      const f32x4 z = *(const f32x4*)(ep + row * EPITCH + cc);
      if (a.part) {
        float* o = a.part + (s * a.I + i) * a.J + j;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j + e < a.J) o[e] = z[e];
        continue;
      }
      typedef T T4 __attribute__((ext_vector_type(4)));
      T4 y4, d4;
      if (OP == FORWARD) {
        T4 r4 = {};
        const bool whole = a.ovec && j + 4 <= a.J;
        if (a.res && whole) r4 = *(const T4*)((const T*)a.res + i * a.ldr + j);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (j + e >= a.J) break;
          float d, x = z[e];
          if (a.bias) x += (float)((const T*)a.bias)[j + e];
          float y = act_eval(a.act, a.beta, x, d);
          if (a.res) y += whole ? (float)r4[e] : (float)((const T*)a.res)[i * a.ldr + j + e];
          y4[e] = (T)y;
          d4[e] = (T)d;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) y4[e] = (T)z[e];
      }
      if (a.ovec && j + 4 <= a.J) {
        *(T4*)(out + i * a.ldo + j) = y4;
        if (OP == FORWARD && a.dact) *(T4*)((T*)a.dact + i * a.J + j) = d4;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (j + e >= a.J) break;
          out[i * a.ldo + j + e] = y4[e];
          if (OP == FORWARD && a.dact) ((T*)a.dact)[i * a.J + j + e] = d4[e];
        }
      }
    }
  }

  if (sums) {                                          // bbar: the CH threads that share a column
    constexpr int NC = Stage<T, SI, BI>::NC, CH = BK / 8;
    float* fl = (float*)lds;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < NC; ++u) fl[si.col(tid, u) * BI + si.row(tid, u)] = bs[u];
    __syncthreads();
    if (tid < BI && i0 + tid < a.I) {
      float x = 0.0f;
      for (int c = 0; c < CH; ++c) x += fl[c * BI + tid];
      if (a.part) a.part_bias[s * a.I + i0 + tid] = x;
      else ((T*)a.bias_bar)[i0 + tid] = (T)x;
    }
  }
}

// joins the S partial outputs in order and finishes them like the tile kernel
template <typename T, int OP>
__global__ __launch_bounds__(256) void reduce_kernel(const Args a) {
  const ll n = a.I * a.J, extra = OP == BACK_WEIGHT && a.bias_bar ? a.I : 0;
  const ll e = (ll)blockIdx.x * 256 + threadIdx.x;
  if (e >= n + extra) return;
  const float* p = e < n ? a.part + e : a.part_bias + (e - n);
  const ll step = e < n ? n : a.I;
  float z = 0.0f;
#pragma unroll 4
  for (int s = 0; s < a.S; ++s) z += p[s * step];
  if (e >= n) {
    ((T*)a.bias_bar)[e - n] = (T)z;
    return;
  }
  const ll i = e / a.J, j = e % a.J;
  float d = 0.0f;
  if (OP == FORWARD) z = finish<T>(a, i, j, z, d);
  ((T*)a.out)[i * a.ldo + j] = (T)z;
  if (OP == FORWARD && a.dact) ((T*)a.dact)[e] = (T)d;
}

// ---- host --------------------------------------------------------------------------------------------------------------------
struct Plan {
  int tile, S;
  ll TI, TJ, chunk;
};

// Which tile and how many splits of the reduction: 256 CUs want at least one workgroup each.
static Plan plan(int dtype, ll I, ll J, ll R) {
  const int BK = dtype == F32 ? 32 : 64;
  auto tiles = [&](int t) { return ((I + t - 1) / t) * ((J + t - 1) / t); };
  Plan p;
  p.tile = tiles(128) >= 192 || (I >= 128 && J >= 128 && R >= 8192) ? 128 : 64;
  const ll n = tiles(p.tile) < 1 ? 1 : tiles(p.tile);
  ll s = n >= 256 ? 1 : 512 / n, most = R / (4 * BK);
  s = s < most ? s : most;
  s = s < 1 ? 1 : (s > 512 ? 512 : s);
  p.chunk = ((R + s - 1) / s + BK - 1) / BK * BK;
  if (p.chunk < BK) p.chunk = BK;                       // R = 0: the gradient of no rows, one pass over nothing
  p.S = (int)((R + p.chunk - 1) / p.chunk);
  if (p.S < 1) p.S = 1;
  p.TI = (I + p.tile - 1) / p.tile;
  p.TJ = (J + p.tile - 1) / p.tile;
  return p;
}

static void shape(int op, ll m, ll n, ll k, ll& I, ll& J, ll& R) {
  I = op == BACK_WEIGHT ? n : m;
  J = op == FORWARD ? n : k;
  R = op == FORWARD ? k : (op == BACK_DATA ? n : m);
}

long long workspace_bytes(int op, int dtype, long long m, long long n, long long k) {
  ll I, J, R;
  shape(op, m, n, k, I, J, R);
  const Plan p = plan(dtype, I, J, R);
  return p.S == 1 ? 0 : 4 * (ll)p.S * (I * J + (op == BACK_WEIGHT ? I : 0));
}

template <typename T, int OP>
static int run(const Call& c, hipStream_t st) {
  Args a = {};
  shape(OP, c.m, c.n, c.k, a.I, a.J, a.R);
  const Plan p = plan(c.dtype, a.I, a.J, a.R);
  const ll need = workspace_bytes(OP, c.dtype, c.m, c.n, c.k);
  if (need > 0 && (!c.ws || c.ws_bytes < need)) return -3;
  const int es = (int)sizeof(T);
  // 16-byte loads of 8 reduction values (two for float32); the transposing loads are narrower
  auto aligned = [&](const void* q, ll ld, int bytes) { return q && ((uintptr_t)q % bytes) == 0 && (ld * es) % bytes == 0 ? 1 : 0; };
  a.ip = OP == FORWARD ? c.x : c.ybar;
  a.ild = OP == FORWARD ? c.ldx : c.ldyb;
  a.iq = OP == FORWARD ? nullptr : c.dact;
  a.iqld = c.ldd;
  a.jp = OP == BACK_WEIGHT ? c.x : c.w;
  a.jld = OP == BACK_WEIGHT ? c.ldx : c.ldw;
  a.ivec = aligned(a.ip, a.ild, 16);
  a.iqvec = aligned(a.iq, a.iqld, 16);
  a.jvec = aligned(a.jp, a.jld, 16);
  a.mask = c.act == RELU;
  a.TI = (int)p.TI;
  a.TJ = (int)p.TJ;
  a.S = p.S;
  a.chunk = p.chunk;
  a.out = c.out;
  a.ldo = c.ldo;
  a.bias = c.bias;
  a.res = c.res;
  a.ldr = c.ldr;
  a.dact = c.dact_out;
  a.act = c.act;
  a.beta = c.beta;
  a.bias_bar = c.bias_bar;
  a.ovec = aligned(a.out, a.ldo, 4 * es) && (!a.res || aligned(a.res, a.ldr, 4 * es)) && (!a.dact || aligned(a.dact, a.J, 4 * es));
  if (p.S > 1) {
    a.part = (float*)c.ws;
    a.part_bias = a.part + (ll)p.S * a.I * a.J;
  }
  const dim3 grid((unsigned)(p.TI * p.TJ * p.S));
  if (p.tile == 128) tile_kernel<T, OP, 2, 2><<<grid, 256, 0, st>>>(a);
  else tile_kernel<T, OP, 1, 1><<<grid, 256, 0, st>>>(a);
  if (p.S > 1) {
    const ll n = a.I * a.J + (a.bias_bar ? a.I : 0);
    reduce_kernel<T, OP><<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>(a);
  }
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

template <typename T> static int run_op(const Call& c, hipStream_t st) {
  if (c.op == FORWARD) return run<T, FORWARD>(c, st);
  if (c.op == BACK_DATA) return run<T, BACK_DATA>(c, st);
  return run<T, BACK_WEIGHT>(c, st);
}

int launch(const Call& c, hipStream_t st) {
  if (c.dtype == F32) return run_op<float>(c, st);
  if (c.dtype == F16) return run_op<_Float16>(c, st);
  return run_op<__bf16>(c, st);
}

}  // namespace nrhlin
