// One layer of a network of any shape:  y = act(x W^T + b) + residual,  and its three gradient products
//   zbar = ybar act'(z),   xbar = zbar W,   Wbar = zbar^T x,   bbar = sum_rows zbar.
// float32, float16 and bfloat16 tensors; sums, bias, activation and residual in float32, one rounding to the tensor's type.
//
// All three products are  out[i, j] = sum_r A(i, r) B(j, r)  (nrh_layers.h) on one tiled kernel: a workgroup of WI x WJ waves owns a
// (32 NI WI) x (32 NJ WJ) tile of the output and walks the reduction in steps of BK, double-buffered in LDS.  The next step travels
// through registers: loaded one step ahead, written to LDS beside the products of the current step, one barrier per step.
// A chunk is 8 consecutive elements of a row in memory, whichever way the row runs:
//   * ROWS (reduction contiguous): LDS rows of BK values per tile row; a lane's MFMA operand - 8 values of the reduction - is one
//     ds_read_b128.
//   * COLS (tile axis contiguous): LDS rows of the tile axis per value of the reduction; the operand is two ds_read_b64_tr_b16, which
//     transpose 4 x 16 blocks on the way to the registers.
// Both are swizzled by 16- or 64-byte groups so that neither the writes nor the reads of a wave meet in a bank.
// act' is applied on the way to LDS: zbar is never stored.
//   * 16-bit types: v_mfma_f32_32x32x16_{f16,bf16}.  zbar = ybar act' is rounded to the type once, as every operand of a 16-bit
//     product is; for NONE and RELU it is exact.  act' itself is kept wider than the type (float32 beside float16, float16 beside
//     bfloat16: 11 bits against 8), so that this one rounding is the only one.
//   * float32: x = x0 + x1 + x2 in three bfloat16 (each the rounded rest of the one before: 24 bits), and the six products x_a w_b
//     with a + b <= 2 on v_mfma_f32_32x32x16_bf16.  What is left out is below 2^-25 of |x w|, under float32's own rounding; six
//     passes at the bf16 rate are 2.6 times the rate of v_mfma_f32_32x32x2_f32.  bfloat16 has float32's exponent range, so nothing
//     is scaled.  Infinities, NaN and values that round up to infinity make the parts NaN: a tile whose sums are not all finite is
//     computed again with v_mfma_f32_32x32x2_f32, so its results are those of float32 arithmetic.
// The MFMA's A role is played by the j operand, its rows permuted (column j = 16 h + 4 q + s of a block of 32 is MFMA row
// 8 q + 4 h + s): a lane then holds 16 consecutive columns of ONE output row.
// A small output with a long reduction (every weight gradient) is split over the reduction; float32 partial tiles are joined in a
// fixed order by reduce_kernel, so results do not depend on the order of execution.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "nrh_layers.h"

namespace nrhlin {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef long long ll;

enum Src { ROWS = 0, COLS = 1 };
enum Deriv { PLAIN = 0, SMOOTH = 1, MASK = 2 };      // A as it is, times act', or kept where act' > 0 (RELU)

template <typename T> struct Ty;                    // BK, planes, LDS element, type act' is kept in
template <> struct Ty<float> { static constexpr int BK = 32, PLANES = 3; typedef __bf16 L; typedef bf16x8 L8; typedef float D; };
template <> struct Ty<_Float16> { static constexpr int BK = 64, PLANES = 1; typedef _Float16 L; typedef f16x8 L8; typedef float D; };
template <> struct Ty<__bf16> { static constexpr int BK = 64, PLANES = 1; typedef __bf16 L; typedef bf16x8 L8; typedef _Float16 D; };

template <bool C, typename A, typename B> struct Pick { typedef A type; };
template <typename A, typename B> struct Pick<false, A, B> { typedef B type; };

// 8 consecutive elements from any element-aligned address (global memory takes unaligned vector loads), as 32-bit words
template <typename X> struct Chunk {
  static constexpr int W = 2 * sizeof(X);
  uint32_t w[W];
  __device__ __forceinline__ void load(const X* p) {
    typedef uint32_t V2 __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t V4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef typename Pick<sizeof(X) == 4, V4, V2>::type V;
#pragma unroll
    for (int h = 0; h < W; h += 4) {
      const V x = *(const V*)((const uint32_t*)p + h);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[h + e] = x[e];
    }
  }
  __device__ __forceinline__ void load_16(const X* p) {      // 16 bytes: 8 elements of 16 bits, 4 of 32
    typedef uint32_t V2 __attribute__((ext_vector_type(4), aligned(2)));
    typedef uint32_t V4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef typename Pick<sizeof(X) == 4, V4, V2>::type V;
    const V x = *(const V*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = x[e];
#pragma unroll
    for (int e = 4; e < W; ++e) w[e] = 0;
  }
  // the 8 elements behind p moved down by k (0 .. 8): p + k .. and zeros
  __device__ __forceinline__ void drop(int k) {
    constexpr int PER = 4 / sizeof(X);                 // elements per word
#pragma unroll
    for (int step = 8; step >= PER; step /= 2) {
      const bool on = (k & step) != 0;
      const int by = step / PER;
#pragma unroll
      for (int e = 0; e < W; ++e) w[e] = on ? (e + by < W ? w[e + by] : 0u) : w[e];
    }
    if (PER == 2) {
      const bool on = (k & 1) != 0;
#pragma unroll
      for (int e = 0; e < W; ++e) w[e] = on ? (w[e] >> 16 | (e + 1 < W ? w[e + 1] << 16 : 0u)) : w[e];
    }
  }
  // the same one by one, for tensors too small to hold 8 elements before the end
  __device__ __forceinline__ void load_single(const X* p, ll n) {
#pragma unroll
    for (int e = 0; e < W; ++e) w[e] = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) {
        if (sizeof(X) == 4) w[e % W] = ((const uint32_t*)p)[e];
        else w[(e / 2) % W] |= (uint32_t)((const uint16_t*)p)[e] << (16 * (e & 1));
      }
  }
  __device__ __forceinline__ void floats(float* x) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (sizeof(X) == 4) x[e] = __builtin_bit_cast(float, w[e]);
      else {
        typedef X X2 __attribute__((ext_vector_type(2)));
        x[e] = (float)__builtin_bit_cast(X2, w[(e / 2) % W])[e & 1];
      }
    }
  }
};

// two floats -> two 16-bit values in a word, round to nearest even (one v_cvt_pk)
template <typename L> __device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float F2 __attribute__((ext_vector_type(2)));
  typedef L L2 __attribute__((ext_vector_type(2)));
  const F2 x = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(x, L2));
}

struct Args {
  const void *ip, *iq, *jp;        // A operand, its act' (or null), B operand
  ll ild, iqld, jld;
  ll I, J, R;
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
// e^-a for a >= 0 on v_exp_f32 (2^x, 1 ulp), the argument a log2(e) in two parts: relative error 2^-23 up to a = 87, 0 beyond 150
__device__ __forceinline__ float exp_minus(float a) {
  a = fminf(a, 150.0f);
  const float h = a * 1.44269502f;
  const float l = fmaf(a, 1.92596299e-8f, fmaf(a, 1.44269502f, -h));
  return __builtin_amdgcn_exp2f(-h) * fmaf(l, -0.693147182f, 1.0f);
}

// act(z) and act'(z); every exponential has a non-positive argument, so none overflows, and NaN passes through
__device__ __forceinline__ float act_eval(int act, float beta, float z, float& d) {
  if (act == NONE) { d = 1.0f; return z; }
  if (act == RELU) { d = z > 0.0f ? 1.0f : 0.0f; return z < 0.0f ? 0.0f : z; }
  if (act == SOFTPLUS) {
    const float e = exp_minus(fabsf(beta * z));
    const float s = __builtin_amdgcn_rcpf(1.0f + e);
    d = z != z ? z : (z > 0.0f ? s : e * s);
    return (z < 0.0f ? 0.0f : z) + log1pf(e) / beta;
  }
  if (act == GELU) {
    const float phi = 0.5f * erfcf(-0.70710678118654752f * z);      // erfc: no cancellation for negative z
    d = phi + z * (0.3989422804014327f * exp_minus(0.5f * z * z));
    return z * phi;
  }
  const float e = exp_minus(fabsf(z));
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  const float s = z < 0.0f ? e * r : r, c = z < 0.0f ? r : e * r;   // sigmoid(z), sigmoid(-z)
  if (act == SIGMOID) { d = z != z ? z : s * c; return z != z ? z : s; }
  d = s * (1.0f + z * c);
  return z * s;
}

// ---- LDS ---------------------------------------------------------------------------------------------------------------------
// byte offset of a chunk in one plane of an operand's tile (BA tile rows x BK values of the reduction)
template <int SRC, int BA, int BK> struct Tile {
  static constexpr int BYTES = BA * BK * 2;
  // ROWS: row = tile row, c = chunk along the reduction.  Rows of 128 or 64 bytes; 16 rows x one c fill the 64 banks once.
  // COLS: row = value of the reduction, c = chunk along the tile axis.  4 rows x one 64-byte group fill the banks once.
  static __device__ __forceinline__ int at(int row, int c) {
    if (SRC == ROWS) return row * BK * 2 + ((BK == 64 ? c ^ ((row >> 1) & 7) : c ^ ((row >> 2) & 3)) << 4);
    const int g = (c >> 2) ^ (BA == 64 ? (row >> 1) & 1 : row & 3);
    return row * BA * 2 + (g << 6) + ((c & 3) << 4);
  }
};

__device__ __forceinline__ int perm32(int j) {      // column 16 h + 4 q + s of a block of 32 -> MFMA row 8 q + 4 h + s
  return (j & ~31) | (((j >> 2) & 3) << 3) | (((j >> 4) & 1) << 2) | (j & 3);
}

__device__ __forceinline__ f32x16 mfma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mfma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// the lane's MFMA operand: tile rows 32 blk + (lane & 31), reduction 16 kk + 8 (lane >> 5) + 0..7.  PERM: the rows permuted (COLS; a
// ROWS tile is stored permuted)
template <typename L8, int SRC, int BA, int BK, bool PERM> __device__ __forceinline__ L8 fragment(const char* plane, int blk, int kk, int lane) {
  if (SRC == ROWS) return *(const L8*)(plane + Tile<SRC, BA, BK>::at(blk * 32 + (lane & 31), 2 * kk + (lane >> 5)));
  // ds_read_b64_tr_b16: lane s of 16 addresses 4 columns of one row; lane i receives column i of the four rows 4 s' .. 4 s' + 3
  const int b = (lane >> 4) & 1, s = lane & 15, x = s & 3;
  const int row = 16 * kk + 8 * (lane >> 5) + (s >> 2), col = PERM ? 16 * (x & 1) + 4 * (2 * b + (x >> 1)) : 16 * b + 4 * x;
  const int off = row * BA * 2 + ((blk ^ (BA == 64 ? (row >> 1) & 1 : row & 3)) << 6) + col * 2;
  typedef __attribute__((address_space(3))) i16x4 lds4;
  const i16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(plane + off));
  const i16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(plane + off + 4 * BA * 2));
  return __builtin_bit_cast(L8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// ---- staging -----------------------------------------------------------------------------------------------------------------
template <typename T, int DM> struct Factor { typedef typename Ty<T>::D type; };
template <typename T> struct Factor<T, MASK> { typedef T type; };

// One operand's step in registers: BA tile rows x BK values in chunks, NC per thread of NT.  SINGLE: the tensors may hold fewer than
// 8 elements before an end (reductions shorter than 8, or a tiny tensor).
template <typename T, int SRC, int DM, bool PERM, int BA, int NT, bool SINGLE> struct Stage {
  typedef typename Factor<T, DM>::type Q;
  typedef typename Ty<T>::L L;
  static constexpr int BK = Ty<T>::BK, PL = Ty<T>::PLANES, CH = BK / 8, CW = BA / 8, NC = BA * BK / 8 / NT;
  typedef Tile<SRC, BA, BK> Tl;
  Chunk<T> v[NC];
  Chunk<Q> q[DM != PLAIN ? NC : 1];

  // tile rows from a0 (of n), reduction from r0 (of rn; R in memory).  Rows past n repeat the last one and columns past n hold
  // whatever follows in memory: neither reaches an output.  The reduction past rn is zero.  A step that lies inside the tensor takes
  // addresses of one uniform base per chunk plus one 32-bit lane offset; at the edges every chunk is checked.
  template <typename X> static __device__ __forceinline__ void fetch(Chunk<X>* c, const X* p, ll ld, ll a0, ll n, ll r0, ll rn, ll R, int tid) {
    constexpr int ROW = SRC == ROWS ? CH : CW, STEP = NT / ROW;
    if (a0 + BA <= n && r0 + BK <= rn && ld < (1 << 22)) {
      const X* base = p + (SRC == ROWS ? a0 * ld + r0 : r0 * ld + a0);
      const unsigned lane = (unsigned)(tid / ROW) * (unsigned)ld + 8 * (tid % ROW);
#pragma unroll
      for (int u = 0; u < NC; ++u) c[u].load(base + u * STEP * ld + lane);
    } else {
      int gone[NC];                                     // a chunk at an end: the last 8 elements, and so many of them dropped
#pragma unroll
      for (int u = 0; u < NC; ++u) {
        const int row = tid / ROW + u * STEP, col = 8 * (tid % ROW);
        ll a = a0 + (SRC == ROWS ? row : col);
        const ll r = r0 + (SRC == ROWS ? col : row);
        const X* at;
        ll left;                                        // elements that may be taken from here
        if (SRC == ROWS) {
          a = a < n ? a : n - 1;
          at = p + a * ld + r;
          left = rn - r;
        } else {
          at = p + r * ld + a;
          left = r < rn && a < n ? (R - 1 - r) * ld + n - a : 0;      // past the row's end lies the next row, up to the tensor's end
        }
        if (SINGLE) c[u].load_single(at, left);
        else {
          gone[u] = left >= 8 ? 0 : (left <= 0 ? 8 : 8 - (int)left);
          c[u].load(left <= 0 ? p : at - gone[u]);
        }
        __builtin_amdgcn_sched_barrier(0);               // addresses one after another: this is not the path to hold registers for
      }
      if (!SINGLE) {
#pragma unroll
        for (int u = 0; u < NC; ++u) {
          c[u].drop(gone[u]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  __device__ __forceinline__ void load(const T* p, ll ld, const Q* pq, ll ldq, ll a0, ll n, ll r0, ll rn, ll R, int tid) {
    fetch<T>(v, p, ld, a0, n, r0, rn, R, tid);
    if (DM != PLAIN) fetch<Q>(q, pq, ldq, a0, n, r0, rn, R, tid);
  }
  // chunk u to LDS; SUMS: the chunk's 8 columns added up (COLS)
  template <bool SUMS> __device__ __forceinline__ void put(int u, char* lds, float* sums, int tid) {
    constexpr int ROW = SRC == ROWS ? CH : CW;
    const int row = (tid + NT * u) / ROW, c = tid % ROW;
    char* dst = lds + Tl::at(PERM && SRC == ROWS ? perm32(row) : row, c);
    typedef uint32_t V __attribute__((ext_vector_type(4)));
    if constexpr (PL == 1 && DM == PLAIN && !SUMS) {    // 16-bit, as it is
      *(V*)dst = V{v[u].w[0], v[u].w[1], v[u].w[2], v[u].w[3]};
      return;
    }
    float x[8], f[8];
    v[u].floats(x);
    if (DM != PLAIN) q[u].floats(f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (DM == SMOOTH) x[e] *= f[e];
      if (DM == MASK) x[e] = f[e] > 0.0f ? x[e] : 0.0f;
      if (SUMS) sums[e] += x[e];
    }
#pragma unroll
    for (int p = 0; p < PL; ++p) {
      V y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        y[e] = pack2<L>(x[2 * e], x[2 * e + 1]);
        if (PL == 3 && p < 2) {                         // the rest for the next bfloat16
          x[2 * e] -= __builtin_bit_cast(float, y[e] << 16);
          x[2 * e + 1] -= __builtin_bit_cast(float, y[e] & 0xffff0000u);
        }
      }
      *(V*)(dst + p * Tl::BYTES) = y;
    }
  }
};

// ---- results -----------------------------------------------------------------------------------------------------------------
// bias, activation, residual of one output element; returns y and leaves act' in d
template <typename T>
__device__ __forceinline__ float finish(const Args& a, ll i, ll j, float z, float& d) {
  if (a.bias) z += (float)((const T*)a.bias)[j];
  float y = act_eval(a.act, a.beta, z, d);
  if (a.res) y += (float)((const T*)a.res)[i * a.ldr + j];
  return y;
}

template <typename T> __device__ __forceinline__ void keep(const Args& a, ll e, float d) {
  if (a.act == RELU) ((T*)a.dact)[e] = (T)d;
  else ((typename Ty<T>::D*)a.dact)[e] = (typename Ty<T>::D)d;
}

// N floats -> N elements of type X at any element-aligned address, 16 bytes per store
template <typename X, int N> __device__ __forceinline__ void store(X* p, const float* x) {
  typedef uint32_t V2 __attribute__((ext_vector_type(4), aligned(2)));
  typedef uint32_t V4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef typename Pick<sizeof(X) == 4, V4, V2>::type V;
  constexpr int PER = 16 / sizeof(X);
  static_assert(N % 4 == 0, "");
  if constexpr (N < PER) {                             // 4 16-bit elements
    typedef uint32_t H __attribute__((ext_vector_type(2), aligned(2)));
    *(H*)p = H{pack2<X>(x[0], x[1]), pack2<X>(x[2], x[3])};
  } else {
#pragma unroll
    for (int h = 0; h < N; h += PER) {
      V y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (sizeof(X) == 4) y[e] = __builtin_bit_cast(uint32_t, x[h + e]);
        else y[e] = pack2<X>(x[h + 2 * e], x[h + 2 * e + 1]);
      }
      *(V*)(p + h) = y;
    }
  }
}

// ROWS_ x COLS_ finished values of one wave, wholly inside the output.  MODE: an activation (FORWARD), STORE (as they are) or RAW
// (float32 partial sums).
enum Mode { STORE = 16, RAW = 17 };
template <typename T, int ROWS_, int COLS_, int EPITCH, int MODE>
__device__ __forceinline__ void emit(const Args& a, void* out, ll ldo, const float* ep, ll i0, ll j0, int lane) {
  constexpr int C = MODE == RAW || sizeof(T) == 4 ? 4 : 8, LPR = COLS_ / C, RPI = 64 / LPR, UN = 4;
  static_assert(ROWS_ % (RPI * UN) == 0 || ROWS_ / RPI < UN, "");
  const int col = C * (lane % LPR), row0 = lane / LPR;
  const ll j = j0 + col;
  float b[C];
#pragma unroll
  for (int e = 0; e < C; ++e) b[e] = 0.0f;
  if (MODE < STORE && a.bias) {
#pragma unroll
    for (int e = 0; e < C; ++e) b[e] = (float)((const T*)a.bias)[j + e];
  }
  constexpr int IT = ROWS_ / RPI, U = IT < UN ? IT : UN;
#pragma unroll 1
  for (int it = 0; it < IT; it += U) {
    Chunk<T> r[U];                                     // C elements of the residual (float32: the first half)
    if constexpr (MODE < STORE) if (a.res) {
#pragma unroll
      for (int u = 0; u < U; ++u) r[u].load_16((const T*)a.res + (i0 + row0 + (it + u) * RPI) * a.ldr + j);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = row0 + (it + u) * RPI;
      const ll i = i0 + row;
      float z[C], d[C], f[8];
#pragma unroll
      for (int h = 0; h < C; h += 4) {
        const f32x4 x = *(const f32x4*)(ep + row * EPITCH + col + h);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[h + e] = x[e];
      }
      if constexpr (MODE == RAW) store<float, C>((float*)out + i * ldo + j, z);
      else {
        if constexpr (MODE < STORE) {
          if (a.res) r[u].floats(f);
#pragma unroll
          for (int e = 0; e < C; ++e) {
            z[e] = act_eval(MODE, a.beta, z[e] + b[e], d[e]);
            if (a.res) z[e] += f[e];
          }
          if (a.dact && MODE != NONE) {
            if constexpr (MODE == RELU) store<T, C>((T*)a.dact + i * a.J + j, d);
            else store<typename Ty<T>::D, C>((typename Ty<T>::D*)a.dact + i * a.J + j, d);
          }
        }
        store<T, C>((T*)out + i * ldo + j, z);
      }
    }
  }
}

// ---- the tile kernel ---------------------------------------------------------------------------------------------------------
template <typename T, int OP, int WI, int WJ, int NI, int NJ> struct Shape {
  static constexpr int BK = Ty<T>::BK, PL = Ty<T>::PLANES, BI = 32 * NI * WI, BJ = 32 * NJ * WJ, NT = 64 * WI * WJ;
  static constexpr int BUF = PL * (BI + BJ) * BK * 2;                               // one step
  static constexpr int EPITCH = 32 * NJ + 4, EPI = WI * WJ * 32 * NI * EPITCH * 4;  // the tile on its way out
  static constexpr int EXACT = PL == 3 ? (BI + BJ) * (BK + 1) * 4 : 0;
  static constexpr int SUMS = OP == BACK_WEIGHT ? NT * 8 * 4 : 0;
  static constexpr int m1 = 2 * BUF > EPI ? 2 * BUF : EPI, m2 = EXACT > SUMS ? EXACT : SUMS, LDS = m1 > m2 ? m1 : m2;
};

template <typename T, int OP, int DM, int WI, int WJ, int NI, int NJ, bool SINGLE>
__global__ __launch_bounds__(64 * WI * WJ, 2) void tile_kernel(const Args a) {
  typedef Shape<T, OP, WI, WJ, NI, NJ> Sh;
  constexpr int SI = OP == BACK_WEIGHT ? COLS : ROWS, SJ = OP == FORWARD ? ROWS : COLS;
  constexpr int BK = Sh::BK, PL = Sh::PL, BI = Sh::BI, BJ = Sh::BJ, NT = Sh::NT, EPITCH = Sh::EPITCH, KK = BK / 16;
  typedef typename Ty<T>::L8 L8;
  typedef Stage<T, SI, DM, false, BI, NT, SINGLE> StI;
  typedef Stage<T, SJ, PLAIN, true, BJ, NT, SINGLE> StJ;
  extern __shared__ __align__(16) char lds[];

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
  const typename StI::Q* iq = (const typename StI::Q*)a.iq;
  const T* jp = (const T*)a.jp;
  StI si;
  StJ sj;
  float bs[8] = {};
  auto fill = [&](ll r) {
    si.load(ip, a.ild, iq, a.iqld, i0, a.I, r, rend, a.R, tid);
    sj.load(jp, a.jld, (const typename StJ::Q*)nullptr, 0, j0, a.J, r, rend, a.R, tid);
  };
  auto put = [&](int buf) {
    char* b = lds + buf * Sh::BUF;
#pragma unroll
    for (int u = 0; u < StI::NC; ++u) si.template put<OP == BACK_WEIGHT>(u, b, bs, tid);
#pragma unroll
    for (int u = 0; u < StJ::NC; ++u) sj.template put<false>(u, b + PL * StI::Tl::BYTES, nullptr, tid);
  };

  const int wi = wave / WJ, wj = wave % WJ;
  f32x16 acc[NI][NJ] = {};
  auto products = [&](int buf, int kk) {
    const char* bi = lds + buf * Sh::BUF;
    const char* bj = bi + PL * StI::Tl::BYTES;
    L8 fi[NI][PL], fj[NJ][PL];
#pragma unroll
    for (int p = 0; p < PL; ++p) {
#pragma unroll
      for (int b = 0; b < NI; ++b) fi[b][p] = fragment<L8, SI, BI, BK, false>(bi + p * StI::Tl::BYTES, wi * NI + b, kk, lane);
#pragma unroll
      for (int b = 0; b < NJ; ++b) fj[b][p] = fragment<L8, SJ, BJ, BK, true>(bj + p * StJ::Tl::BYTES, wj * NJ + b, kk, lane);
    }
#pragma unroll
    for (int sum = PL - 1; sum >= 0; --sum)            // the small products first
#pragma unroll
      for (int p = sum; p >= 0; --p)
#pragma unroll
        for (int x = 0; x < NI; ++x)
#pragma unroll
          for (int y = 0; y < NJ; ++y) acc[x][y] = mfma(fj[y][p], fi[x][sum - p], acc[x][y]);
  };
  if (rbeg < rend) {
    fill(rbeg);
    put(0);
    if (rbeg + BK < rend) fill(rbeg + BK);
    __syncthreads();
    int buf = 0;
    for (ll r = rbeg; r + BK < rend; r += BK) {
      products(buf, 0);
      put(buf ^ 1);
      if (r + 2 * BK < rend) fill(r + 2 * BK);
#pragma unroll
      for (int kk = 1; kk < KK; ++kk) products(buf, kk);
      __syncthreads();
      buf ^= 1;
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) products(buf, kk);
  }

  if (PL == 3) {
    int bad = 0;
#pragma unroll
    for (int x = 0; x < NI; ++x)
#pragma unroll
      for (int y = 0; y < NJ; ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          bad |= !(fabsf(acc[x][y][e]) < __builtin_huge_valf()) && j0 + (wj * NJ + y) * 32 + 16 * (lane >> 5) + e < a.J;
    if (__syncthreads_or(bad)) {                       // float32 products: rows of BK + 1 floats, two values of the reduction per MFMA
      float* fl = (float*)lds;
#pragma unroll
      for (int x = 0; x < NI; ++x)
#pragma unroll
        for (int y = 0; y < NJ; ++y) acc[x][y] = f32x16{};
      for (ll r = rbeg; r < rend; r += BK) {
        __syncthreads();
        for (int q = tid; q < (BI + BJ) * BK; q += NT) {
          const int rr = q % BK, row = q / BK;
          const ll rg = r + rr;
          float x = 0.0f;
          if (rg < rend) {
            if (row < BI) {
              ll i = i0 + row;
              i = i < a.I ? i : a.I - 1;
              x = (float)ip[SI == ROWS ? i * a.ild + rg : rg * a.ild + i];
              if (DM != PLAIN) {
                const float d = (float)iq[SI == ROWS ? i * a.iqld + rg : rg * a.iqld + i];
                x = DM == MASK ? (d > 0.0f ? x : 0.0f) : x * d;
              }
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
          for (int x = 0; x < NI; ++x)
#pragma unroll
            for (int y = 0; y < NJ; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x2f32(fj[y], fi[x], acc[x][y], 0, 0, 0);
        }
      }
    }
  }

  // the tile leaves through LDS: a lane then finishes 16 bytes of a row, and rows are stored in whole cache lines
  float* ep = (float*)lds + wave * 32 * NI * EPITCH;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < NI; ++x)
#pragma unroll
    for (int y = 0; y < NJ; ++y)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *(f32x4*)(ep + (x * 32 + (lane & 31)) * EPITCH + y * 32 + 16 * (lane >> 5) + 4 * q) =
            f32x4{acc[x][y][4 * q], acc[x][y][4 * q + 1], acc[x][y][4 * q + 2], acc[x][y][4 * q + 3]};
  __syncthreads();
  const ll iw = i0 + wi * NI * 32, jw = j0 + wj * NJ * 32;
  if (i0 + BI <= a.I && j0 + BJ <= a.J) {
    if (a.part) emit<T, 32 * NI, 32 * NJ, EPITCH, RAW>(a, a.part + s * a.I * a.J, a.J, ep, iw, jw, lane);
    else if (OP != FORWARD) emit<T, 32 * NI, 32 * NJ, EPITCH, STORE>(a, a.out, a.ldo, ep, iw, jw, lane);
    else if (a.act == NONE) emit<T, 32 * NI, 32 * NJ, EPITCH, NONE>(a, a.out, a.ldo, ep, iw, jw, lane);
    else if (a.act == RELU) emit<T, 32 * NI, 32 * NJ, EPITCH, RELU>(a, a.out, a.ldo, ep, iw, jw, lane);
    else if (a.act == SOFTPLUS) emit<T, 32 * NI, 32 * NJ, EPITCH, SOFTPLUS>(a, a.out, a.ldo, ep, iw, jw, lane);
    else if (a.act == SIGMOID) emit<T, 32 * NI, 32 * NJ, EPITCH, SIGMOID>(a, a.out, a.ldo, ep, iw, jw, lane);
    else if (a.act == SILU) emit<T, 32 * NI, 32 * NJ, EPITCH, SILU>(a, a.out, a.ldo, ep, iw, jw, lane);
    else emit<T, 32 * NI, 32 * NJ, EPITCH, GELU>(a, a.out, a.ldo, ep, iw, jw, lane);
  } else {                                             // a tile at an edge: one element per lane
    const int rows = a.I - iw < 32 * NI ? (int)(a.I - iw) : 32 * NI, cols = a.J - jw < 32 * NJ ? (int)(a.J - jw) : 32 * NJ;
    for (int e = lane; e < rows * cols && cols > 0; e += 64) {
      const int row = e / cols, col = e % cols;
      const ll i = iw + row, j = jw + col;
      float z = ep[row * EPITCH + col], d;
      if (a.part) {
        a.part[(s * a.I + i) * a.J + j] = z;
        continue;
      }
      if (OP == FORWARD) z = finish<T>(a, i, j, z, d);
      ((T*)a.out)[i * a.ldo + j] = (T)z;
      if (OP == FORWARD && a.dact) keep<T>(a, i * a.J + j, d);
    }
  }

  if (OP == BACK_WEIGHT && a.bias_bar && tj == 0) {    // bbar: the threads that share 8 columns
    float* fl = (float*)lds;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) fl[(tid / StI::CW) * BI + 8 * (tid % StI::CW) + e] = bs[e];
    __syncthreads();
    if (tid < BI && i0 + tid < a.I) {
      float x = 0.0f;
      for (int c = 0; c < NT / StI::CW; ++c) x += fl[c * BI + tid];
      if (a.part) a.part_bias[s * a.I + i0 + tid] = x;
      else ((T*)a.bias_bar)[i0 + tid] = (T)x;
    }
  }
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------
// FORWARD for at most 8 rows of x: one wave per column of the output reads its row of W once, 16 bytes per lane, against all rows of
// x (float32 FMA), and adds up over the wave.  Bound by reading W; x stays in the caches.
template <typename T, int M>
__global__ __launch_bounds__(256) void few_kernel(const Args a) {
  constexpr int C = 16 / sizeof(T);
  const int lane = threadIdx.x & 63;
  const ll j = (ll)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (j >= a.J) return;
  const T* w = (const T*)a.jp + j * a.jld;
  const T* x = (const T*)a.ip;
  float acc[M] = {};
  const ll whole = a.R / C * C;
#pragma unroll 2
  for (ll r = lane * C; r < whole; r += 64 * C) {
    Chunk<T> cw, cx;
    float fw[8], fx[8];
    cw.load_16(w + r);
    cw.floats(fw);
#pragma unroll
    for (int m = 0; m < M; ++m) {
      cx.load_16(x + m * a.ild + r);
      cx.floats(fx);
#pragma unroll
      for (int e = 0; e < C; ++e) acc[m] = fmaf(fw[e], fx[e], acc[m]);
    }
  }
  if (whole + lane < a.R) {
    const float fw = (float)w[whole + lane];
#pragma unroll
    for (int m = 0; m < M; ++m) acc[m] = fmaf(fw, (float)x[m * a.ild + whole + lane], acc[m]);
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int d = 32; d > 0; d /= 2) acc[m] += __shfl_xor(acc[m], d);
  float z = acc[0], d;
#pragma unroll
  for (int m = 1; m < M; ++m) z = lane == m ? acc[m] : z;
  if (lane < M) {
    z = finish<T>(a, lane, j, z, d);
    ((T*)a.out)[lane * a.ldo + j] = (T)z;
    if (a.dact) keep<T>(a, lane * a.J + j, d);
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
  if (OP == FORWARD && a.dact) keep<T>(a, e, d);
}

// ---- host --------------------------------------------------------------------------------------------------------------------
struct Plan {
  bool few, big, tiny;
  int S;
  ll TI, TJ, chunk;
};

// tile edges of the large variant (the small one is 64 x 64)
static constexpr int big_i(int dtype) { return dtype == F32 ? 256 : 128; }
static constexpr int big_j(int dtype) { return 128; }

// Which tile and how many splits of the reduction: 256 CUs want at least one workgroup each.
static Plan plan(int op, int dtype, ll I, ll J, ll R) {
  const int BK = dtype == F32 ? 32 : 64;
  auto tiles = [&](int ti, int tj) { return ((I + ti - 1) / ti) * ((J + tj - 1) / tj); };
  Plan p = {};
  p.S = 1;
  p.few = op == FORWARD && I <= 8;
  if (p.few) return p;
  p.tiny = R < 8 || I < 8 || J < 8;         // an operand may hold fewer than 8 elements before its end: loaded one by one
  p.big = !p.tiny && (tiles(big_i(dtype), big_j(dtype)) >= 192 || (I >= 128 && J >= 128 && R >= 8192));
  const int ti = p.big ? big_i(dtype) : 64, tj = p.big ? big_j(dtype) : 64;
  const ll n = tiles(ti, tj) < 1 ? 1 : tiles(ti, tj);
  ll s = n >= 256 ? 1 : 512 / n, most = R / (4 * BK);
  s = s < most ? s : most;
  s = s < 1 ? 1 : (s > 512 ? 512 : s);
  p.chunk = ((R + s - 1) / s + BK - 1) / BK * BK;
  if (p.chunk < BK) p.chunk = BK;                       // R = 0: the gradient of no rows, one pass over nothing
  p.S = (int)((R + p.chunk - 1) / p.chunk);
  if (p.S < 1) p.S = 1;
  p.TI = (I + ti - 1) / ti;
  p.TJ = (J + tj - 1) / tj;
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
  const Plan p = plan(op, dtype, I, J, R);
  return p.S == 1 ? 0 : 4 * (ll)p.S * (I * J + (op == BACK_WEIGHT ? I : 0));
}

// more than 64 KB of LDS has to be asked for, once per kernel and device (idempotent: no lock)
template <typename T, int OP, int DM, int WI, int WJ, int NI, int NJ, bool SINGLE = false> static int start(const Args& a, unsigned grid, hipStream_t st) {
  typedef Shape<T, OP, WI, WJ, NI, NJ> Sh;
  static bool ready[64];
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -2;
  auto* kernel = tile_kernel<T, OP, DM, WI, WJ, NI, NJ, SINGLE>;
  if (!ready[dev]) {
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, Sh::LDS) != hipSuccess) return -2;
    ready[dev] = true;
  }
  kernel<<<dim3(grid), Sh::NT, Sh::LDS, st>>>(a);
  return 0;
}

template <typename T, int OP, int DM> static int start_tile(const Args& a, bool big, bool tiny, unsigned grid, hipStream_t st) {
  if (tiny) return start<T, OP, DM, 2, 2, 1, 1, true>(a, grid, st);
  if (!big) return start<T, OP, DM, 2, 2, 1, 1>(a, grid, st);
  if constexpr (sizeof(T) == 4) return start<T, OP, DM, 4, 2, 2, 2>(a, grid, st);
  else return start<T, OP, DM, 2, 2, 2, 2>(a, grid, st);
}

template <typename T, int OP>
static int run(const Call& c, hipStream_t st) {
  Args a = {};
  shape(OP, c.m, c.n, c.k, a.I, a.J, a.R);
  const Plan p = plan(OP, c.dtype, a.I, a.J, a.R);
  const ll need = workspace_bytes(OP, c.dtype, c.m, c.n, c.k);
  if (need > 0 && (!c.ws || c.ws_bytes < need)) return -3;
  a.ip = OP == FORWARD ? c.x : c.ybar;
  a.ild = OP == FORWARD ? c.ldx : c.ldyb;
  a.iq = OP == FORWARD ? nullptr : c.dact;
  a.iqld = c.ldd;
  a.jp = OP == BACK_WEIGHT ? c.x : c.w;
  a.jld = OP == BACK_WEIGHT ? c.ldx : c.ldw;
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
  if (p.S > 1) {
    a.part = (float*)c.ws;
    a.part_bias = a.part + (ll)p.S * a.I * a.J;
  }
  if constexpr (OP == FORWARD) {
    if (p.few) {
      const dim3 grid((unsigned)((a.J + 3) / 4));
      switch (a.I) {
        case 1: few_kernel<T, 1><<<grid, 256, 0, st>>>(a); break;
        case 2: few_kernel<T, 2><<<grid, 256, 0, st>>>(a); break;
        case 3: few_kernel<T, 3><<<grid, 256, 0, st>>>(a); break;
        case 4: few_kernel<T, 4><<<grid, 256, 0, st>>>(a); break;
        case 5: few_kernel<T, 5><<<grid, 256, 0, st>>>(a); break;
        case 6: few_kernel<T, 6><<<grid, 256, 0, st>>>(a); break;
        case 7: few_kernel<T, 7><<<grid, 256, 0, st>>>(a); break;
        default: few_kernel<T, 8><<<grid, 256, 0, st>>>(a);
      }
      return hipGetLastError() == hipSuccess ? 0 : -2;
    }
  }
  const unsigned grid = (unsigned)(p.TI * p.TJ * p.S);
  int rc;
  if constexpr (OP == FORWARD) rc = start_tile<T, OP, PLAIN>(a, p.big, p.tiny, grid, st);
  else rc = c.act == NONE ? start_tile<T, OP, PLAIN>(a, p.big, p.tiny, grid, st) : (c.act == RELU ? start_tile<T, OP, MASK>(a, p.big, p.tiny, grid, st)
                                                                                          : start_tile<T, OP, SMOOTH>(a, p.big, p.tiny, grid, st));
  if (rc) return rc;
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
