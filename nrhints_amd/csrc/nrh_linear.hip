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
//   * 16-bit types: v_mfma_f32_32x32x16_{f16,bf16}.  zbar = ybar act' has more bits than the type, and more range than float16.  For
//     NONE and RELU it is exact.  For the smooth activations:
//     bfloat16: two parts of the type, the rounded value and the rounded rest (16 bits), and two products, whatever the tile: the same
//     rows have the same precision in every batch.  Rounded once, the gradients' rms error was 1.4 times that of rounding the outputs
//     alone, at 49 us for dx of 16 384 x 1 024 x 1 024 against 77 (dW 68 against 84) and 20 against 25 of 16 384 x 512 x 512.
//     float16: zbar as two bfloat16 parts (16 bits, float32's range), x and W as two (exact: 11 bits), three products - the rests' product
//     is at most 2^-16 of the pair.  As float16 numbers, products of 2^-12 and 2^-13 would be zero and those past 65 504 infinite,
//     though their sums fit the type (16 384 x 1 024 x 1 024: dx 108 us, dW 116 against 50 and 66 in float16).
//     act' itself is kept in float32: no other rounding joins these, and a saturated unit's act' (1e-9 of a sigmoid at -20)
//     keeps all its bits.  In parts, large tiles are 128 x 256: A, which is formed from two tensors, for as many columns as fit (256 x 128
//     take 97 us where these take 77; 256 x 256 spill registers, 98).
//   * float32: x = x0 + x1 + x2 in three bfloat16 (each the rounded rest of the one before: 24 bits), and the six products x_a w_b
//     with a + b <= 2 on v_mfma_f32_32x32x16_bf16.  What is left out is at most 2^-23 of |x w|, two of float32's own half steps
//     (x1 w2 and x2 w1, 2^-24 each); six passes at the bf16 rate are 2.6 times the rate of v_mfma_f32_32x32x2_f32.  bfloat16 has
//     float32's exponents, so nothing is scaled; but its numbers end at 2^-133, float32's at 2^-149: below 2^-109 the parts leave out up
//     to 2^-134 of x itself.
// Operands in parts: infinities, NaN and values that round up to infinity make the parts NaN, and an infinity on the other side
// meets parts that are zero or of the other sign.  A tile whose sums are not all finite is computed again with
// v_mfma_f32_32x32x2_f32, so its results are those of float32 arithmetic.
// The MFMA's A role is played by the j operand, its rows permuted (column j = 16 h + 4 q + s of a block of 32 is MFMA row
// 8 q + 4 h + s): a lane then holds 16 consecutive columns of ONE output row.
// Measured: 16 384 x 1 024 x 1 024 bf16 38 us (0.9 PFLOP/s; a large library product reaches 1.6), 8 192 x 2 048 x 2 048 67 us (1.0);
// 163 840 x 256 x 256 f32 145 us (148 TFLOP/s; the library's float32 products reach 154): of its 3.0e5 cycles (2.1 GHz) the MFMAs take 40 %
// and vector instructions 36 %, mostly the three-way split, which every row tile repeats for W; 655 360 x 256 x 256 bf16 with a residual
// 218 us (1.0 GB at 4.6 TB/s, the rate of a copy).  Small products are bound by the latency of their steps, about 0.4 us each.
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
enum Deriv { PLAIN = 0, SMOOTH = 1, MASK = 2, PARTS = 3 };      // A as it is, times act', kept where act' > 0 (RELU), times act' in two parts

template <typename T> struct Ty;                    // planes, LDS element
template <> struct Ty<float> { static constexpr int PLANES = 3; typedef __bf16 L; typedef bf16x8 L8; };
template <> struct Ty<_Float16> { static constexpr int PLANES = 1; typedef _Float16 L; typedef f16x8 L8; };
template <> struct Ty<__bf16> { static constexpr int PLANES = 1; typedef __bf16 L; typedef bf16x8 L8; };

// how a product of tensors of type T with A's act' taken as DM is formed: planes (the parts an operand is split into) of A and B, their type
template <typename T, int DM> struct How : Ty<T> { static constexpr int PI = Ty<T>::PLANES, PJ = PI; };
template <> struct How<_Float16, PARTS> : Ty<__bf16> { static constexpr int PI = 2, PJ = 2; };
template <> struct How<__bf16, PARTS> : Ty<__bf16> { static constexpr int PI = 2, PJ = 1; };

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
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < W; ++e) w[e] = 0;
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
  // the first k (0 .. 8) elements and zeros
  __device__ __forceinline__ void first(int k) {
    constexpr int PER = 4 / sizeof(X);
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const int have = k - PER * e;
      w[e] = have >= PER ? w[e] : (PER == 2 && have == 1 ? w[e] & 0xffffu : 0u);
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
  __device__ __forceinline__ void pair(int e, float& a, float& b) const {      // elements 2 e and 2 e + 1
    if constexpr (sizeof(X) == 4) {
      a = __builtin_bit_cast(float, w[(2 * e) % W]);
      b = __builtin_bit_cast(float, w[(2 * e + 1) % W]);
    } else {
      typedef X X2 __attribute__((ext_vector_type(2)));
      const X2 t = __builtin_bit_cast(X2, w[e]);
      a = (float)t[0];
      b = (float)t[1];
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

// log(1 + e), 0 <= e <= 1: a series below 1/64 (the next term is under 2^-26 of it), above it log(u) e / (u - 1) of the rounded
// u = 1 + e (Goldberg, What Every Computer Scientist Should Know About Floating-Point Arithmetic, theorem 4)
__device__ __forceinline__ float log1p_unit(float e) {
  if (e < 0.015625f) return e * (1.0f - e * (0.5f - e * (0.333333343f - e * 0.25f)));
  const float u = 1.0f + e;
  return 0.693147182f * __builtin_amdgcn_logf(u) * (e * __builtin_amdgcn_rcpf(u - 1.0f));
}

// erfc(x), 0 <= x <= 14, as e^(-x^2) t P(t), t = 1 / (1 + x / 2) (the substitution of Press et al., Numerical Recipes, section 6.2): P
// is the polynomial of degree 8 with the least relative error over that range (4.5e-8, by reweighted least squares on Chebyshev nodes in
// float64; 5.6 2^-24 as evaluated here).  ex2: e^(-x^2).
__device__ __forceinline__ float erfc_positive(float x, float ex2) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.5f, x, 1.0f));
  float q = fmaf(t, -0.05938727781f, 0.28612756729f);
  q = fmaf(t, q, -0.49041295052f);
  q = fmaf(t, q, 0.28173971176f);
  q = fmaf(t, q, -0.02915211208f);
  q = fmaf(t, q, 0.20375365019f);
  q = fmaf(t, q, 0.24283494055f);
  q = fmaf(t, q, 0.28241211176f);
  q = fmaf(t, q, 0.28208434582f);
  return ex2 * (t * q);
}

// act(z) and act'(z); every exponential has a non-positive argument, so none overflows, and NaN passes through.  The rounding of an
// exponential's argument is a relative error of its value, so it is kept beside it (fma) and multiplied on: in the tails y and act' are
// right to 8 units of their own last place (with the argument as rounded 180 for GELU at -12, 66 for softplus at beta z = -80).
__device__ __forceinline__ float act_eval(int act, float beta, float z, float& d) {
  if (act == NONE) { d = 1.0f; return z; }
  if (act == RELU) { d = z > 0.0f ? 1.0f : 0.0f; return z < 0.0f ? 0.0f : z; }
  if (act == SOFTPLUS) {
    const float a = fminf(fabsf(beta * z), 150.0f), rest = fmaf(beta, fabsf(z), -a);
    const float e = exp_minus(a) * (1.0f - (a < 150.0f ? rest : 0.0f));
    const float s = __builtin_amdgcn_rcpf(1.0f + e);
    d = z != z ? z : (z > 0.0f ? s : e * s);
    return (z < 0.0f ? 0.0f : z) + log1p_unit(e) * __builtin_amdgcn_rcpf(beta);
  }
  if (act == GELU) {                                   // z Phi(z), Phi(z) = erfc(-z / sqrt 2) / 2
    const float a = fminf(fabsf(z), 19.75f), s = a * a;
    const float ex2 = exp_minus(0.5f * s) * fmaf(-0.5f, fmaf(a, a, -s), 1.0f);
    const float half = 0.5f * erfc_positive(a * 0.70710678118654752f, ex2), phi = z < 0.0f ? half : 1.0f - half;
    d = phi + z * (0.3989422804014327f * ex2);
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
  // ROWS: row = tile row, c = chunk along the reduction.  Rows of 128, 64 or 32 bytes; 16 rows x one c fill the 64 banks once.
  // COLS: row = value of the reduction, c = chunk along the tile axis.  4 rows x one 64-byte group fill the banks once.
  static __device__ __forceinline__ int at(int row, int c) {
    if (SRC == ROWS) return row * BK * 2 + ((BK == 64 ? c ^ ((row >> 1) & 7) : (BK == 32 ? c ^ ((row >> 2) & 3) : c ^ ((row >> 3) & 1))) << 4);
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

template <typename L> __device__ __forceinline__ void halves(uint32_t w, float& a, float& b) {      // the two 16-bit floats of a word
  typedef L L2 __attribute__((ext_vector_type(2)));
  const L2 t = __builtin_bit_cast(L2, w);
  a = (float)t[0];
  b = (float)t[1];
}

// ---- staging -----------------------------------------------------------------------------------------------------------------
template <typename T, int DM> struct Factor { typedef float type; };      // act' in memory
template <typename T> struct Factor<T, MASK> { typedef T type; };

// One operand's step in registers: BA tile rows x BK values in chunks, NC per thread of NT.  SINGLE: a tensor may hold fewer than
// 16 elements.
template <typename T, typename L, int PL, int SRC, int DM, bool PERM, int BA, int BK, int NT, bool SINGLE> struct Stage {
  typedef typename Factor<T, DM>::type Q;
  static constexpr int CH = BK / 8, CW = BA / 8, NC = BA * BK / 8 / NT;
  typedef Tile<SRC, BA, BK> Tl;
  Chunk<T> v[NC];
  Chunk<Q> q[DM != PLAIN ? NC : 1];

  // tile rows from a0 (of n), reduction from r0 (of rn; R in memory).  Rows past n repeat the last one and columns past n hold
  // whatever follows in memory: neither reaches an output.  The reduction past rn is zero.  A step that lies inside the tensor takes
  // addresses of one uniform base per chunk plus one 32-bit lane offset; at the edges every chunk is checked.
  template <typename X> static __device__ __forceinline__ void fetch(Chunk<X>* c, const X* p, ll ld, ll a0, ll n, ll r0, ll rn, ll R, int tid) {
    constexpr int ROW = SRC == ROWS ? CH : CW, STEP = NT / ROW;
    const bool axis = a0 + BA <= n || (SRC == COLS && (R - r0 - BK) * ld + n >= a0 + BA);      // (COLS: rows enough behind the step)
    if (axis && r0 + BK <= rn && ld < (1 << 22)) {
      const X* base = p + (SRC == ROWS ? a0 * ld + r0 : r0 * ld + a0);
      const unsigned lane = (unsigned)(tid / ROW) * (unsigned)ld + 8 * (tid % ROW);
#pragma unroll
      for (int u = 0; u < NC; ++u) c[u].load(base + u * STEP * ld + lane);
    } else {
      // (addresses are worked out here, every time: moved out of the loop they would hold dozens of registers)
      asm volatile("" : "+v"(tid));
      // a chunk at an end: the tensor's last 8 elements, and so many of them dropped; a short row's, when others follow: loaded on
      // into the next row, and all but so many cut off (below zero)
      int some = 0, gone[NC];
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
        const bool any = SRC == COLS && r < rn && a >= n;              // columns past n: any values

        if (SINGLE) c[u].load_single(at, left);
        else {
          gone[u] = left >= 8 || any ? 0 : (left <= 0 ? 8 : 8 - (int)left);
          some |= gone[u];
          const bool on = SRC == ROWS && left < 8 && at + 8 <= p + (n - 1) * ld + R;
          c[u].load(left <= 0 ? p : at - (on ? 0 : gone[u]));
          if (on && left > 0) gone[u] = -(int)left;
        }
        __builtin_amdgcn_sched_barrier(0);               // addresses one after another: this is not the path to hold registers for
      }
      if (!SINGLE && __ballot(some != 0)) {              // (dropping waits for the loads: only where an end is in reach)
#pragma unroll
        for (int u = 0; u < NC; ++u) {
          c[u].drop(gone[u] > 0 ? gone[u] : 0);
          if (SRC == ROWS) c[u].first(gone[u] < 0 ? -gone[u] : 8);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  __device__ __forceinline__ void load(const T* p, ll ld, const Q* pq, ll ldq, ll a0, ll n, ll r0, ll rn, ll R, int tid) {
    fetch<T>(v, p, ld, a0, n, r0, rn, R, tid);
    if (DM != PLAIN) fetch<Q>(q, pq, ldq, a0, n, r0, rn, R, tid);
  }
  // The way to LDS in pieces of a few instructions, to stand between MFMAs: piece q of PIECES.  SUMS: the 8 columns of the chunks added
  // up (COLS).
  static constexpr bool COPY = PL == 1 && DM == PLAIN;
  static constexpr int PPC = COPY ? 1 : 4 * PL, PIECES = NC * PPC;       // pieces per chunk, in all
  template <bool SUMS> __device__ __forceinline__ void piece(int q, float (&x)[8], uint32_t (&y)[3][4], char* lds, float* sums, int tid) const {
    constexpr int ROW = SRC == ROWS ? CH : CW;
    const int u = q / PPC, e = q % PPC / PL, p = q % PL;
    typedef uint32_t V __attribute__((ext_vector_type(4)));
    const int row = (tid + NT * u) / ROW, c = tid % ROW;
    char* dst = lds + Tl::at(PERM && SRC == ROWS ? perm32(row) : row, c);
    if (COPY) {
      *(V*)dst = V{v[u].w[0], v[u].w[1], v[u].w[2], v[u].w[3]};
      if (SUMS) {
        v[u].floats(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[i] += x[i];
      }
      return;
    }
    if (p == 0) {
      v[u].pair(e, x[2 * e], x[2 * e + 1]);
      if (DM != PLAIN) {
        float f0, f1;
        q_pair(u, e, f0, f1);
        if (DM == SMOOTH || DM == PARTS) { x[2 * e] *= f0; x[2 * e + 1] *= f1; }
        if (DM == MASK) { x[2 * e] = f0 > 0.0f ? x[2 * e] : 0.0f; x[2 * e + 1] = f1 > 0.0f ? x[2 * e + 1] : 0.0f; }
      }
      if (SUMS) { sums[2 * e] += x[2 * e]; sums[2 * e + 1] += x[2 * e + 1]; }
    }
    y[p][e] = pack2<L>(x[2 * e], x[2 * e + 1]);
    if (p < PL - 1) {                                   // the rest for the next part
      float h0, h1;
      halves<L>(y[p][e], h0, h1);
      x[2 * e] -= h0;                                   // (NaN of an infinity: the tile is computed again)
      x[2 * e + 1] -= h1;
    }
    if (e == 3) *(V*)(dst + p * Tl::BYTES) = V{y[p][0], y[p][1], y[p][2], y[p][3]};
  }
  __device__ __forceinline__ void q_pair(int u, int e, float& a, float& b) const { q[DM != PLAIN ? u : 0].pair(e, a, b); }
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
  else ((float*)a.dact)[e] = d;
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

template <typename X, int N> __device__ __forceinline__ void put(X* p, const float* x, int left) {      // ... the first `left` of them
  if (left >= N) store<X, N>(p, x);
  else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < left) p[e] = (X)x[e];
  }
}

// 32 x COLS_ finished values of one wave, of which rows x cols lie in the output.  MODE: an activation (FORWARD), STORE (as they are) or
// RAW (float32 partial sums).  WHOLE: all do, and nothing is asked per row (655 360 x 256 x 256 bf16 with a residual: 215 us against 247).
enum Mode { STORE = 16, RAW = 17 };
template <typename T, int COLS_, int EPITCH, int MODE, bool WHOLE>
__device__ __forceinline__ void emit(const Args& a, void* out, ll ldo, const float* ep, ll i0, ll j0, int rows, int cols, int lane) {
  constexpr int C = MODE == RAW || sizeof(T) == 4 ? 4 : 8, LPR = COLS_ / C, RPI = 64 / LPR, UN = 4;
  constexpr int IT = 32 / RPI, U = IT < UN ? IT : UN;
  const int col = C * (lane % LPR), row0 = lane / LPR, left = WHOLE ? C : cols - col;      // columns of this lane that exist
  if (left <= 0) return;
  const ll j = j0 + col;
  float b[C];
#pragma unroll
  for (int e = 0; e < C; ++e) b[e] = 0.0f;
  if (MODE < STORE && a.bias) {
#pragma unroll
    for (int e = 0; e < C; ++e)
      if (e < left) b[e] = (float)((const T*)a.bias)[j + e];
  }
#pragma unroll 1
  for (int it = 0; it < IT; it += U) {
    Chunk<T> r[U];                                     // C elements of the residual (float32: the first half)
    if constexpr (MODE < STORE) if (a.res) {
      const T* p = (const T*)a.res + (i0 + row0 + it * RPI) * a.ldr + j;
      if (WHOLE) {
#pragma unroll
        for (int u = 0; u < U; ++u) r[u].load_16(p + u * RPI * a.ldr);
      } else {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (row0 + (it + u) * RPI >= rows) r[u].zero();
          else if (left >= C) r[u].load_16(p + u * RPI * a.ldr);
          else r[u].load_single(p + u * RPI * a.ldr, left);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int row = row0 + (it + u) * RPI;
      if (!WHOLE && row >= rows) break;
      const ll i = i0 + row;
      float z[C], d[C], f[8];
#pragma unroll
      for (int h = 0; h < C; h += 4) {
        const f32x4 x = *(const f32x4*)(ep + row * EPITCH + col + h);
#pragma unroll
        for (int e = 0; e < 4; ++e) z[h + e] = x[e];
      }
      if constexpr (MODE == RAW) put<float, C>((float*)out + i * ldo + j, z, left);
      else {
        if constexpr (MODE < STORE) {
          if (a.res) r[u].floats(f);
#pragma unroll
          for (int e = 0; e < C; ++e) {
            z[e] = act_eval(MODE, a.beta, z[e] + b[e], d[e]);
            if (a.res) z[e] += f[e];
          }
          if (a.dact && MODE != NONE) {
            if constexpr (MODE == RELU) put<T, C>((T*)a.dact + i * a.J + j, d, left);
            else put<float, C>((float*)a.dact + i * a.J + j, d, left);
          }
        }
        put<T, C>((T*)out + i * ldo + j, z, left);
      }
    }
  }
}

template <int N> struct Const { constexpr operator int() const { return N; } };

// ---- the tile kernel ---------------------------------------------------------------------------------------------------------
template <typename T, int OP, int DM, int WI, int WJ, int NI, int NJ, int BK> struct Shape {
  static constexpr int PI = How<T, DM>::PI, PJ = How<T, DM>::PJ, BI = 32 * NI * WI, BJ = 32 * NJ * WJ, NT = 64 * WI * WJ;
  static constexpr int BUF = (PI * BI + PJ * BJ) * BK * 2;                               // one step
  static constexpr int EPITCH = 32 * NJ + 4, EPI = WI * WJ * 32 * EPITCH * 4;       // the tile on its way out
  static constexpr int EXACT = PI > 1 ? (BI + BJ) * (BK + 1) * 4 : 0;
  static constexpr int SUMS = OP == BACK_WEIGHT ? NT * 8 * 4 : 0;
  static constexpr int m1 = 2 * BUF > EPI ? 2 * BUF : EPI, m2 = EXACT > SUMS ? EXACT : SUMS, LDS = m1 > m2 ? m1 : m2;
};

template <typename T, int OP, int DM, int WI, int WJ, int NI, int NJ, int BK, int OCC, bool SINGLE>
__global__ __launch_bounds__(64 * WI * WJ, OCC) void tile_kernel(const Args a) {
  typedef Shape<T, OP, DM, WI, WJ, NI, NJ, BK> Sh;
  constexpr int SI = OP == BACK_WEIGHT ? COLS : ROWS, SJ = OP == FORWARD ? ROWS : COLS;
  constexpr int PI = Sh::PI, PJ = Sh::PJ, BI = Sh::BI, BJ = Sh::BJ, NT = Sh::NT, EPITCH = Sh::EPITCH, KK = BK / 16;
  typedef typename How<T, DM>::L L;
  typedef typename How<T, DM>::L8 L8;
  typedef Stage<T, L, PI, SI, DM, false, BI, BK, NT, SINGLE> StI;
  typedef Stage<T, L, PJ, SJ, PLAIN, true, BJ, BK, NT, SINGLE> StJ;
  extern __shared__ __align__(16) char lds[];

  const int tid = threadIdx.x, lane = tid & 63;
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
  float bs[8] = {}, px[8];
  uint32_t py[3][4];
  auto fill = [&](ll r) {
    si.load(ip, a.ild, iq, a.iqld, i0, a.I, r, rend, a.R, tid);
    sj.load(jp, a.jld, (const typename StJ::Q*)nullptr, 0, j0, a.J, r, rend, a.R, tid);
  };
  constexpr int PIECES = StI::PIECES + StJ::PIECES;
  auto piece = [&](int q, int buf) {
    char* b = lds + buf * Sh::BUF;
    if (q < StI::PIECES) si.template piece<OP == BACK_WEIGHT>(q, px, py, b, bs, tid);
    else sj.template piece<false>(q - StI::PIECES, px, py, b + PI * StI::Tl::BYTES, nullptr, tid);
  };

  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wave / WJ, wj = wave % WJ;
  f32x16 acc[NI][NJ] = {};
  constexpr int READS = NI * PI + NJ * PJ, MF = NI * NJ * (PJ == 3 ? 6 : PI + PJ - 1);      // per 16 values of the reduction
  constexpr int PUT0 = KK > 2 ? KK - 3 : 0, PUTS = KK - 1 - PUT0;              // the sixteens beside which the next step goes to LDS
  static_assert(KK >= 2, "");
  struct Operands { L8 i[NI][PI], j[NJ][PJ]; };
  Operands f[2];
  auto read = [&](Operands& o, int kk, int q, int buf) {
    const char* bi = lds + buf * Sh::BUF;
    const char* bj = bi + PI * StI::Tl::BYTES;
    // the plane that both have first, then the others
    const int both = PI < PJ ? PI : PJ, p = q < both * (NI + NJ) ? q / (NI + NJ) : both + (q - both * (NI + NJ)) / NI;
    const int b = q < both * (NI + NJ) ? q % (NI + NJ) : (q - both * (NI + NJ)) % NI;
    if (b < NI) o.i[b % NI][p] = fragment<L8, SI, BI, BK, false>(bi + p * StI::Tl::BYTES, wi * NI + b, kk, lane);
    else o.j[(b - NI) % NJ][p % PJ] = fragment<L8, SJ, BJ, BK, true>(bj + p * StJ::Tl::BYTES, wj * NJ + b - NI, kk, lane);
  };
  auto product = [&](const Operands& o, int q) {       // the small products first
    constexpr int QI[6] = {2, 0, 1, 0, 1, 0}, QJ[6] = {0, 2, 1, 1, 0, 0};      // three parts each: a + b <= 2
    constexpr int HI[3] = {1, 0, 0}, HJ[3] = {0, 1, 0};                        // two and two: a + b <= 1; two and one
    const int t = q / (NI * NJ), x = q % (NI * NJ) / NJ, y = q % NJ;
    acc[x][y] = mfma(o.j[y][(PJ == 3 ? QJ[t] : HJ[t]) % PJ], o.i[x][(PJ == 3 ? QI[t] : HI[t]) % PI], acc[x][y]);
  };
  // The kk-th 16 values of a step, and between their MFMAs - in this order, a few instructions after each - the reads of the next
  // sixteen's operands (READ; the last one reads the next step's first, from the other buffer) and pieces of the next step's way to LDS.
  auto sixteen = [&](auto KK_, auto READ, auto PUT, int buf) {
    constexpr int kk = KK_, R = READ ? READS : 0;
    constexpr int P = PUT && kk >= PUT0 && kk < KK - 1 ? PIECES : 0, p0 = P * (kk - PUT0) / PUTS, p1 = P * (kk - PUT0 + 1) / PUTS;
#pragma unroll
    for (int q = 0; q < MF; ++q) {
      product(f[kk & 1], q);
#pragma unroll
      for (int e = 2 * R * q / MF; e < 2 * R * (q + 1) / MF; ++e)      // operands in the first half
        if (e < R) read(f[(kk + 1) & 1], (kk + 1) % KK, e, kk + 1 < KK ? buf : buf ^ 1);
#pragma unroll
      for (int e = p0 + (p1 - p0) * q / MF; e < p0 + (p1 - p0) * (q + 1) / MF; ++e) piece(e, buf ^ 1);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  typedef Const<1> Yes;
  typedef Const<0> No;
  if (rbeg < rend) {
    fill(rbeg);
#pragma unroll
    for (int q = 0; q < PIECES; ++q) piece(q, 0);
    if (rbeg + BK < rend) fill(rbeg + BK);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < READS; ++e) read(f[0], 0, e, 0);
    int buf = 0;
    // One barrier per step, before its last sixteen: behind it lie the next step's chunks, and nobody reads the buffer that is
    // written next (its last operands were read before the barrier of the step before).
    for (ll r = rbeg; r + BK < rend; r += BK) {
      sixteen(Const<0>(), Yes(), Yes(), buf);
      if constexpr (KK > 2) sixteen(Const<1>(), Yes(), Yes(), buf);
      if constexpr (KK > 3) sixteen(Const<2>(), Yes(), Yes(), buf);
      if (r + 2 * BK < rend) fill(r + 2 * BK);
      __syncthreads();
      sixteen(Const<KK - 1>(), Yes(), No(), buf);
      buf ^= 1;
    }
    sixteen(Const<0>(), Yes(), No(), buf);
    if constexpr (KK > 2) sixteen(Const<1>(), Yes(), No(), buf);
    if constexpr (KK > 3) sixteen(Const<2>(), Yes(), No(), buf);
    sixteen(Const<KK - 1>(), No(), No(), buf);
  }

  if (PI > 1) {                                        // operands in parts
    int bad = 0;
#pragma unroll
    for (int x = 0; x < NI; ++x)
#pragma unroll
      for (int y = 0; y < NJ; ++y)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          bad |= !(fabsf(acc[x][y][e]) < __builtin_huge_valf()) && j0 + (wj * NJ + y) * 32 + 16 * (lane >> 5) + e < a.J &&
                 i0 + (wi * NI + x) * 32 + (lane & 31) < a.I;
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

  // the tile leaves through LDS, 32 rows of a wave at a time: a lane then finishes 16 bytes of a row, and rows are stored in whole
  // cache lines
  float* ep = (float*)lds + wave * 32 * EPITCH;
  const ll jw = j0 + wj * NJ * 32;
#pragma unroll 1
  for (int x = 0; x < NI; ++x) {
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NI; ++v)                       // (registers have no index)
      if (v == x) {
#pragma unroll
        for (int y = 0; y < NJ; ++y)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            *(f32x4*)(ep + (lane & 31) * EPITCH + y * 32 + 16 * (lane >> 5) + 4 * q) =
                f32x4{acc[v][y][4 * q], acc[v][y][4 * q + 1], acc[v][y][4 * q + 2], acc[v][y][4 * q + 3]};
      }
    __syncthreads();
    const ll iw = i0 + (wi * NI + x) * 32;
    const int rows = a.I - iw < 32 ? (int)(a.I - iw) : 32, cols = a.J - jw < 32 * NJ ? (int)(a.J - jw) : 32 * NJ;
    auto leave = [&](auto WHOLE) {
      constexpr bool W = WHOLE;
      if (a.part) emit<T, 32 * NJ, EPITCH, RAW, W>(a, a.part + s * a.I * a.J, a.J, ep, iw, jw, rows, cols, lane);
      else if (OP != FORWARD) emit<T, 32 * NJ, EPITCH, STORE, W>(a, a.out, a.ldo, ep, iw, jw, rows, cols, lane);
      else if (a.act == NONE) emit<T, 32 * NJ, EPITCH, NONE, W>(a, a.out, a.ldo, ep, iw, jw, rows, cols, lane);
      else if (a.act == RELU) emit<T, 32 * NJ, EPITCH, RELU, W>(a, a.out, a.ldo, ep, iw, jw, rows, cols, lane);
      else if (a.act == SOFTPLUS) emit<T, 32 * NJ, EPITCH, SOFTPLUS, W>(a, a.out, a.ldo, ep, iw, jw, rows, cols, lane);
      else if (a.act == SIGMOID) emit<T, 32 * NJ, EPITCH, SIGMOID, W>(a, a.out, a.ldo, ep, iw, jw, rows, cols, lane);
      else if (a.act == SILU) emit<T, 32 * NJ, EPITCH, SILU, W>(a, a.out, a.ldo, ep, iw, jw, rows, cols, lane);
      else emit<T, 32 * NJ, EPITCH, GELU, W>(a, a.out, a.ldo, ep, iw, jw, rows, cols, lane);
    };
    if (rows == 32 && cols == 32 * NJ) leave(Const<1>());
    else leave(Const<0>());
  }
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------
// FORWARD for at most 8 rows of x: one wave per column of the output reads its row of W once, 16 bytes per lane, against all rows of
// x (float32 FMA), and adds up over the wave.  Bound by reading W; x stays in the caches.  1 024 x 1 024 bf16: 2.8 us for one row, 5.6 for 8,
// against 7.6 for 9 on 64 x 64 tiles; 256 x 256 f32 2.6, 3.3 and 8.7.
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

// Joins the S partial outputs in a fixed order and finishes them like the tile kernel: 4 elements per thread, each as SLICES sums over
// every SLICES-th part (a thread's loads come in turns of 8, each a trip to memory: 67 x 6 elements of 512
// parts take 48 us with the product on 64 slices and 58 on 16, 256 x 256 elements of 256 parts 77 and 63).  Bound by reading the parts.
template <typename T, int OP, int SLICES>
__global__ __launch_bounds__(256) void reduce_kernel(const Args a) {
  constexpr int LANES = 256 / SLICES;
  __shared__ f32x4 buf[SLICES][LANES];
  const int lane = threadIdx.x % LANES, slice = threadIdx.x / LANES;
  const ll n = a.I * a.J, extra = OP == BACK_WEIGHT && a.bias_bar ? a.I : 0, groups = (n + 3) / 4;
  const ll g = (ll)blockIdx.x * LANES + lane;
  const bool main = g < groups;
  const ll e = 4 * (main ? g : g - groups), step = main ? n : a.I, left = (main ? n : extra) - e;
  f32x4 z = {};
  if (left > 0) {
    typedef float V __attribute__((ext_vector_type(4), aligned(4)));
    const float* p = (main ? a.part : a.part_bias) + e;
    if (left >= 4) {
#pragma unroll 8
      for (int s = slice; s < a.S; s += SLICES) {
        const V x = *(const V*)(p + s * step);
#pragma unroll
        for (int q = 0; q < 4; ++q) z[q] += x[q];
      }
    } else {
      for (int s = slice; s < a.S; s += SLICES)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q < left) z[q] += p[s * step + q];
    }
  }
  if (SLICES > 1) {
    buf[slice][lane] = z;
    __syncthreads();
    if (slice != 0) return;
    for (int s = 1; s < SLICES; ++s)
#pragma unroll
      for (int q = 0; q < 4; ++q) z[q] += buf[s][lane][q];
  }
  if (left <= 0) return;
  if (!main) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < left) ((T*)a.bias_bar)[e + q] = (T)z[q];
    return;
  }
  ll i = e / a.J, j = e % a.J;
  const bool row = j + 4 <= a.J;                       // one row's: a single store
  float y[4], d[4];
  ll at[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    at[q] = i * a.ldo + j;
    y[q] = z[q];
    if (OP == FORWARD && q < left) y[q] = finish<T>(a, i, j, z[q], d[q]);
    if (++j == a.J) { j = 0; ++i; }
  }
  if (row) store<T, 4>((T*)a.out + at[0], y);
  else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < left) ((T*)a.out)[at[q]] = (T)y[q];
  }
  if (OP == FORWARD && a.dact) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (q < left) keep<T>(a, e + q, d[q]);
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------------
// Tile variants: rows x columns of the output.  Long reductions reach (8 192 x 4 096 x 4 096 bf16) 480, 880 and 1 180 TFLOP/s on SMALL,
// MIDDLE and LARGE, (8 192 x 2 048 x 2 048 f32) 130 and 212 on SMALL and LARGE; small outputs want many small tiles.
enum Variant { FEW = 0, TINY, SMALL, MIDDLE, LARGE };
struct Size { int i, j; };
static Size size_of(int dtype, bool parts, int v) {
  if (v <= SMALL) return {64, 64};
  if (parts) return {128, 256};
  if (v == MIDDLE) return {128, 128};                   // 16-bit types
  return dtype == F32 ? Size{256, 128} : Size{256, 256};
}

// What a launch takes, in microseconds, with w tiles per CU that each reduce L values: start + L max(alone, w each) + (w - 1) tile; and
// S > 1 splits' parts: JOIN + I J (S PART + LAST).  Fitted (rms 12 %) to 2 034 timings of 20 shapes from 64 x 1 024 x 1 024 to
// 400 000 x 256 x 256, every variant at 1 to 256 splits; the choice by it is on average 2 % above the best of each.  (Gradients in parts:
// 748 timings of 18 shapes, rms 10 %, 1 %.)
struct Cost { float start, alone, each, tile; };
static Cost cost_of(int dtype, bool act_bar, bool parts, int v) {
  if (v == TINY) return {4.0f, 0.036f, 0.006f, 0.30f};
  if (dtype == F32) return v <= SMALL ? Cost{4.0f, 0.0234f, 0.0156f, 0.31f} : Cost{7.9f, 0.0388f, 0.0644f, 7.6f};
  if (parts && dtype == F16) return v <= SMALL ? Cost{4.34f, 0.0155f, 0.0110f, 0.82f} : Cost{7.92f, 0.0137f, 0.0426f, 5.18f};
  if (parts) return v <= SMALL ? Cost{4.48f, 0.0134f, 0.0085f, 0.40f} : Cost{7.83f, 0.0228f, 0.0278f, 6.02f};
  if (v <= SMALL) return act_bar ? Cost{3.6f, 0.0109f, 0.0065f, 0.18f} : Cost{3.4f, 0.0092f, 0.0042f, 0.46f};
  if (v == MIDDLE) return act_bar ? Cost{5.6f, 0.0121f, 0.0164f, 0.60f} : Cost{5.75f, 0.0011f, 0.0121f, 0.89f};
  return act_bar ? Cost{8.3f, 0.0093f, 0.0343f, 7.2f} : Cost{8.2f, 0.0040f, 0.0295f, 7.1f};
}
constexpr float JOIN = 3.24f, PART = 1.07e-6f, LAST = 1.1e-7f;

struct Plan {
  int variant, S;
  ll TI, TJ, chunk;
};

// the variant and the number of splits with the least cost
static Plan plan(int op, int dtype, int act, ll I, ll J, ll R) {
  const int CHUNK = 64, MOST = 512;                     // CHUNK: a multiple of every variant's step
  Plan p = {};
  p.S = 1;
  if (op == FORWARD && I <= 8) return p;                // FEW
  const bool act_bar = op != FORWARD && act != NONE, parts = act_bar && act != RELU && dtype != F32;
  const ll steps = R > 0 ? (R + CHUNK - 1) / CHUNK : 1; // R = 0: the gradient of no rows, one pass over nothing
  // Loaded one by one: operands of less than two chunks, reductions that end inside the first chunk (305 747 x 2 x 20 bf16 16 us against
  // 24) and columns that do (the weight gradient of 510 170 x 50 x 3 f16 34 us against 41: chunks would read on into the rows behind).
  const bool tiny = R < 8 || I * R < 16 || J * R < 16 || (op != FORWARD && J < 8) || (op == BACK_WEIGHT && I < 8);
  float best = 0.0f;
  for (int v = tiny ? TINY : SMALL; v <= (tiny ? TINY : LARGE); ++v) {
    if (v == MIDDLE && (dtype == F32 || parts)) continue;
    const Size z = size_of(dtype, parts, v);
    const Cost c = cost_of(dtype, act_bar, parts, v);
    const ll TI = (I + z.i - 1) / z.i, TJ = (J + z.j - 1) / z.j;
    for (int s = 1; s <= MOST && s <= steps; s = s < 4 ? s + 1 : s + (s & (s - 1) ? s / 3 : s / 2)) {      // 1 2 3 4 6 8 12 16 ..
      const ll chunk = (steps + s - 1) / s, S = (steps + chunk - 1) / chunk, n = TI * TJ * S;
      const float w = n > 2048 ? n / 256.0f : (float)((n + 255) / 256);
      const float each = c.each * w;
      const float t = c.start + chunk * CHUNK * (each > c.alone ? each : c.alone) + (w - 1) * c.tile + (S > 1 ? JOIN + (float)I * J * (S * PART + LAST) : 0);
      if (p.variant == FEW || t < best) {
        best = t;
        p = {v, (int)S, TI, TJ, chunk * CHUNK};
      }
    }
  }
  return p;
}

static void shape(int op, ll m, ll n, ll k, ll& I, ll& J, ll& R) {
  I = op == BACK_WEIGHT ? n : m;
  J = op == FORWARD ? n : k;
  R = op == FORWARD ? k : (op == BACK_DATA ? n : m);
}

long long workspace_bytes(int op, int dtype, int act, long long m, long long n, long long k) {
  ll I, J, R;
  shape(op, m, n, k, I, J, R);
  const Plan p = plan(op, dtype, act, I, J, R);
  return p.S == 1 ? 0 : 4 * (ll)p.S * (I * J + (op == BACK_WEIGHT ? I : 0));
}

// more than 64 KB of LDS has to be asked for, once per kernel and device (idempotent: no lock)
template <typename T, int OP, int DM, int WI, int WJ, int NI, int NJ, int BK, int OCC, bool SINGLE = false> static int start(const Args& a, unsigned grid, hipStream_t st) {
  typedef Shape<T, OP, DM, WI, WJ, NI, NJ, BK> Sh;
  static bool ready[64];
  int dev = -1;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return -2;
  auto* kernel = tile_kernel<T, OP, DM, WI, WJ, NI, NJ, BK, OCC, SINGLE>;
  if (!ready[dev]) {
    if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, Sh::LDS) != hipSuccess) return -2;
    ready[dev] = true;
  }
  kernel<<<dim3(grid), Sh::NT, Sh::LDS, st>>>(a);
  return 0;
}

template <typename T, int OP, int DM> static int start_tile(const Args& a, int variant, unsigned grid, hipStream_t st) {
  constexpr int DS = sizeof(T) == 2 && DM == SMOOTH ? PARTS : DM;
  if (variant == TINY) return start<T, OP, DS, 2, 2, 1, 1, 32, 2, true>(a, grid, st);
  if constexpr (sizeof(T) == 4) {
    if (variant == SMALL) return start<T, OP, DM, 2, 2, 1, 1, 32, 2>(a, grid, st);
    return start<T, OP, DM, 4, 2, 2, 2, 32, 2>(a, grid, st);
  } else if constexpr (DS == PARTS) {
    if (variant == SMALL) return start<T, OP, DS, 2, 2, 1, 1, 64, 2>(a, grid, st);
    return start<T, OP, DS, 2, 4, 2, 2, How<T, DS>::PJ == 1 ? 64 : 32, 2>(a, grid, st);      // (float16: 64 is more than LDS holds)
  } else {
    if (variant == SMALL) return start<T, OP, DM, 2, 2, 1, 1, 64, 2>(a, grid, st);
    if (variant == LARGE) return start<T, OP, DM, 2, 4, 4, 2, DM == PLAIN ? 64 : 32, 2>(a, grid, st);      // (act' takes registers)
    return start<T, OP, DM, 2, 2, 2, 2, 64, 2>(a, grid, st);
  }
}

template <typename T, int OP>
static int run(const Call& c, hipStream_t st) {
  Args a = {};
  shape(OP, c.m, c.n, c.k, a.I, a.J, a.R);
  const Plan p = plan(OP, c.dtype, c.act, a.I, a.J, a.R);
  const ll need = workspace_bytes(OP, c.dtype, c.act, c.m, c.n, c.k);
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
    if (p.variant == FEW) {
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
  if constexpr (OP == FORWARD) rc = start_tile<T, OP, PLAIN>(a, p.variant, grid, st);
  else rc = c.act == NONE ? start_tile<T, OP, PLAIN>(a, p.variant, grid, st) : (c.act == RELU ? start_tile<T, OP, MASK>(a, p.variant, grid, st)
                                                                                          : start_tile<T, OP, SMOOTH>(a, p.variant, grid, st));
  if (rc) return rc;
  if (p.S > 1) {
    const ll n = (a.I * a.J + 3) / 4 + (a.bias_bar ? (a.I + 3) / 4 : 0);
    if (p.S < 8) reduce_kernel<T, OP, 1><<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>(a);
    else if (p.S < 32) reduce_kernel<T, OP, 4><<<dim3((unsigned)((n + 63) / 64)), 256, 0, st>>>(a);
    else if (p.S < 128 || n > 8192) reduce_kernel<T, OP, 16><<<dim3((unsigned)((n + 15) / 16)), 256, 0, st>>>(a);
    else reduce_kernel<T, OP, 64><<<dim3((unsigned)((n + 3) / 4)), 256, 0, st>>>(a);
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
