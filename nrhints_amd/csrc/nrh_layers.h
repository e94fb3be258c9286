// Host-side interface between nrh_api.hip and the layer operators' translation units (nrh_linear.hip, nrh_embedding.hip).
#pragma once
#include <hip/hip_runtime.h>

namespace nrhlin {

enum Dtype { F32 = 0, F16 = 1, BF16 = 2 };
enum Act { NONE = 0, RELU = 1, SOFTPLUS = 2, SIGMOID = 3, SILU = 4, GELU = 5 };
enum Op { FORWARD = 0, BACK_DATA = 1, BACK_WEIGHT = 2 };

// One product  out[i, j] = sum_r A(i, r) B(j, r)  of a layer  y = act(x W^T + b) + residual,  x [m, k], W [n, k], y [m, n]:
//   FORWARD      i = m, j = n, r = k   A = x, B = W                        (then bias, activation, residual)
//   BACK_DATA    i = m, j = k, r = n   A = zbar = ybar * act'(z), B = W
//   BACK_WEIGHT  i = n, j = k, r = m   A = zbar, B = x                     (and the bias gradient, the row sums of A)
struct Call {
  int op, dtype, act;
  float beta;               // softplus
  long long m, n, k;
  const void* x;            // FORWARD, BACK_WEIGHT
  long long ldx;
  const void* w;            // FORWARD, BACK_DATA
  long long ldw;
  const void* bias;         // FORWARD, may be null
  const void* res;          // FORWARD, may be null
  long long ldr;
  const void* ybar;         // BACK_*
  long long ldyb;
  const void* dact;         // BACK_*: act'(z) in float32, or - RELU - anything of the tensors' type that is positive exactly where z
                            // is; null: activation NONE
  long long ldd;
  void* out;                // y | xbar | wbar, rows of ldo elements
  long long ldo;
  void* dact_out;           // FORWARD: act'(z) [m, n] in the type above, may be null
  void* bias_bar;           // BACK_WEIGHT: [n], may be null
  void* ws;
  long long ws_bytes;
};
long long workspace_bytes(int op, int dtype, int act, long long m, long long n, long long k);
int launch(const Call& c, hipStream_t st);     // 0 ok, -2 launch error, -3 workspace too small

}  // namespace nrhlin

namespace nrhemb {

// rows [n, d] = scale * table[index] and the table's gradient; an index outside [0, v) stands for no row (zeros, no gradient)
struct Call {
  int dtype;                // nrhlin::Dtype
  int index64;              // index is int64 (else int32)
  const void* index;        // [n]
  long long n, v, d;
  float scale;
  const void* src;          // table [v, d] | rows_bar [n, d]
  long long lds;
  void* dst;                // rows [n, d] | table_bar [v, d]
  long long ldd;
  void* ws;
  long long ws_bytes;
};
long long backward_workspace_bytes(long long n, long long v, long long d);
int forward(const Call& c, hipStream_t st);    // 0 ok, -2 launch error
int backward(const Call& c, hipStream_t st);   // 0 ok, -2 launch error, -3 workspace too small

}  // namespace nrhemb
