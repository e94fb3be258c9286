// Table lookup with scaling,  rows[i] = s T[idx[i]],  and its gradient  Tbar[v] = s sum_{idx[i] = v} rowsbar[i].
//
// The gradient sorts the tokens by index - stable, so a row's tokens stay in their order - and sums runs of equal index: no atomics on
// floating point numbers, the same bits on every run, float32 sums, one rounding.
//   low tables (at most 255 rows, partial tables of at most 8 MB): a workgroup sorts 512 tokens in LDS and sums them into its own [rows, d]
//             partial table; a second launch adds the partial tables up (one workgroup of tokens: no second launch).  131 072 tokens of 12
//             float32: 13.7 us into 255 rows, 43.7 by the general way into 256; 62 000 x 64 18 against 40.
//   others    sort: up to 1 024 tokens bitonic in LDS, one launch (25 us with the sums; 2 048 that way 33, by digits 28); more: least
//             significant digit first, 8 bits per pass (histogram per tile of 1 024 tokens, ranked scatter; the scan between them is part
//             of the scatter up to 64 tiles, one launch less for each pass at the same time).
//             sum: a group of lanes - one lane per 16 bytes of a row - walks 16 or 32 sorted tokens.  A run that begins and ends inside is
//             written to the table; the first and the last run of a group may go on in its neighbours and are handed, as float32
//             rows with their keys, to the next level, which does the same with 16 entries per group, until at most 2 048 are left:
//             those meet in one launch.  A row named by every token and a table named once per row cost the same.  Rows that no token
//             names are found by bisection in the sorted keys and cleared beside the first level: every row is written once.
// Both directions are bound by HBM at large sizes (the tokens' rows are read once, the table's gradient is written once): the lookup of
// 16 384 rows of 1 024 bf16 takes 13 us (5 TB/s), the gradient of 40 000 of them into 50 000 rows 74 us (184 MB, 39 us of a copy), of which
// the sort is 25.  Small ones are bound by launches.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "nrh_layers.h"

namespace nrhemb {

typedef long long ll;
typedef unsigned long long ull;
constexpr unsigned NONE = 0xffffffffu;
constexpr int TILE = 1024, SMALL = 1024, FOLD = 64, RUN1 = 16, LOW = 255, LOW_TOKENS = 512, TAIL = 2048, TAIL_GROUPS = 64;

// V elements at any element-aligned address (global memory takes unaligned vector accesses).  A row of d >= V elements is covered by
// ceil(d / V) vectors, the last one drawn back to end with the row: what two of them share is the same values twice.
template <typename T, int V> struct Vec;
template <> struct Vec<float, 4> { typedef float type __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct Vec<float, 8> { typedef float type __attribute__((ext_vector_type(8), aligned(4))); };
template <> struct Vec<_Float16, 8> { typedef _Float16 type __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct Vec<__bf16, 8> { typedef __bf16 type __attribute__((ext_vector_type(8), aligned(2))); };
template <typename T> struct Vec<T, 1> { typedef T type; };
template <int V> __device__ __forceinline__ int column(int c, int d) { return c * V < d - V ? c * V : d - V; }
template <typename T, int V> __device__ __forceinline__ float at(const typename Vec<T, V>::type& x, int e) {
  if constexpr (V == 1) return (float)x;
  else return (float)x[e];
}
template <typename T, int V> __device__ __forceinline__ void put(typename Vec<T, V>::type& x, int e, float f) {
  if constexpr (V == 1) x = (T)f;
  else x[e] = (T)f;
}

__device__ __forceinline__ ll load_index(const void* index, int index64, ll i) {
  return index64 ? ((const ll*)index)[i] : (ll)((const int*)index)[i];
}

// one lane per V columns of a row
template <typename T, int V>
__global__ __launch_bounds__(256) void lookup_kernel(const void* index, int index64, ll n, ll v, int cols, int d, float scale, const T* __restrict__ table,
                                                     ll ldt, T* __restrict__ rows, ll ldr) {
  typedef typename Vec<T, V>::type VT;
  for (ll e = (ll)blockIdx.x * 256 + threadIdx.x; e < n * cols; e += (ll)gridDim.x * 256) {
    const ll i = e / cols, c = column<V>((int)(e % cols), d);
    const ll k = load_index(index, index64, i);
    VT y = {};
    if (k >= 0 && k < v) {
      const VT x = *(const VT*)(table + k * ldt + c);
#pragma unroll
      for (int q = 0; q < V; ++q) put<T, V>(y, q, scale * at<T, V>(x, q));
    }
    *(VT*)(rows + i * ldr + c) = y;
  }
}

// ---- sort --------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned key_of(const void* index, int index64, ll i, ll v) {
  const ll k = load_index(index, index64, i);
  return (unsigned)(k >= 0 && k < v ? k : v);
}

__global__ __launch_bounds__(1024) void sort_small_kernel(const void* index, int index64, int n, ll v, unsigned* keys, unsigned* perm) {
  __shared__ ull a[SMALL];
  const int tid = threadIdx.x;
  int m = 2;
  while (m < n) m *= 2;
  for (int i = tid; i < m; i += 1024) a[i] = i < n ? ((ull)key_of(index, index64, i, v) << 32) | (unsigned)i : ~0ull;
  for (int k = 2; k <= m; k *= 2)
    for (int j = k / 2; j > 0; j /= 2) {
      __syncthreads();
      for (int t = tid; t < m / 2; t += 1024) {
        const int lo = 2 * t - (t & (j - 1)), hi = lo + j;
        const ull x = a[lo], y = a[hi];
        if ((x > y) == ((lo & k) == 0)) {
          a[lo] = y;
          a[hi] = x;
        }
      }
    }
  __syncthreads();
  for (int i = tid; i < n; i += 1024) {
    keys[i] = (unsigned)(a[i] >> 32);
    perm[i] = (unsigned)a[i];
  }
}

struct Pass {
  const void* index;      // first pass: keys come from the caller's index, positions count up
  int index64, first, shift;
  ll n, v;
  const unsigned *keys_in, *perm_in;
  unsigned *keys_out, *perm_out;
  unsigned *hist, *total;  // [tiles][256]; [256] (more than FOLD tiles: after scan_kernel)
  ll tiles;
};

__device__ __forceinline__ unsigned pass_key(const Pass& p, ll i) { return p.first ? key_of(p.index, p.index64, i, p.v) : p.keys_in[i]; }

__global__ __launch_bounds__(256) void hist_kernel(const Pass p) {
  __shared__ unsigned h[256];
  h[threadIdx.x] = 0;
  __syncthreads();
  const ll base = (ll)blockIdx.x * TILE;
  for (int r = 0; r < TILE / 256; ++r) {
    const ll i = base + r * 256 + threadIdx.x;
    if (i < p.n) atomicAdd(&h[(pass_key(p, i) >> p.shift) & 255], 1u);      // counts: the order does not matter
  }
  __syncthreads();
  p.hist[(ll)blockIdx.x * 256 + threadIdx.x] = h[threadIdx.x];
}

// exclusive scan over 256 values, one per thread; buf [256]
__device__ __forceinline__ unsigned scan256(unsigned x, unsigned* buf, unsigned& total) {
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  unsigned in = x;                                       // inclusive within the wave
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const unsigned y = __shfl_up(in, d);
    if (lane >= d) in += y;
  }
  __syncthreads();
  if (lane == 63) buf[wave] = in;
  __syncthreads();
  const unsigned w0 = buf[0], w1 = buf[1], w2 = buf[2];
  total = w0 + w1 + w2 + buf[3];
  return in - x + (wave > 0 ? w0 : 0) + (wave > 1 ? w1 : 0) + (wave > 2 ? w2 : 0);
}

__global__ __launch_bounds__(256) void scan_kernel(const Pass p) {
  __shared__ unsigned buf[256];
  unsigned* h = p.hist + blockIdx.x;                     // one digit
  unsigned carry = 0;
  for (ll b = 0; b < p.tiles; b += 256) {
    const ll i = b + threadIdx.x;
    unsigned total;
    const unsigned ex = scan256(i < p.tiles ? h[i * 256] : 0, buf, total);
    if (i < p.tiles) h[i * 256] = carry + ex;
    carry += total;
  }
  if (threadIdx.x == 0) p.total[blockIdx.x] = carry;
}

__global__ __launch_bounds__(256) void scatter_kernel(const Pass p) {
  constexpr int ROUNDS = TILE / 256;
  __shared__ unsigned cnt[4][256];
  __shared__ unsigned buf[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const ll base = (ll)blockIdx.x * TILE + wave * (TILE / 4);
  unsigned key[ROUNDS], from[ROUNDS], rank[ROUNDS];      // everything that is read, first
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const ll i = base + r * 64 + lane;
    key[r] = i < p.n ? pass_key(p, i) : 0;
    from[r] = p.first ? (unsigned)i : (i < p.n ? p.perm_in[i] : 0);
  }
  for (int w = 0; w < 4; ++w) cnt[w][tid] = 0;
  unsigned all, before_me = 0, total = 0;                // of digit tid: in the tiles before this one, in all
  if (p.tiles <= FOLD) {
#pragma unroll 8
    for (int t = 0; t < (int)p.tiles; ++t) {
      const unsigned x = p.hist[t * 256 + tid];
      before_me += t < (int)blockIdx.x ? x : 0;
      total += x;
    }
  } else {
    before_me = p.hist[(ll)blockIdx.x * 256 + tid];
    total = p.total[tid];
  }
  const unsigned digit_base = scan256(total, buf, all) + before_me;
  __syncthreads();
  volatile unsigned* mine = cnt[wave];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const bool live = base + r * 64 + lane < p.n;
    const unsigned d = (key[r] >> p.shift) & 255;
    ull peers = __ballot(live);
#pragma unroll
    for (int b = 0; b < 8; ++b) {
      const ull on = __ballot((d >> b) & 1);
      peers &= (d >> b) & 1 ? on : ~on;
    }
    const unsigned before = (unsigned)__popcll(peers & ((1ull << lane) - 1));
    if (live) {
      const unsigned c = mine[d];
      rank[r] = c + before;
      if (before == 0) mine[d] = c + (unsigned)__popcll(peers);
    }
  }
  __syncthreads();
  unsigned c = digit_base;
  for (int w = 0; w < 4; ++w) {
    const unsigned x = cnt[w][tid];
    cnt[w][tid] = c;
    c += x;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const ll i = base + r * 64 + lane;
    if (i < p.n) {
      const unsigned to = cnt[wave][(key[r] >> p.shift) & 255] + rank[r];
      p.keys_out[to] = key[r];
      p.perm_out[to] = from[r];
    }
  }
}

// ---- sums --------------------------------------------------------------------------------------------------------------------
struct Level {
  const unsigned *keys, *perm;   // perm: first level only
  const void* rows;              // first level: T [.., ldr], else float [n][d]
  ll ldr, n, v;
  int d, cols, width;            // cols: vectors per row; width: lanes per group
  float scale;
  void* out;
  ll ldo;
  unsigned* next_keys;           // null: the last level
  float* next_rows;
  int run;                       // entries per group
  unsigned sum_blocks;           // first level: the workgroups after these clear rows
};

// 16 table rows per wave: zeros where no sorted key equals the row
template <typename T, int V> __device__ __forceinline__ void clear_rows(const Level& a, ll wave, ll waves) {
  typedef typename Vec<T, V>::type VT;
  const int lane = threadIdx.x & 63;
  for (ll r0 = wave * 16; r0 < a.v; r0 += waves * 16) {
    bool clear = false;
    if (lane < 16 && r0 + lane < a.v) {
      const unsigned row = (unsigned)(r0 + lane);
      ll lo = 0, hi = a.n;
      while (lo < hi) {
        const ll mid = (lo + hi) / 2;
        if (a.keys[mid] < row) lo = mid + 1;
        else hi = mid;
      }
      clear = !(lo < a.n && a.keys[lo] == row);
    }
    const VT z = {};
    for (ull todo = __ballot(clear); todo; todo &= todo - 1) {
      T* out = (T*)a.out + (r0 + __builtin_ctzll(todo)) * a.ldo;
      for (int c = lane; c < a.cols; c += 64) *(VT*)(out + column<V>(c, a.d)) = z;
    }
  }
}

template <typename T, int V, bool FIRST>
__global__ __launch_bounds__(256) void sum_kernel(const Level a) {
  typedef typename Vec<T, V>::type VT;
  typedef typename Vec<float, V>::type FT;
  constexpr int BATCH = FIRST ? 8 : 16;
  if (FIRST && blockIdx.x >= a.sum_blocks) {
    if (blockIdx.y == 0) clear_rows<T, V>(a, (ll)(blockIdx.x - a.sum_blocks) * 4 + (threadIdx.x >> 6), (ll)(gridDim.x - a.sum_blocks) * 4);
    return;
  }
  const ll g = (ll)blockIdx.x * (256 / a.width) + threadIdx.x / a.width;
  const int c = blockIdx.y * a.width + threadIdx.x % a.width;
  const ll beg = g * a.run, end = beg + a.run < a.n ? beg + a.run : a.n;
  if (beg >= a.n || c >= a.cols) return;
  const ll col = column<V>(c, a.d);
  unsigned cur = NONE;
  bool head = true;              // the run in hand is the group's first
  float acc[V];
#pragma unroll
  for (int q = 0; q < V; ++q) acc[q] = 0.0f;
  auto to_table = [&](unsigned k) {
    VT y;
#pragma unroll
    for (int q = 0; q < V; ++q) put<T, V>(y, q, a.scale * acc[q]);
    *(VT*)((T*)a.out + (ll)k * a.ldo + col) = y;
  };
  auto to_next = [&](ll slot, unsigned k) {
    if (c == 0) a.next_keys[slot] = k;
    if (k == NONE) return;
    FT y;
#pragma unroll
    for (int q = 0; q < V; ++q) put<float, V>(y, q, acc[q]);
    *(FT*)(a.next_rows + slot * a.d + col) = y;
  };
  unsigned k[BATCH], from[BATCH], k1[BATCH], from1[BATCH];       // keys and positions of this batch and the next
  auto look = [&](ll e, unsigned (&kk)[BATCH], unsigned (&ff)[BATCH]) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      kk[b] = e + b < end ? a.keys[e + b] : NONE;
      if (FIRST) {
        ff[b] = e + b < end ? a.perm[e + b] : 0;
        if (kk[b] >= (unsigned)a.v) kk[b] = NONE;                // tokens that name no row
      }
    }
  };
  look(beg, k1, from1);
  for (ll e = beg; e < end; e += BATCH) {
    float x[BATCH][V];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      k[b] = k1[b];
      from[b] = from1[b];
    }
    look(e + BATCH, k1, from1);
#pragma unroll
    for (int b = 0; b < BATCH; ++b)
      if (k[b] != NONE) {
        if constexpr (FIRST) {
          const VT y = *(const VT*)((const T*)a.rows + (ll)from[b] * a.ldr + col);
#pragma unroll
          for (int q = 0; q < V; ++q) x[b][q] = at<T, V>(y, q);
        } else {
          const FT y = *(const FT*)((const float*)a.rows + (e + b) * a.ldr + col);
#pragma unroll
          for (int q = 0; q < V; ++q) x[b][q] = at<float, V>(y, q);
        }
      }
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      if (k[b] == NONE) continue;
      if (k[b] != cur) {
        if (cur != NONE) {
          if (head && a.next_keys) to_next(2 * g, cur);
          else to_table(cur);
          head = false;
        }
        cur = k[b];
#pragma unroll
        for (int q = 0; q < V; ++q) acc[q] = 0.0f;
      }
#pragma unroll
      for (int q = 0; q < V; ++q) acc[q] += x[b][q];
    }
  }
  if (!a.next_keys) {
    if (cur != NONE) to_table(cur);
    return;
  }
  if (head) {
    to_next(2 * g, cur);
    to_next(2 * g + 1, NONE);
  } else {
    to_next(2 * g + 1, cur);
  }
}

// One workgroup's sorted entries: groups of `width` lanes (group g, lane l) walk equal shares beg .. end of them, BATCH loads at a time.  A
// run that ends inside a share is done; the first and the last run of a share meet their neighbours' in LDS (edge: [group][first |
// last][lane][V], edge_key), where the share in which a run starts adds up the rest.  key(e): the row of entry e or NONE; load(e, x): its
// values in this lane's columns; finish(row, sums).  Every thread of the workgroup calls it; `on`: the lane has columns (lane 0 of a
// group does if any does).
template <int V, int BATCH, typename KEY, typename LOAD, typename FINISH>
__device__ __forceinline__ void add_shares(int g, int groups, int l, int width, int beg, int end, bool on, float* edge, unsigned* edge_key,
                                           const KEY& key, const LOAD& load, const FINISH& finish) {
  float acc[V];
#pragma unroll
  for (int q = 0; q < V; ++q) acc[q] = 0.0f;
  auto keep = [&](int slot, unsigned k) {
    if (l == 0) edge_key[slot] = k;
#pragma unroll
    for (int q = 0; q < V; ++q) edge[(slot * width + l) * V + q] = acc[q];
  };
  if (on) {
    unsigned cur = NONE;
    bool head = true;
    for (int e = beg; e < end; e += BATCH) {
      unsigned k[BATCH];
      float x[BATCH][V];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        k[b] = e + b < end ? key(e + b) : NONE;
        if (e + b < end) load(e + b, x[b]);
      }
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        if (k[b] == NONE) continue;
        if (k[b] != cur) {
          if (cur != NONE) {
            if (head) keep(2 * g, cur);
            else finish(cur, acc);
            head = false;
          }
          cur = k[b];
#pragma unroll
          for (int q = 0; q < V; ++q) acc[q] = 0.0f;
        }
#pragma unroll
        for (int q = 0; q < V; ++q) acc[q] += x[b][q];
      }
    }
    if (head) {
      keep(2 * g, cur);
      if (l == 0) edge_key[2 * g + 1] = NONE;
    } else {
      keep(2 * g + 1, cur);
    }
  }
  __syncthreads();
  if (!on) return;
  for (int slot = 2 * g; slot < 2 * g + 2; ++slot) {
    const unsigned k = edge_key[slot];
    bool starts = k != NONE;
    if (starts) {                                        // ... unless the entry before it is of the same row
      int s = slot - 1;
      while (s >= 0 && edge_key[s] == NONE) --s;
      starts = s < 0 || edge_key[s] != k;
    }
    if (!starts) continue;
#pragma unroll
    for (int q = 0; q < V; ++q) acc[q] = edge[(slot * width + l) * V + q];
    bool open = true;
    for (int s0 = slot + 1; open && s0 < 2 * groups; s0 += BATCH) {
      unsigned ks[BATCH];
      float x[BATCH][V];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int s = s0 + b < 2 * groups ? s0 + b : slot;
        ks[b] = s0 + b < 2 * groups ? edge_key[s] : NONE;
#pragma unroll
        for (int q = 0; q < V; ++q) x[b][q] = edge[(s * width + l) * V + q];
      }
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        open = open && (ks[b] == NONE || ks[b] == k);
        if (open && ks[b] == k)
#pragma unroll
          for (int q = 0; q < V; ++q) acc[q] += x[b][q];
      }
    }
    finish(k, acc);
  }
}

// The last level: at most TAIL entries, 8 vectors of the rows per workgroup.  (Levels of RUN1 down to one run instead: 5 us each.)
template <typename T, int V>
__global__ __launch_bounds__(512) void tail_kernel(const Level a) {
  typedef typename Vec<T, V>::type VT;
  typedef typename Vec<float, V>::type FT;
  __shared__ float edge[2 * 512 * V];
  __shared__ unsigned edge_key[2 * TAIL_GROUPS];
  const int g = threadIdx.x / a.width, l = threadIdx.x % a.width, c = blockIdx.y * a.width + l;
  const bool on = g < TAIL_GROUPS && c < a.cols;
  const ll col = column<V>(c < a.cols ? c : 0, a.d);
  const int share = ((int)a.n + TAIL_GROUPS - 1) / TAIL_GROUPS, beg = g * share, end = beg + share < a.n ? beg + share : (int)a.n;
  auto load = [&](int e, float* x) {
    const FT y = *(const FT*)((const float*)a.rows + (ll)e * a.ldr + col);
#pragma unroll
    for (int q = 0; q < V; ++q) x[q] = at<float, V>(y, q);
  };
  auto finish = [&](unsigned row, const float* acc) {
    VT y;
#pragma unroll
    for (int q = 0; q < V; ++q) put<T, V>(y, q, a.scale * acc[q]);
    *(VT*)((T*)a.out + (ll)row * a.ldo + col) = y;
  };
  add_shares<V, 8>(g, TAIL_GROUPS, l, a.width, beg, end, on, edge, edge_key, [&](int e) { return a.keys[e]; }, load, finish);
}

// ---- low tables --------------------------------------------------------------------------------------------------------------
struct Low {
  const void* index;
  int index64;
  ll n, ldr, ldo;
  int v, d, cols, width;
  float scale;
  const void* rows;
  void* out;
  float* part;                   // [workgroups][v][d]; null: one workgroup, which writes the table
};

// 512 tokens: counting sort by row in LDS (stable), then their sums.  blockIdx.y: 64 vectors of the row each.
template <typename T, int V>
__global__ __launch_bounds__(LOW_TOKENS) void low_kernel(const Low a) {
  typedef typename Vec<T, V>::type VT;
  typedef typename Vec<float, V>::type FT;
  constexpr int WAVES = LOW_TOKENS / 64, GROUPS = 32;
  __shared__ unsigned cnt[WAVES][256];
  __shared__ unsigned buf[256];
  __shared__ unsigned start[257];
  __shared__ unsigned short order[LOW_TOKENS], sorted[LOW_TOKENS];
  __shared__ float edge[2 * LOW_TOKENS * V];             // [group][first | last][lane][V]
  __shared__ unsigned edge_key[2 * GROUPS];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (tid < 256)
    for (int w = 0; w < WAVES; ++w) cnt[w][tid] = 0;
  __syncthreads();
  const ll tok0 = (ll)blockIdx.x * LOW_TOKENS;
  const bool live = tok0 + tid < a.n;
  const unsigned key = live ? key_of(a.index, a.index64, tok0 + tid, a.v) : 0;
  ull peers = __ballot(live);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const ull on = __ballot((key >> b) & 1);
    peers &= (key >> b) & 1 ? on : ~on;
  }
  const unsigned before = (unsigned)__popcll(peers & ((1ull << lane) - 1));
  if (live && before == 0) cnt[wave][key] = (unsigned)__popcll(peers);
  __syncthreads();
  unsigned own = 0;
  if (tid < 256)
    for (int w = 0; w < WAVES; ++w) own += cnt[w][tid];
  // exclusive scan of the 256 counts by the first four waves
  unsigned in = own;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const unsigned y = __shfl_up(in, d);
    if (lane >= d) in += y;
  }
  if (tid < 256 && lane == 63) buf[wave] = in;
  __syncthreads();
  if (tid < 256) {
    unsigned c = in - own + (wave > 0 ? buf[0] : 0) + (wave > 1 ? buf[1] : 0) + (wave > 2 ? buf[2] : 0);
    start[tid] = c;
    if (tid == 255) start[256] = c + own;
    for (int w = 0; w < WAVES; ++w) {
      const unsigned x = cnt[w][tid];
      cnt[w][tid] = c;
      c += x;
    }
  }
  __syncthreads();
  if (live) {
    const unsigned to = cnt[wave][key] + before;
    order[to] = (unsigned short)tid;
    sorted[to] = (unsigned short)key;
  }
  __syncthreads();
  const int named = (int)start[a.v];                     // tokens that name a row (the others have key v and come last)
  const int groups = LOW_TOKENS / a.width < GROUPS ? LOW_TOKENS / a.width : GROUPS, share = LOW_TOKENS / groups;
  const int g = tid / a.width, l = tid % a.width, c = blockIdx.y * a.width + l;
  const bool on = g < groups && c < a.cols;
  const ll col = column<V>(c < a.cols ? c : 0, a.d);
  auto finish = [&](unsigned row, const float* acc) {
    if (a.part) {
      FT y;
#pragma unroll
      for (int q = 0; q < V; ++q) put<float, V>(y, q, acc[q]);
      *(FT*)(a.part + ((ll)blockIdx.x * a.v + row) * a.d + col) = y;
    } else {
      VT y;
#pragma unroll
      for (int q = 0; q < V; ++q) put<T, V>(y, q, a.scale * acc[q]);
      *(VT*)((T*)a.out + row * a.ldo + col) = y;
    }
  };
  auto load = [&](int e, float* x) {
    const VT y = *(const VT*)((const T*)a.rows + (tok0 + order[e]) * a.ldr + col);
#pragma unroll
    for (int q = 0; q < V; ++q) x[q] = at<T, V>(y, q);
  };
  const int beg = g * share, end = beg + share < named ? beg + share : named;
  add_shares<V, 8>(g, groups, l, a.width, beg, end, on, edge, edge_key, [&](int e) { return (unsigned)sorted[e]; }, load, finish);
  if (on) {                                              // rows that none of these tokens names
    const float acc[V] = {};
    for (int row = g; row < a.v; row += groups)
      if (start[row] == start[row + 1]) finish(row, acc);
  }
}

// 64 elements of the table per workgroup, each as 16 sums over every 16th partial table, joined in order
template <typename T>
__global__ __launch_bounds__(1024) void low_join_kernel(const Low a, int parts) {
  __shared__ float buf[16][64];
  const int lane = threadIdx.x & 63, slice = threadIdx.x >> 6;
  const ll size = (ll)a.v * a.d, e = (ll)blockIdx.x * 64 + lane;
  float x = 0.0f;
  if (e < size) {
#pragma unroll 8
    for (int p = slice; p < parts; p += 16) x += a.part[p * size + e];
  }
  buf[slice][lane] = x;
  __syncthreads();
  if (slice == 0 && e < size) {
    float sum = 0.0f;
#pragma unroll
    for (int q = 0; q < 16; ++q) sum += buf[q][lane];
    ((T*)a.out)[e / a.d * a.ldo + e % a.d] = (T)(a.scale * sum);
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------------
static ll align256(ll x) { return (x + 255) / 256 * 256; }
// entries per group of the first level: 16 while that leaves few groups (8 192 x 256 bf16 40 us against 45 with 32), 32 beyond (40 000 x 1 024
// bf16 74 against 76, 46 602 x 723 f16 56 against 61)
static int first_run(ll n) { return n <= 8192 ? 16 : 32; }
static ll groups(ll n, int level) { const int run = level == 0 ? first_run(n) : RUN1; return (n + run - 1) / run; }
static ll low_parts(ll n) { return (n + LOW_TOKENS - 1) / LOW_TOKENS; }
// (both sides measured at the top)
static bool low(ll n, ll v, ll d) { return v <= LOW && (low_parts(n) <= 1 || 4 * low_parts(n) * v * d <= (8 << 20)); }

struct Layout {
  ll keys[2], perm[2], hist, total, lkeys[2], lrows[2], bytes;
};

static Layout layout(ll n, ll d) {
  Layout l;
  ll at = 0;
  auto take = [&](ll bytes) {
    const ll here = at;
    at += align256(bytes);
    return here;
  };
  for (int b = 0; b < 2; ++b) {
    l.keys[b] = take(4 * n);
    l.perm[b] = take(4 * n);
  }
  l.hist = take(1024 * ((n + TILE - 1) / TILE));
  l.total = take(1024);
  const ll n1 = 2 * groups(n, 0), n2 = 2 * groups(n1, 1);
  l.lkeys[0] = take(4 * n1);
  l.lrows[0] = take(4 * n1 * d);
  l.lkeys[1] = take(4 * n2);
  l.lrows[1] = take(4 * n2 * d);
  l.bytes = at;
  return l;
}

long long backward_workspace_bytes(long long n, long long v, long long d) {
  if (n <= 0) return 0;
  if (low(n, v, d)) return low_parts(n) > 1 ? 4 * low_parts(n) * v * d : 0;
  return layout(n, d).bytes;
}

// a grid's threads are counted in 32 bits: larger ranges loop
static dim3 blocks(ll n) { return dim3((unsigned)(n < (1 << 22) ? n : (1 << 22))); }

template <typename T, int V> static int forward_as(const Call& c, hipStream_t st) {
  const ll cols = (c.d + V - 1) / V;
  lookup_kernel<T, V><<<blocks((c.n * cols + 255) / 256), 256, 0, st>>>(c.index, c.index64, c.n, c.v, (int)cols, (int)c.d, c.scale,
                                                                                  (const T*)c.src, c.lds, (T*)c.dst, c.ldd);
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

template <typename T, int V> static int low_as(const Call& c, hipStream_t st) {
  Low a;
  a.index = c.index;
  a.index64 = c.index64;
  a.n = c.n;
  a.ldr = c.lds;
  a.ldo = c.ldd;
  a.v = (int)c.v;
  a.d = (int)c.d;
  a.cols = (int)((c.d + V - 1) / V);
  a.width = 1;
  while (a.width < a.cols && a.width < 64) a.width *= 2;
  a.scale = c.scale;
  a.rows = c.src;
  a.out = c.dst;
  const ll parts = c.n > 0 ? low_parts(c.n) : 1;
  a.part = parts > 1 ? (float*)c.ws : nullptr;
  low_kernel<T, V><<<dim3((unsigned)parts, (unsigned)((a.cols + a.width - 1) / a.width)), LOW_TOKENS, 0, st>>>(a);
  if (parts > 1) low_join_kernel<T><<<dim3((unsigned)((c.v * c.d + 63) / 64)), 1024, 0, st>>>(a, (int)parts);
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

template <typename T, int V> static int backward_as(const Call& c, hipStream_t st) {
  const ll need = backward_workspace_bytes(c.n, c.v, c.d);
  if (need > 0 && (!c.ws || c.ws_bytes < need)) return -3;
  if (low(c.n, c.v, c.d)) return low_as<T, V>(c, st);
  const int cols = (int)((c.d + V - 1) / V);
  const Layout l = layout(c.n, c.d);
  char* ws = (char*)c.ws;
  unsigned *keys[2], *perm[2];
  for (int b = 0; b < 2; ++b) {
    keys[b] = (unsigned*)(ws + l.keys[b]);
    perm[b] = (unsigned*)(ws + l.perm[b]);
  }
  int cur = 0;
  if (c.n > 0 && c.n <= SMALL) {
    sort_small_kernel<<<1, 1024, 0, st>>>(c.index, c.index64, (int)c.n, c.v, keys[0], perm[0]);
  } else if (c.n > 0) {
    Pass p;
    p.index = c.index;
    p.index64 = c.index64;
    p.n = c.n;
    p.v = c.v;
    p.hist = (unsigned*)(ws + l.hist);
    p.total = (unsigned*)(ws + l.total);
    p.tiles = (c.n + TILE - 1) / TILE;
    int bits = 1;
    while (bits < 32 && (c.v >> bits) != 0) ++bits;           // keys 0 .. v
    for (p.shift = 0; p.shift < bits; p.shift += 8) {
      p.first = p.shift == 0;
      p.keys_in = keys[1 - cur];
      p.perm_in = perm[1 - cur];
      p.keys_out = keys[cur];
      p.perm_out = perm[cur];
      hist_kernel<<<dim3((unsigned)p.tiles), 256, 0, st>>>(p);
      if (p.tiles > FOLD) scan_kernel<<<256, 256, 0, st>>>(p);
      scatter_kernel<<<dim3((unsigned)p.tiles), 256, 0, st>>>(p);
      cur = 1 - cur;
    }
    cur = 1 - cur;
  }
  Level a;
  a.v = c.v;
  a.d = (int)c.d;
  a.cols = cols;
  a.width = 1;
  while (a.width < cols && a.width < 64) a.width *= 2;
  a.scale = c.scale;
  a.out = c.dst;
  a.ldo = c.ldd;
  const unsigned wide = (unsigned)((cols + a.width - 1) / a.width);
  ll n = c.n;
  for (int level = 0;; ++level) {
    const ll g = groups(n, level);
    a.n = n;
    a.keys = level == 0 ? keys[cur] : (const unsigned*)(ws + l.lkeys[(level - 1) & 1]);
    a.perm = perm[cur];
    a.rows = level == 0 ? c.src : (const void*)(ws + l.lrows[(level - 1) & 1]);
    a.ldr = level == 0 ? c.lds : c.d;
    if (level > 0 && n <= TAIL) {
      while (a.width > 512 / TAIL_GROUPS) a.width /= 2;
      tail_kernel<T, V><<<dim3(1, (unsigned)((cols + a.width - 1) / a.width)), 512, 0, st>>>(a);
      break;
    }
    a.run = level == 0 ? first_run(n) : RUN1;
    a.next_keys = g <= 1 ? nullptr : (unsigned*)(ws + l.lkeys[level & 1]);
    a.next_rows = (float*)(ws + l.lrows[level & 1]);
    const int per = 256 / a.width;
    a.sum_blocks = (unsigned)((g + per - 1) / per);
    if (level == 0) {
      const ll clear = (c.v + 63) / 64 < (1 << 20) ? (c.v + 63) / 64 : (1 << 20);      // 16 rows per wave
      sum_kernel<T, V, true><<<dim3(a.sum_blocks + (unsigned)clear, wide), 256, 0, st>>>(a);
    } else {
      sum_kernel<T, V, false><<<dim3(a.sum_blocks, wide), 256, 0, st>>>(a);
    }
    if (g <= 1) break;
    n = 2 * g;
  }
  return hipGetLastError() == hipSuccess ? 0 : -2;
}

int forward(const Call& c, hipStream_t st) {
  const bool vec = c.d >= (c.dtype == nrhlin::F32 ? 4 : 8);      // rows of at least 16 bytes
  if (c.dtype == nrhlin::F32) return vec ? forward_as<float, 4>(c, st) : forward_as<float, 1>(c, st);
  if (c.dtype == nrhlin::F16) return vec ? forward_as<_Float16, 8>(c, st) : forward_as<_Float16, 1>(c, st);
  return vec ? forward_as<__bf16, 8>(c, st) : forward_as<__bf16, 1>(c, st);
}

int backward(const Call& c, hipStream_t st) {
  const bool vec = c.d >= (c.dtype == nrhlin::F32 ? 4 : 8);      // rows of at least 16 bytes
  if (c.dtype == nrhlin::F32) return vec ? backward_as<float, 4>(c, st) : backward_as<float, 1>(c, st);
  if (c.dtype == nrhlin::F16) return vec ? backward_as<_Float16, 8>(c, st) : backward_as<_Float16, 1>(c, st);
  return vec ? backward_as<__bf16, 8>(c, st) : backward_as<__bf16, 1>(c, st);
}

}  // namespace nrhemb
