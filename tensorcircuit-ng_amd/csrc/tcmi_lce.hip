// Softmax cross entropy of a linear head over many classes, without its logits:
//   l[t][v] = <h_t, w_v> + b_v,   loss_t = log sum_v exp l[t][v] - l[t][y_t],
//   P = exp(l - lse) - onehot(y),  dh_t = r_t P_t w,  dw = (r P)^T h,  db = P^T r      (r_t = dloss_t, 0 for ignored rows)
// Forward: one product on the matrix pipe whose epilogue keeps, per row and tile of classes, the running maximum and the
// sum of exponentials (T x V / 128 pairs instead of T x V logits).  Backward: per piece of the classes the logits are
// formed again, become P (f16, row-major and transposed) in the epilogue, and two products use it while it is there.
// Bound by the matrix pipe: 2 T D V multiply-adds forward, 6 T D V more backward.
//
// Operand precision.  bf16 / f16 heads: the logits from the inputs as they are (products exact in the f32 accumulator);
// P is one f16 piece (2^-11 relative; bf16 would cost 2^-8, two pieces a second product), h and w enter the two gradient
// products as f16, each feature under a power of two taken from its largest value (exact down to 2^-29 of it for 11 bits).
// f32 heads: two f16 pieces everywhere (2^-22 down to 2^-17 of what the scale was taken from, 2^-39 of it below), three
// products per product.  The scales: h and w in the logits per row, in the gradients per feature, P for dh 2^14 (P lies in [-1, 1]),
// (r P)^T for dw per class.  So a logit is off by 2^-22 sum |h||w| of the rows' largest, an entry of dw by that share of its class's
// largest r P times its feature's largest h, of dh by that of the largest w of its feature.
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/tcmi.h"
#include "tcmi_mm16.h"

extern "C" int tcmi_set_error_(int code, const char* msg);

namespace tcmi {
namespace lce {

using namespace mm16;

constexpr int PEXP = 14;                     // P lies in [-1, 1]
constexpr float PSCALE = 1 << PEXP;
constexpr int PARTS = 1024;                   // workgroups of a pass over an operand

template <int DT>
__device__ __forceinline__ float fetch(const void* p, long long at) {
  if constexpr (DT == TCMI_F32) return ((const float*)p)[at];
  else if constexpr (DT == TCMI_F16) return (float)((const f16*)p)[at];
  else return (float)((const __bf16*)p)[at];
}
__device__ __forceinline__ float fetch_any(const void* p, int dt, long long at) {
  return dt == TCMI_F32 ? ((const float*)p)[at] : dt == TCMI_F16 ? (float)((const f16*)p)[at] : (float)((const __bf16*)p)[at];
}
__device__ __forceinline__ void put(void* p, int dt, long long at, float v) {
  if (dt == TCMI_F32) ((float*)p)[at] = v;
  else if (dt == TCMI_F16) ((f16*)p)[at] = (f16)v;
  else ((__bf16*)p)[at] = (__bf16)v;
}

// four neighbouring elements; vec: the address is aligned for one load
template <int DT>
__device__ __forceinline__ f32x4 fetch4(const void* p, long long at, bool vec) {
  if (vec) {
    if constexpr (DT == TCMI_F32) return *reinterpret_cast<const f32x4*>((const float*)p + at);
    else if constexpr (DT == TCMI_F16) return __builtin_convertvector(*reinterpret_cast<const f16x4*>((const f16*)p + at), f32x4);
    else return __builtin_convertvector(*reinterpret_cast<const bf16x4*>((const __bf16*)p + at), f32x4);
  }
  return f32x4{fetch<DT>(p, at), fetch<DT>(p, at + 1), fetch<DT>(p, at + 2), fetch<DT>(p, at + 3)};
}

// four elements from column c of a row of `cols`, zero behind its end
template <int DT>
__device__ __forceinline__ f32x4 fetch_row4(const void* p, long long row, int c, int cols, bool vec) {
  if (c + 3 < cols) return fetch4<DT>(p, row + c, vec);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 3; ++k)
    if (c + k < cols) v[k] = fetch<DT>(p, row + c + k);
  return v;
}

// power of two that brings `top` into [2^14, 2^15); 1 for zero and for what is not finite
__device__ __forceinline__ float scale_of(float top) {
  const unsigned e = __float_as_uint(top) >> 23;
  if (e == 0 || e >= 255) return 1.f;
  const int k = 14 - ((int)e - 127);
  return ldexpf(1.f, k > 100 ? 100 : k < -100 ? -100 : k);
}

// One pass over the rows of h and of w, a wave per row, bound by its reads (and writes, where a copy is made):
//   out   the row with k padded.  16-bit types are copied; f32 rows are cut into two pieces under a power of two per row, whose
//         inverse goes to inv[row] (the second read of the row comes from the cache).
//   r     h only: the factor of row t in the gradients, from its target and dloss.
//   top   cleared, for top_kernel: a word per feature and one more.
struct Operand {
  const void* src;
  long long rs;
  int rows, cols, colsp, vec, blocks;
  f16* out;
  float* inv;
};

struct Prep {
  Operand h, w;
  const long long* y;
  long long ignore;
  const float *dloss, *count;
  int per_row;
  float* r;                      // null: no factors (forward)
  unsigned* top;
  int tops;
};

template <int DT>
__global__ __launch_bounds__(256) void prep_kernel(Prep a) {
  for (int k = blockIdx.x * 256 + threadIdx.x; k < a.tops; k += gridDim.x * 256) a.top[k] = 0;
  const bool is_h = (int)blockIdx.x < a.h.blocks;
  const Operand& o = is_h ? a.h : a.w;
  const int block = is_h ? blockIdx.x : blockIdx.x - a.h.blocks, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int row = block * 4 + wave; row < o.rows; row += o.blocks * 4) {
    const long long in = row * o.rs;
    if (is_h && a.r) {
      float f = a.per_row ? a.dloss[row] : a.count ? a.dloss[0] / a.count[0] : a.dloss[0];
      if (a.y[row] == a.ignore) f = 0.f;
      if (lane == 0) a.r[row] = f;
    }
    if (!o.out) continue;
    if constexpr (DT == TCMI_F32) {
      float t = 0.f;
#pragma unroll 4
      for (int c = 4 * lane; c < o.cols; c += 256) {
        const f32x4 v = fetch_row4<DT>(o.src, in, c, o.cols, o.vec);
        t = fmaxf(fmaxf(fmaxf(t, fabsf(v[0])), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
      }
#pragma unroll
      for (int k = 32; k > 0; k >>= 1) t = fmaxf(t, __shfl_xor(t, k));
      const float s = scale_of(t);
      f16* q = o.out + (long long)row * 2 * o.colsp;
      for (int c = 4 * lane; c < o.colsp; c += 256) {
        const f32x4 v = fetch_row4<DT>(o.src, in, c, o.cols, o.vec);
        f16x4 hi, lo;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f16 h, l;
          two_pieces(v[k] * s, h, l);
          hi[k] = h;
          lo[k] = l;
        }
        store_four<2>(q, c, hi, lo);
      }
      if (lane == 0) o.inv[row] = 1.f / s;
    } else {
      typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
      const unsigned short* p = (const unsigned short*)o.src + in;
      unsigned short* q = (unsigned short*)o.out + (long long)row * o.colsp;
      for (int c = 4 * lane; c < o.colsp; c += 256) {
        u16x4 v = {0, 0, 0, 0};
        if (o.vec && c + 3 < o.cols) {
          v = *reinterpret_cast<const u16x4*>(p + c);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (c + k < o.cols) v[k] = p[c + k];
        }
        *reinterpret_cast<u16x4*>(q + c) = v;
      }
    }
  }
}

// Largest |x| of every feature, over the rows that count, and of the whole operand behind them: the gradients' products take
// each feature under its own power of two.  A thread holds four features and walks down the rows; workgroups join by atomic
// maxima (of non-negative floats as whole numbers: the order does not matter).  h and w in one launch, at most 64 shares of
// the rows: 512 of them waited 60 us for each other's atomics.  Bound by its reads.
struct Top {
  const void* src;
  long long rs;
  int rows, cols, vec, lanes, panels, blocks;        // lanes: threads along a row; panels: of 4 lanes features; blocks = panels * shares of the rows
  const float* r;                // rows with r = 0 do not count (null: all do)
  unsigned* top;                 // [cols + 1]
};

constexpr int TOP_THREADS = 1024, TOP_SHARES = 64;

template <int DT>
__global__ __launch_bounds__(TOP_THREADS) void top_kernel(Top x, Top y) {
  __shared__ f32x4 red[TOP_THREADS];
  const bool first = (int)blockIdx.x < x.blocks;
  const Top& a = first ? x : y;
  const int block = first ? blockIdx.x : blockIdx.x - x.blocks, share = block / a.panels, shares = a.blocks / a.panels;
  const int per = TOP_THREADS / a.lanes, lane = threadIdx.x % a.lanes, c = (block % a.panels * a.lanes + lane) * 4;
  f32x4 t = {0.f, 0.f, 0.f, 0.f};
  const bool whole = a.vec && c + 3 < a.cols;
  if (c < a.cols)
    for (int row = share * per + threadIdx.x / a.lanes; row < a.rows; row += 8 * shares * per) {
      f32x4 v[8];                                    // eight rows under way at once; behind the last one that one again
      float f[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const long long at = min((long long)row + (long long)u * shares * per, a.rows - 1ll);
        v[u] = whole ? fetch4<DT>(a.src, at * a.rs + c, true) : fetch_row4<DT>(a.src, at * a.rs, c, a.cols, false);
        f[u] = a.r ? a.r[at] : 1.f;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u)
#pragma unroll
        for (int k = 0; k < 4; ++k) t[k] = fmaxf(t[k], f[u] == 0.f ? 0.f : fabsf(v[u][k]));
    }
  red[threadIdx.x] = t;
  __syncthreads();
  if ((int)threadIdx.x >= a.lanes || c >= a.cols) return;
  for (int q = 1; q < per; ++q) {
    const f32x4 v = red[threadIdx.x + q * a.lanes];
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = fmaxf(t[k], v[k]);
  }
  float all = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (c + k < a.cols) {
      atomicMax(a.top + c + k, __float_as_uint(t[k]));
      all = fmaxf(all, t[k]);
    }
  if (all == INFINITY) atomicMax(a.top + a.cols, __float_as_uint(all));      // only whether it is finite matters
}

// the power of two that brings a feature's largest value into [2^14, 2^15)
__device__ __forceinline__ int feature_exp(unsigned top) { return 14 + 127 - (int)(top >> 23); }

// out[c][row] = src[row][c] 2^exp[c] as f16 pieces (two for f32), rows padded with zeros.  A row whose factor r is zero gives
// zero whatever it holds; an infinity anywhere else makes everything NaN (no scale would hold the rest beside it).
// 64 x 64 tiles through LDS, four elements a thread on both sides; h and w in one launch.
struct Turn {
  const void* src;
  long long rs;
  int rows, cols, rowsp, vec, tx, tiles;
  const float* r;
  const unsigned* top;
  f16* out;
};

template <int DT>
__global__ __launch_bounds__(256) void turn_kernel(Turn x, Turn y) {
  constexpr int P = DT == TCMI_F32 ? 2 : 1;
  __shared__ float tile[64][65];
  const bool first = (int)blockIdx.x < x.tiles;
  const Turn& a = first ? x : y;
  const int tid = threadIdx.x, block = first ? blockIdx.x : blockIdx.x - x.tiles;
  const bool lost = a.top[a.cols] != 0;            // an infinity
  const int r0 = block % a.tx * 64, c0 = block / a.tx * 64, u = (tid & 15) * 4, w = tid >> 4;
  int ex[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) ex[e] = c0 + u + e < a.cols ? feature_exp(a.top[c0 + u + e]) : 0;
#pragma unroll
  for (int k = w; k < 64; k += 16) {
    const int row = r0 + k;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    if (row < a.rows) {
      if (!a.r || a.r[row] != 0.f) {
        v = fetch_row4<DT>(a.src, row * a.rs, c0 + u, a.cols, a.vec);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = lost ? NAN : ldexpf(v[e], ex[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) tile[k][u + e] = v[e];
  }
  __syncthreads();
#pragma unroll
  for (int k = w; k < 64; k += 16) {
    const int c = c0 + k, row = r0 + u;
    if (c < a.cols && row < a.rowsp) {
      f16x4 hi, lo;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        f16 h, l;
        two_pieces(tile[u + e][k], h, l);
        hi[e] = h;
        lo[e] = l;
      }
      store_four<P>(a.out + (long long)c * P * a.rowsp, row, hi, lo);
    }
  }
}

// logits of a tile: acc times the rows' scales (two pieces only) plus the bias
struct Logits {
  const float *hs, *ws;          // f32: inverse scales of the rows of h and of w
  const void* bias;              // null: none
  int dtype;
  int v0;                        // first class of the piece
};

template <int P, class T>
__device__ __forceinline__ void logits(const Logits& q, const Args& g, int m0, int n0, f32x4 (&acc)[T::MI][T::NI]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / T::WN, wn = wave % T::WN;
  if constexpr (P == 2) {
    float rs[T::MI];
#pragma unroll
    for (int i = 0; i < T::MI; ++i) rs[i] = q.hs[min(m0 + wm * T::MI * 16 + i * 16 + (lane & 15), g.M - 1)];
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      const int col = n0 + wn * T::NI * 16 + j * 16 + 4 * (lane >> 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float cs = q.ws[min(col + r, g.N - 1) + q.v0];
#pragma unroll
        for (int i = 0; i < T::MI; ++i) acc[i][j][r] *= rs[i] * cs;
      }
    }
  }
  if (q.bias) {
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      const int col = n0 + wn * T::NI * 16 + j * 16 + 4 * (lane >> 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float cb = fetch_any(q.bias, q.dtype, min(col + r, g.N - 1) + q.v0);
#pragma unroll
        for (int i = 0; i < T::MI; ++i) acc[i][j][r] += cb;
      }
    }
  }
  if (n0 + T::BN > g.N) {                            // the last tile of classes
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      const int col = n0 + wn * T::NI * 16 + j * 16 + 4 * (lane >> 4);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r >= g.N)
#pragma unroll
          for (int i = 0; i < T::MI; ++i) acc[i][j][r] = -INFINITY;
    }
  }
}

// where a row's target lies among the piece's columns; a column that does not exist if it is elsewhere
__device__ __forceinline__ int local_target(long long y, int v0, int n) {
  const long long k = y - v0;
  return k >= 0 && k < n ? (int)k : -8;
}

// forward: per row the tile's maximum and sum of exponentials, and the target's logit where it lies in the tile
template <int P>
struct EpiLse {
  static constexpr bool TILE = true, FOUR = false;
  template <class T>
  static constexpr int lds() { return T::WN * T::BM * 8; }
  Logits q;
  float2* part;                  // [T][tiles of classes]
  float* target;                 // [T]
  const long long* y;
  template <class T>
  __device__ void tile(const Args& g, int m0, int n0, int, bool, char* lds, f32x4 (&acc)[T::MI][T::NI]) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / T::WN, wn = wave % T::WN;
    const int c0 = n0 + wn * T::NI * 16 + 4 * (lane >> 4);
    float2* stat = reinterpret_cast<float2*>(lds);                    // [WN][BM]
    logits<P, T>(q, g, m0, n0, acc);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < T::MI; ++i) {
      const int rl = wm * T::MI * 16 + i * 16 + (lane & 15), row = m0 + rl;
      const int yl = row < g.M ? local_target(y[row], 0, g.N) : -8;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < T::NI; ++j) {
        const f32x4 x = acc[i][j];
        top = fmaxf(fmaxf(fmaxf(top, x[0]), x[1]), fmaxf(x[2], x[3]));
        const int k = yl - c0 - 16 * j;
        if ((unsigned)k < 4u) target[row] = k == 0 ? x[0] : k == 1 ? x[1] : k == 2 ? x[2] : x[3];
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float at = top == -INFINITY ? 0.f : top;                  // a row of -inf has sum 0, not NaN
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < T::NI; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum += __expf(acc[i][j][r] - at);
      sum += __shfl_xor(sum, 16);
      sum += __shfl_xor(sum, 32);
      if (lane < 16) stat[wn * T::BM + rl] = make_float2(top, sum);
    }
    __syncthreads();
    for (int rl = threadIdx.x; rl < T::BM; rl += T::THREADS) {
      if (m0 + rl >= g.M) continue;
      float2 a = stat[rl];
#pragma unroll
      for (int k = 1; k < T::WN; ++k) {
        const float2 b = stat[k * T::BM + rl];
        const float top = fmaxf(a.x, b.x), at = top == -INFINITY ? 0.f : top;
        a = make_float2(top, a.y * __expf(a.x - at) + b.y * __expf(b.x - at));
      }
      part[(long long)(m0 + rl) * g.tn + n0 / T::BN] = a;
    }
  }
};

// Up to 16 rows without a gradient (evaluating or serving single samples; before a gradient the logits of forward and
// backward have to come from the same product, or exp(l - lse) - 1 of a certain row is their difference): w is read once,
// straight into the matrix instructions, whatever its alignment, and no operand is copied.  A wave takes 32 classes at a time
// and keeps its rows' running maximum and sum of exponentials; f32 heads use the f32 matrix instruction (exact products).
// Bound by the read of w: 10 x 3466 x 59851 bf16 124 us (3.3 TB/s; with copies and 128 x 128 tiles 436), 16 x 4096 x 65536
// f32 256 us (4.2 TB/s; 707), the same in bf16, which the tiles read in place, 130 us either way.
constexpr int FEW_ROWS = 16, FEW_BLOCKS = 1024;

template <int DT>
struct FewArgs {
  const void *h, *w, *bias;
  long long hrs, wrs;
  int T, D, V;
  const long long* y;
  float2* part;                  // [T][gridDim.x]
  float* target;
};

// 16 bytes of a row from element c, zero behind its end; the row may start anywhere
template <class V, class E>
__device__ __forceinline__ V few_load(const E* row, int c, int cols) {
  constexpr int N = 16 / sizeof(E);
  V v;
  if (c + N <= cols) {
    __builtin_memcpy(&v, row + c, 16);
  } else {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = c + k < cols ? row[c + k] : (E)0.f;
  }
  return v;
}

__device__ __forceinline__ f32x4 few_mul(f16x8 a, f16x8 b, f32x4 c) { return mfma(a, b, c); }
__device__ __forceinline__ f32x4 few_mul(bf16x8 a, bf16x8 b, f32x4 c) { return mfma(a, b, c); }
__device__ __forceinline__ f32x4 few_mul(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
  for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k], b[k], c, 0, 0, 0);
  return c;
}

template <class V, class E, int DT>
__global__ __launch_bounds__(256) void few_kernel(FewArgs<DT> a) {
  constexpr int N = 16 / sizeof(E), K = 16 * N;      // elements of a load, of a pass of four loads
  __shared__ float2 stat[4][FEW_ROWS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const E* h = (const E*)a.h + min(l, a.T - 1) * a.hrs;
  const long long yt = l < a.T ? a.y[l] : -8;
  float top = -INFINITY, sum = 0.f;
  for (int v0 = (blockIdx.x * 4 + wave) * 32; v0 < a.V; v0 += gridDim.x * 128) {
    const E* w0 = (const E*)a.w + (long long)min(v0 + l, a.V - 1) * a.wrs;
    const E* w1 = (const E*)a.w + (long long)min(v0 + 16 + l, a.V - 1) * a.wrs;
    f32x4 acc[2] = {};
    for (int k = 0; k < a.D; k += K) {
      V x[4], p[4], q[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int c = k + (4 * u + g) * N;            // the four lane groups read 64 neighbouring bytes of a row
        p[u] = few_load<V, E>(w0, c, a.D);
        q[u] = few_load<V, E>(w1, c, a.D);
        x[u] = few_load<V, E>(h, c, a.D);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        acc[0] = few_mul(p[u], x[u], acc[0]);
        acc[1] = few_mul(q[u], x[u], acc[1]);
      }
    }
    // the lane holds classes v0 + 16 t + 4 g + r of row l
    float most = top;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int v = v0 + 16 * t + 4 * g + r;
        float x = acc[t][r];
        if (a.bias) x += fetch<DT>(a.bias, min(v, a.V - 1));
        if (v >= a.V) x = -INFINITY;
        if (v == yt && v < a.V) a.target[l] = x;
        acc[t][r] = x;
        most = fmaxf(most, x);
      }
    const float at = most == -INFINITY ? 0.f : most;
    sum *= __expf(top - at);                       // 0 while top is -inf
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) sum += __expf(acc[t][r] - at);
    top = most;
  }
  auto join = [&](float2 b) {
    const float most = fmaxf(top, b.x), at = most == -INFINITY ? 0.f : most;
    sum = sum * __expf(top - at) + b.y * __expf(b.x - at);
    top = most;
  };
#pragma unroll
  for (int o = 16; o < 64; o *= 2) {
    const float2 b = make_float2(__shfl_xor(top, o), __shfl_xor(sum, o));
    join(b);
  }
  if (lane < 16) stat[wave][l] = make_float2(top, sum);
  __syncthreads();
  if (threadIdx.x >= a.T) return;
  float2 s = stat[0][threadIdx.x];
  top = s.x;
  sum = s.y;
#pragma unroll
  for (int k = 1; k < 4; ++k) join(stat[k][threadIdx.x]);
  a.part[(long long)threadIdx.x * gridDim.x + blockIdx.x] = make_float2(top, sum);
}

// the loss of row t from its tiles' statistics, by one wave.  lse: the log sum as a value and its remainder.  In one float it would
// be off by 2^-24 of itself, which of a row that is certain to 1e-6 at logits of 20 leaves nothing in 1 - p; with the
// remainder what is left is the sum's own rounding, 2^-24.
__device__ __forceinline__ float row_loss(const float2* part, int tiles, const float* target, const long long* y, long long ignore, int t,
                                          int V, float* lse) {
  const int lane = threadIdx.x & 63;
  const float2* p = part + (long long)t * tiles;
  float top = -INFINITY, bad = 0.f;
  for (int k = lane; k < tiles; k += 64) {
    top = fmaxf(top, p[k].x);
    if (p[k].y != p[k].y) bad = p[k].y;              // fmaxf drops a NaN, the sums do not
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  const float at = top == -INFINITY ? 0.f : top;
  float sum = bad;
  for (int k = lane; k < tiles; k += 64) sum += p[k].x == -INFINITY ? 0.f : p[k].y * expf(p[k].x - at);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
  const float ls = logf(sum), l = at + ls, b = l - at, rest = fabsf(l) < INFINITY ? (at - (l - b)) + (ls - b) : 0.f;
  if (lane == 0) reinterpret_cast<float2*>(lse)[t] = make_float2(l, rest);
  const long long yt = y[t];
  return yt == ignore ? 0.f : yt < 0 || yt >= V ? NAN : (l - target[t]) + rest;
}

// sum or mean over the rows that count, in f64 and a fixed order; 16 waves
__device__ __forceinline__ void total_of(double s, int c, int mean, float* out, float* count) {
  __shared__ double rs[16];
  __shared__ int rc[16];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    s += __shfl_xor(s, o);
    c += __shfl_xor(c, o);
  }
  if ((threadIdx.x & 63) == 0) {
    rs[threadIdx.x >> 6] = s;
    rc[threadIdx.x >> 6] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    c = 0;
    for (int k = 0; k < 16; ++k) {
      s += rs[k];
      c += rc[k];
    }
    *count = (float)c;
    *out = (float)(mean ? s / c : s);                // no row counts: 0 / 0
  }
}

__global__ __launch_bounds__(256) void rowstat_kernel(const float2* part, int tiles, const float* target, const long long* y,
                                                      long long ignore, int T, int V, float* lse, float* loss) {
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= T) return;
  const float x = row_loss(part, tiles, target, y, ignore, t, V, lse);
  if ((threadIdx.x & 63) == 0) loss[t] = x;
}

__global__ __launch_bounds__(1024) void total_kernel(const float* loss, const long long* y, long long ignore, int T, int mean, float* out,
                                                     float* count) {
  double s = 0.0;
  int c = 0;
  for (int t = threadIdx.x; t < T; t += 1024) {
    s += loss[t];
    c += y[t] != ignore;
  }
  total_of(s, c, mean, out, count);
}

// both in one workgroup, where there is little to read
__global__ __launch_bounds__(1024) void rowstat_total_kernel(const float2* part, int tiles, const float* target, const long long* y,
                                                             long long ignore, int T, int V, float* lse, float* loss, int mean, float* out,
                                                             float* count) {
  double s = 0.0;
  int c = 0;
  for (int t = threadIdx.x >> 6; t < T; t += 16) {
    const float x = row_loss(part, tiles, target, y, ignore, t, V, lse);
    if ((threadIdx.x & 63) == 0) {
      loss[t] = x;
      s += x;
      c += y[t] != ignore;
    }
  }
  total_of(s, c, mean, out, count);
}

// over the 16 lanes of a lane group, the rows of a fragment: by rotations, in registers
template <int N>
__device__ __forceinline__ float turned16(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xf, 0xf, false));
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, turned16<8>(v));
  v = fmaxf(v, turned16<4>(v));
  v = fmaxf(v, turned16<2>(v));
  return fmaxf(v, turned16<1>(v));
}
__device__ __forceinline__ float sum16(float v) {
  v += turned16<8>(v);
  v += turned16<4>(v);
  v += turned16<2>(v);
  return v + turned16<1>(v);
}

// Exponent of a class: P^T's entries leave under 2^(16 k), which brings their largest into [2^-1, 2^15); NO_EXP: all are zero.
constexpr int NO_EXP = 127, EXP_STEP = 16;
__device__ __forceinline__ int exp_of(float top) {
  return top == 0.f ? NO_EXP : (14 + 127 - (int)(__float_as_uint(top) >> 23)) >> 4;
}

// Backward: P as f16 pieces, row-major for dh and transposed for dw, zero in the padding and in ignored rows.
//   dh  a row's entries under 2^14: what falls below 2^-39 is lost, where P of the target, 1 less than a probability, is off by
//       2^-24 in any f32 arithmetic.
//   dw  a class sees its own column of P only, and most classes of a large head are improbable in every row: each class has its
//       own power of two.  The rows' factors are in it too: h stays as it is, and a row of a small factor is small in the classes
//       that others know better, not in all.  A wave takes it from its rows and leaves it in `exps`; class_kernel brings the waves' rows of a class
//       to a common one where they differ (by steps of 2^16, so few do).
// sums: the wave's rows added up, for the bias's gradient.
template <int P>
struct EpiProb {
  static constexpr bool TILE = true, FOUR = false;
  Logits q;
  const float2* lse;
  const long long* y;
  long long ignore;
  int V;
  f16 *p, *pt;                   // [T][P * vp], [classes][P * tp]
  int vp, tp;                    // padded classes of the piece, padded rows
  const float* r;
  signed char* exps;             // [waves' rows][ldv]
  float* sums;                   // the same
  int ldv;
  template <class T>
  static constexpr int lds() { return Transposed<T, P>::BYTES; }
  // P goes out from the registers, eight bytes a lane; P^T through LDS, sixteen (from the registers two, which alone took 50 us
  // of 1021 x 28 x 16384 f32)
  template <class T>
  __device__ void tile(const Args& g, int m0, int n0, int, bool, char* lds, f32x4 (&acc)[T::MI][T::NI]) const {
    const Transposed<T, P> turned{reinterpret_cast<f16*>(lds)};
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / T::WN, wn = wave % T::WN;
    const int cl = wn * T::NI * 16 + 4 * (lane >> 4);
    logits<P, T>(q, g, m0, n0, acc);                 // -inf behind the last class: probability 0
    f32x4 top[T::NI] = {}, sum[T::NI] = {};
#pragma unroll
    for (int i = 0; i < T::MI; ++i) {
      const int row = m0 + wm * T::MI * 16 + i * 16 + (lane & 15);
      const bool in = row < g.M;
      const long long yt = in ? y[row] : ignore;
      const bool keep = in && yt != ignore;
      // a target outside the classes poisons its row
      const float2 l = !keep ? float2{0.f, 0.f} : yt < 0 || yt >= V ? float2{NAN, NAN} : lse[row];
      const float f = keep ? r[row] : 0.f;
      const int yl = keep ? local_target(yt, q.v0, g.N) : -8;
#pragma unroll
      for (int j = 0; j < T::NI; ++j) {
        const f32x4 x = acc[i][j];
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = keep ? __expf((x[r] - l.x) - l.y) : 0.f;        // whatever an ignored row holds
        const int k = yl - n0 - cl - 16 * j;
        if ((unsigned)k < 4u) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (r == k) v[r] = expm1f((x[r] - l.x) - l.y);
        }
        f16x4 vh, vl;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f16 a, b;
          two_pieces(v[r] * PSCALE, a, b);
          vh[r] = a;
          vl[r] = b;
          v[r] = f == 0.f ? 0.f : v[r] * f;
          top[j][r] = fmaxf(top[j][r], fabsf(v[r]));
          sum[j][r] += v[r];
        }
        const int col = n0 + cl + 16 * j;
        if (in && col < vp) store_four<P>(p + (long long)row * P * vp, col, vh, vl);
        acc[i][j] = v;
      }
    }
    const long long line = (long long)(m0 / (T::MI * 16) + wm) * ldv;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < T::NI; ++j) {
      int e[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        e[r] = exp_of(max16(top[j][r]));
        sum[j][r] = sum16(sum[j][r]);
      }
      const int col = n0 + cl + 16 * j;
      if ((lane & 15) == 0 && col < ldv) {
        *reinterpret_cast<unsigned*>(exps + line + col) =
            (e[0] & 255) | (e[1] & 255) << 8 | (e[2] & 255) << 16 | (unsigned)(e[3] & 255) << 24;
        *reinterpret_cast<f32x4*>(sums + line + col) = sum[j];
      }
#pragma unroll
      for (int i = 0; i < T::MI; ++i) {
        f16x4 vh, vl;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f16 a, b;
          two_pieces(ldexpf(acc[i][j][r], e[r] == NO_EXP ? 0 : EXP_STEP * e[r]), a, b);
          vh[r] = a;
          vl[r] = b;
        }
        turned.stage(wm * T::MI * 16 + i * 16 + (lane & 15), cl + 16 * j, vh, vl);
      }
    }
    __syncthreads();
    turned.flush(pt, (long long)P * tp, n0, g.N, m0, tp);
  }
};

// 64 classes a workgroup: the class's exponent, the smallest of its waves' (their largest entry stays where it was, a row's
// further below may lose its last bits, as in any sum with the largest), its rows of P^T brought to it, and the bias's gradient.
// Reads one value per wave's rows and class, rewrites what differs: 8192 x 65536 bf16 a tenth of P^T, 2 x 100 us; 15 us at 1021 x 32768.
template <int P>
__global__ __launch_bounds__(256) void class_kernel(const signed char* exps, const float* sums, int ldv, int chunks, int rows, int n, f16* pt, int tp,
                                                    int* cexp, void* db, int dtype, int v0) {
  __shared__ int lo[4][64];
  __shared__ double part[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, v = blockIdx.x * 64 + lane;        // v < ldv
  int k = NO_EXP;
  double s = 0.0;
  for (int c = wave; c < chunks; c += 4) {
    k = min(k, (int)exps[(long long)c * ldv + v]);
    if (db) s += sums[(long long)c * ldv + v];
  }
  lo[wave][lane] = k;
  part[wave][lane] = s;
  __syncthreads();
  k = min(min(lo[0][lane], lo[1][lane]), min(lo[2][lane], lo[3][lane]));
  if (wave == 0 && v < n) {
    if (cexp) cexp[v] = k == NO_EXP ? 0 : EXP_STEP * k;
    if (db) put(db, dtype, (long long)v0 + v, (float)(part[0][lane] + part[1][lane] + part[2][lane] + part[3][lane]));
  }
  if (!cexp) return;
  for (int c = wave; c < chunks; c += 4) {
    const int e = exps[(long long)c * ldv + v], less = v >= n || e == NO_EXP ? 0 : e - k;
    unsigned long long todo = __ballot(less > 0);
    const int len = P * min(rows, tp - c * rows);
    while (todo) {                                   // four classes at a time, 16 lanes each
      int mine = -1;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (q == lane >> 4 && todo) mine = __ffsll((long long)todo) - 1;
        todo &= todo - 1;
      }
      const int by = -EXP_STEP * __shfl(less, mine < 0 ? 0 : mine);
      if (mine < 0) continue;
      f16* p = pt + (long long)(blockIdx.x * 64 + mine) * P * tp + (long long)P * c * rows;
      for (int i = 4 * (lane & 15); i < len; i += 64) {
        f16x4 x = *reinterpret_cast<f16x4*>(p + i);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = (f16)ldexpf((float)x[r], by);
        *reinterpret_cast<f16x4*>(p + i) = x;
      }
    }
  }
}

// a gradient: value = acc 2^-(rexp or 14, + the feature's) (+ what earlier pieces left in `sum`), kept in `sum` or written out
// times the row's factor
struct EpiGrad {
  static constexpr bool TILE = false, FOUR = true;
  const unsigned* top;           // largest value of each feature of the other operand
  float* sum;                    // f32 [rows][cols] (null: only one piece)
  int first, last;
  const float* r;                // null: 1
  void* out;
  int dtype, cols;
  const int* rexp;               // exponents of the rows of the other operand (null: PSCALE's)
  int vec;                       // rows of `out` and `sum` are aligned for four elements
  __device__ __forceinline__ void four(const Args& g, int, bool, int row, int col, f32x4 v) const {
    if (row >= g.M) return;
    const int ex = rexp ? rexp[row] : PEXP;
    int e4[4];
    if (col + 3 < cols) {
      const uint4 t = *reinterpret_cast<const uint4*>(top + col);
      e4[0] = -(ex + feature_exp(t.x));
      e4[1] = -(ex + feature_exp(t.y));
      e4[2] = -(ex + feature_exp(t.z));
      e4[3] = -(ex + feature_exp(t.w));
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) e4[k] = -(ex + feature_exp(top[min(col + k, cols - 1)]));
    }
    if (vec && col + 3 < cols) {
      const long long at = (long long)row * cols + col;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = ldexpf(v[k], e4[k]);
      if (!first) {
        const f32x4 old = *reinterpret_cast<const f32x4*>(sum + at);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] += old[k];
      }
      if (!last) {
        *reinterpret_cast<f32x4*>(sum + at) = v;
        return;
      }
      if (r) {
        const float f = r[row];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = f == 0.f ? 0.f : v[k] * f;
      }
      if (dtype == TCMI_F32) *reinterpret_cast<f32x4*>((float*)out + at) = v;
      else if (dtype == TCMI_F16) *reinterpret_cast<f16x4*>((f16*)out + at) = __builtin_convertvector(v, f16x4);
      else *reinterpret_cast<bf16x4*>((__bf16*)out + at) = __builtin_convertvector(v, bf16x4);
      return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (col + k >= g.N) continue;
      float x = ldexpf(v[k], e4[k]);
      const long long at = (long long)row * cols + col + k;
      if (!first) x += sum[at];
      if (!last) sum[at] = x;
      else put(out, dtype, at, r ? (r[row] == 0.f ? 0.f : x * r[row]) : x);
    }
  }
};

// ---------------------------------------------------------------------------------------------------------- host side
struct Arena {
  char* base;
  long long used = 0;
  template <class P>
  P* take(long long count) {
    P* p = base ? reinterpret_cast<P*>(base + used) : nullptr;
    used += (count * (long long)sizeof(P) + 255) & ~255ll;
    return p;
  }
};

struct Shape {
  int T, D, V, dtype;
  int P;                         // pieces per operand: 2 for f32
  int dp, tp;                    // padded features, padded rows
  bool few;                      // the forward of up to 16 rows without a gradient
  bool h_direct, w_direct;       // the operand is read where it lies
};

struct Rows {                    // the forward operands when they are not read in place
  f16 *h, *w;
  float *hs, *ws;
};

Rows take_rows(Arena& a, const Shape& s) {
  Rows r{};
  if (!s.h_direct) r.h = a.take<f16>((long long)s.T * s.P * s.dp);
  if (!s.w_direct) r.w = a.take<f16>((long long)s.V * s.P * s.dp);
  if (s.P == 2) {
    r.hs = a.take<float>(s.T);
    r.ws = a.take<float>(s.V);
  }
  return r;
}

struct FwdWork {
  Rows rows;
  float2* part;
  float* target;
};

int few_blocks(const Shape& s) { return s.V >= 128 * FEW_BLOCKS ? FEW_BLOCKS : (s.V + 127) / 128; }

FwdWork take_fwd(Arena& a, const Shape& s) {
  FwdWork w{};
  if (!s.few) w.rows = take_rows(a, s);
  w.part = a.take<float2>((long long)s.T * ((s.V + 63) / 64));          // the narrowest tile of classes is 64 wide
  w.target = a.take<float>(s.T);
  return w;
}

// classes per piece of the backward: P and its transpose take at most about 1 GiB, pieces of equal size
int piece_of(const Shape& s) {
  const long long per = (long long)(s.T + s.tp) * 2 * s.P;
  long long most = (1ll << 30) / per / 256 * 256;
  if (most < 1024) most = 1024;
  if (most > (1 << 20)) most = 1 << 20;            // P's rows within the longest ones a product takes
  const long long pieces = (s.V + most - 1) / most;
  const long long c = ((s.V + pieces - 1) / pieces + 255) / 256 * 256;
  return (int)(c < s.V ? c : s.V);
}

struct BwdWork {
  Rows rows;
  float *r, *sum, *split;
  unsigned* top;                                   // of h's features, then of w's
  f16 *p, *pt, *ht, *wt;                           // P, P^T, h^T, w^T of the piece
  signed char* exps;                               // EpiProb's, and what class_kernel makes of them
  float* sums;
  int* cexp;
};

int tops_of(const Shape& s) { return (s.D + 4) & ~3; }                // a word per feature and one more, aligned for four

int chunks_of(const Shape& s) { return (s.T + 127) / 128 * 4; }        // at most: the fewest rows a wave has are 32


BwdWork take_bwd(Arena& a, const Shape& s) {
  BwdWork w{};
  const long long vc = piece_of(s), vp = kpad(vc, s.P);
  w.rows = take_rows(a, s);
  w.r = a.take<float>(s.T);
  w.top = a.take<unsigned>(2ll * tops_of(s));
  w.sum = vc < s.V ? a.take<float>((long long)s.T * s.D) : nullptr;
  w.split = a.take<float>(PART_BYTES / 4);
  w.p = a.take<f16>(s.T * vp * s.P);
  w.pt = a.take<f16>(vc * s.tp * s.P);
  w.ht = a.take<f16>((long long)s.D * s.tp * s.P);
  w.wt = a.take<f16>(s.D * vp * s.P);
  const long long ldv = (vc + 63) & ~63ll;
  w.exps = a.take<signed char>(chunks_of(s) * ldv);
  w.sums = a.take<float>(chunks_of(s) * ldv);
  w.cexp = a.take<int>(ldv);
  return w;
}

#define TRY(x)                                   \
  do {                                           \
    const hipError_t e_ = (x);                   \
    if (e_ != hipSuccess) return e_;             \
  } while (0)

template <int P, class Epi>
hipError_t run(Args& g, const Epi& e, hipStream_t st) {
  return launch_best<f16x8, P>(g, false, e, st);
}

// the logits' product: 16-bit heads in their own type
template <int P, class Epi>
hipError_t run_logits(Args& g, int dtype, const Epi& e, hipStream_t st) {
  if constexpr (P == 1) {
    if (dtype == TCMI_BF16) return launch_best<bf16x8, 1>(g, false, e, st);
  }
  return run<P>(g, e, st);
}

// whether rows can be read four elements at a time
int vec4(const void* p, long long rs, int dtype) { return rs % 4 == 0 && ((uintptr_t)p & (dtype == TCMI_F32 ? 15 : 7)) == 0; }

struct In {
  const void *h, *w, *bias;
  long long hrs, wrs;
  const long long* y;
  long long ignore;
};

// the pass over the operands: what the logits' product cannot read in place, and for the backward the factors and maxima
hipError_t prepare(const Shape& s, const In& in, const Rows& rows, Prep a, hipStream_t st) {
  auto one = [&](Operand& o, const void* src, long long rs, int n, f16* out, float* inv) {
    o.src = src;
    o.rs = rs;
    o.rows = n;
    o.cols = s.D;
    o.colsp = s.dp;
    o.vec = vec4(src, rs, s.dtype);
    o.out = out;
    o.inv = inv;
    const bool work = out || (&o == &a.h && a.r);
    o.blocks = !work ? 0 : n / 4 < 1 ? 1 : n / 4 > PARTS ? PARTS : n / 4;
  };
  one(a.h, in.h, in.hrs, s.T, rows.h, rows.hs);
  one(a.w, in.w, in.wrs, s.V, rows.w, rows.ws);
  const int blocks = a.h.blocks + a.w.blocks;
  if (!blocks) return hipSuccess;
  if (s.dtype == TCMI_F32) hipLaunchKernelGGL(prep_kernel<TCMI_F32>, dim3(blocks), dim3(256), 0, st, a);
  else if (s.dtype == TCMI_F16) hipLaunchKernelGGL(prep_kernel<TCMI_F16>, dim3(blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(prep_kernel<TCMI_BF16>, dim3(blocks), dim3(256), 0, st, a);
  return hipGetLastError();
}

// workgroups of the pass for the features' largest values
Top top_of(const Shape& s, const void* src, long long rs, int rows, const float* r, unsigned* top) {
  Top t{src, rs, rows, s.D, vec4(src, rs, s.dtype), 64, 0, 0, r, top};
  while (t.lanes > 1 && t.lanes * 2 >= s.D) t.lanes /= 2;        // half of 4 lanes would do
  t.panels = (s.D + 4 * t.lanes - 1) / (4 * t.lanes);
  const int per = TOP_THREADS / t.lanes;
  const int shares = (rows + 8 * per - 1) / (8 * per);           // eight rows a thread at least
  t.blocks = t.panels * (shares < TOP_SHARES ? shares : TOP_SHARES);
  return t;
}

hipError_t tops(const Shape& s, const Top& x, const Top& y, hipStream_t st) {
  const int blocks = x.blocks + y.blocks;
  if (!blocks) return hipSuccess;
  if (s.dtype == TCMI_F32) hipLaunchKernelGGL(top_kernel<TCMI_F32>, dim3(blocks), dim3(TOP_THREADS), 0, st, x, y);
  else if (s.dtype == TCMI_F16) hipLaunchKernelGGL(top_kernel<TCMI_F16>, dim3(blocks), dim3(TOP_THREADS), 0, st, x, y);
  else hipLaunchKernelGGL(top_kernel<TCMI_BF16>, dim3(blocks), dim3(TOP_THREADS), 0, st, x, y);
  return hipGetLastError();
}

hipError_t turn(const Shape& s, const Turn& x, const Turn& y, hipStream_t st) {
  const int blocks = x.tiles + y.tiles;
  if (!blocks) return hipSuccess;
  if (s.dtype == TCMI_F32) hipLaunchKernelGGL(turn_kernel<TCMI_F32>, dim3(blocks), dim3(256), 0, st, x, y);
  else if (s.dtype == TCMI_F16) hipLaunchKernelGGL(turn_kernel<TCMI_F16>, dim3(blocks), dim3(256), 0, st, x, y);
  else hipLaunchKernelGGL(turn_kernel<TCMI_BF16>, dim3(blocks), dim3(256), 0, st, x, y);
  return hipGetLastError();
}

// the logits' product for the classes [v0, v0 + vc)
Args logit_args(const Shape& s, const In& in, const Rows& r, int v0, int vc) {
  Args g{};
  g.M = s.T;
  g.N = vc;
  g.K = s.P * s.dp;
  g.lda = s.h_direct ? in.hrs : s.P * s.dp;
  g.ldb = s.w_direct ? in.wrs : s.P * s.dp;
  g.batch = 1;
  g.nseg = 1;
  g.a[0] = s.h_direct ? in.h : r.h;
  g.b[0] = (const f16*)(s.w_direct ? in.w : r.w) + v0 * g.ldb;
  return g;
}

template <int P>
hipError_t forward(const Shape& s, const In& in, const FwdWork& w, float* lse, float* loss, float* total, float* count, int mean,
                   hipStream_t st) {
  int tiles;
  if (s.few) {
    tiles = few_blocks(s);
    auto go = [&](auto kernel, auto args) {
      args.h = in.h;
      args.w = in.w;
      args.bias = in.bias;
      args.hrs = in.hrs;
      args.wrs = in.wrs;
      args.T = s.T;
      args.D = s.D;
      args.V = s.V;
      args.y = in.y;
      args.part = w.part;
      args.target = w.target;
      hipLaunchKernelGGL(kernel, dim3(tiles), dim3(256), 0, st, args);
    };
    if (s.dtype == TCMI_F32) go(few_kernel<f32x4, float, TCMI_F32>, FewArgs<TCMI_F32>{});
    else if (s.dtype == TCMI_F16) go(few_kernel<f16x8, f16, TCMI_F16>, FewArgs<TCMI_F16>{});
    else go(few_kernel<bf16x8, __bf16, TCMI_BF16>, FewArgs<TCMI_BF16>{});
    TRY(hipGetLastError());
  } else {
    TRY(prepare(s, in, w.rows, Prep{}, st));
    Args g = logit_args(s, in, w.rows, 0, s.V);
    TRY(run_logits<P>(g, s.dtype, EpiLse<P>{{w.rows.hs, w.rows.ws, in.bias, s.dtype, 0}, w.part, w.target, in.y}, st));
    tiles = g.tn;
  }
  // one workgroup for both while its 16 waves have at most four rows each: 7 us for 64 rows (two launches: 3 + 3 and a gap), 26
  // for 256
  if (total && s.T <= 64 && (long long)s.T * tiles <= 8192) {       // 64 KB of statistics
    hipLaunchKernelGGL(rowstat_total_kernel, dim3(1), dim3(1024), 0, st, w.part, tiles, w.target, in.y, in.ignore, s.T, s.V, lse, loss, mean,
                       total, count);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(rowstat_kernel, dim3((s.T + 3) / 4), dim3(256), 0, st, w.part, tiles, w.target, in.y, in.ignore, s.T, s.V, lse, loss);
  TRY(hipGetLastError());
  if (total) {
    hipLaunchKernelGGL(total_kernel, dim3(1), dim3(1024), 0, st, loss, in.y, in.ignore, s.T, mean, total, count);
    TRY(hipGetLastError());
  }
  return hipSuccess;
}

template <int P>
hipError_t backward(const Shape& s, const In& in, const BwdWork& w, const float* lse, const float* dloss, int per_row, const float* count,
                    void* dh, void* dw, void* db, hipStream_t st) {
  Prep a{};
  a.y = in.y;
  a.ignore = in.ignore;
  a.dloss = dloss;
  a.count = count;
  a.per_row = per_row;
  a.r = w.r;
  a.top = w.top;
  a.tops = 2 * tops_of(s);
  TRY(prepare(s, in, w.rows, a, st));
  TRY(tops(s, dw ? top_of(s, in.h, in.hrs, s.T, w.r, w.top) : Top{}, dh ? top_of(s, in.w, in.wrs, s.V, nullptr, w.top + tops_of(s)) : Top{}, st));
  const int size = s.dtype == TCMI_F32 ? 4 : 2, vc = piece_of(s);
  for (int v0 = 0; v0 < s.V; v0 += vc) {
    const int n = s.V - v0 < vc ? s.V - v0 : vc, np = (int)kpad(n, P), ldv = (n + 63) & ~63;
    Turn th{}, tw{};
    if (dw && v0 == 0) {
      th = Turn{in.h, in.hrs, s.T, s.D, s.tp, vec4(in.h, in.hrs, s.dtype), (s.tp + 63) / 64, 0, w.r, w.top, w.ht};
      th.tiles = th.tx * ((s.D + 63) / 64);
    }
    if (dh) {
      tw = Turn{(const char*)in.w + v0 * in.wrs * size, in.wrs, n, s.D, np, vec4(in.w, in.wrs, s.dtype), (np + 63) / 64, 0, nullptr,
                w.top + tops_of(s), w.wt};
      tw.tiles = tw.tx * ((s.D + 63) / 64);
    }
    TRY(turn(s, th, tw, st));
    Args g = logit_args(s, in, w.rows, v0, n);
    TRY(run_logits<P>(g, s.dtype,
                      EpiProb<P>{{w.rows.hs, w.rows.ws, in.bias, s.dtype, v0}, reinterpret_cast<const float2*>(lse), in.y, in.ignore, s.V, w.p, w.pt, np, s.tp, w.r, w.exps, w.sums, ldv}, st));
    if (dw || db) {
      hipLaunchKernelGGL(class_kernel<P>, dim3(ldv / 64), dim3(256), 0, st, w.exps, w.sums, ldv, (s.T + g.wave_rows - 1) / g.wave_rows, g.wave_rows, n,
                         w.pt, s.tp, dw ? w.cexp : nullptr, db, s.dtype, v0);
      TRY(hipGetLastError());
    }
    Args d{};
    d.batch = 1;
    d.nseg = 1;
    d.part = w.split;
    if (dh) {
      d.M = s.T;
      d.N = s.D;
      d.K = P * np;
      d.lda = d.ldb = d.K;
      d.a[0] = w.p;
      d.b[0] = w.wt;
      TRY(run<P>(d, EpiGrad{w.top + tops_of(s), w.sum, v0 == 0, v0 + vc >= s.V, w.r, dh, s.dtype, s.D, nullptr, vec4(dh, s.D, s.dtype)}, st));
    }
    if (dw) {
      d.M = n;
      d.N = s.D;
      d.K = P * s.tp;
      d.lda = d.ldb = d.K;
      d.a[0] = w.pt;
      d.b[0] = w.ht;
      TRY(run<P>(d, EpiGrad{w.top, nullptr, 1, 1, nullptr, (char*)dw + (long long)v0 * s.D * size, s.dtype, s.D, w.cexp,
                            vec4(dw, s.D, s.dtype)}, st));
    }
  }
  return hipSuccess;
}

bool shape_ok(int T, int D, int V, int dtype) {
  return T >= 1 && D >= 1 && V >= 1 && T <= (1 << 21) && D <= (1 << 20) && V <= (1 << 28) &&
         (dtype == TCMI_F32 || dtype == TCMI_F16 || dtype == TCMI_BF16);
}

// an operand is read in place when its rows are whole k steps and 16-byte aligned
bool direct(const void* p, long long rs, int D, int dtype) {
  return dtype != TCMI_F32 && D % 64 == 0 && rs % 8 == 0 && rs <= MAX_ROW && ((uintptr_t)p & 15) == 0;
}

Shape shape_of(int T, int D, int V, int dtype, bool h_direct, bool w_direct, bool alone) {
  Shape s{};
  s.few = alone && T <= FEW_ROWS;
  s.T = T;
  s.D = D;
  s.V = V;
  s.dtype = dtype;
  s.P = dtype == TCMI_F32 ? 2 : 1;
  s.dp = (int)kpad(D, s.P);
  s.tp = (int)kpad(T, s.P);
  s.h_direct = h_direct;
  s.w_direct = w_direct;
  return s;
}

}  // namespace lce
}  // namespace tcmi

using namespace tcmi::lce;

extern "C" {

long long tcmi_lce_work_bytes(const void* h, long long h_rs, const void* w, long long w_rs, int tokens, int features, int classes,
                              int dtype, int what) {
  if (!shape_ok(tokens, features, classes, dtype) || what < 0 || what > 2) return -1;
  const Shape s = shape_of(tokens, features, classes, dtype, direct(h, h_rs, features, dtype), direct(w, w_rs, features, dtype),
                           what == TCMI_LCE_ALONE);
  Arena a{nullptr};
  if (what == TCMI_LCE_GRAD) take_bwd(a, s);
  else take_fwd(a, s);
  return a.used;
}

int tcmi_linear_cross_entropy(const void* h, long long h_rs, const void* w, long long w_rs, const void* bias, const long long* target,
                              long long ignore_index, int tokens, int features, int classes, float* lse, float* loss, float* total,
                              float* count, int mean, int for_grad, void* work, long long work_bytes, int dtype, void* stream) {
  if (!shape_ok(tokens, features, classes, dtype) || !h || !w || !target || !lse || !loss || !work || (total && !count) || h_rs < features ||
      w_rs < features || ((uintptr_t)lse & 7))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_linear_cross_entropy: bad argument");
  const Shape s = shape_of(tokens, features, classes, dtype, direct(h, h_rs, features, dtype), direct(w, w_rs, features, dtype),
                           !for_grad);
  Arena a{(char*)work};
  const FwdWork k = take_fwd(a, s);
  if (a.used > work_bytes || ((uintptr_t)work & 255))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_linear_cross_entropy: workspace too small or not 256-byte aligned");
  const In in{h, w, bias, h_rs, w_rs, target, ignore_index};
  const hipError_t e = (s.P == 2 ? forward<2> : forward<1>)(s, in, k, lse, loss, total, count, mean, reinterpret_cast<hipStream_t>(stream));
  return e == hipSuccess ? TCMI_OK : tcmi_set_error_(TCMI_ERR_HIP, hipGetErrorString(e));
}

int tcmi_linear_cross_entropy_grad(const void* h, long long h_rs, const void* w, long long w_rs, const void* bias,
                                   const long long* target, long long ignore_index, int tokens, int features, int classes,
                                   const float* lse, const float* dloss, int per_row, const float* count, void* dh, void* dw, void* db,
                                   void* work, long long work_bytes, int dtype, void* stream) {
  if (!shape_ok(tokens, features, classes, dtype) || !h || !w || !target || !lse || !dloss || !work || (!dh && !dw && !db) ||
      h_rs < features || w_rs < features || ((uintptr_t)lse & 7))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_linear_cross_entropy_grad: bad argument");
  const Shape s = shape_of(tokens, features, classes, dtype, direct(h, h_rs, features, dtype), direct(w, w_rs, features, dtype), false);
  Arena a{(char*)work};
  const BwdWork k = take_bwd(a, s);
  if (a.used > work_bytes || ((uintptr_t)work & 255))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_linear_cross_entropy_grad: workspace too small or not 256-byte aligned");
  const In in{h, w, bias, h_rs, w_rs, target, ignore_index};
  const hipError_t e = (s.P == 2 ? backward<2> : backward<1>)(s, in, k, lse, dloss, per_row, count, dh, dw, db, reinterpret_cast<hipStream_t>(stream));
  return e == hipSuccess ? TCMI_OK : tcmi_set_error_(TCMI_ERR_HIP, hipGetErrorString(e));
}

}  // extern "C"
