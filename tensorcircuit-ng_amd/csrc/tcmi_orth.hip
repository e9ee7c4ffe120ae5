// Newton-Schulz orthogonalisation of (batches of) matrices, its gradient, and the optimiser step built on it.
//
//   N = |G|_F + eps,  X_0 = G / N;   A = X X^H,  B = b A + c A A,  X <- a X + B X        (steps times)
// A and B are symmetric, so only the tiles on and below the diagonal are computed and written twice (ns_factor).  Singular values are
// at most 1 at the start (Frobenius norm) and the polynomial bounds them afterwards, so every operand has a bound known
// on the host: operands are f16 under a power-of-two scale, products run on the f16 matrix pipe (mm16.h).
//
// Precision.  X is carried in f32: a X is exact, the matrix pipe sees only B X.
//   full (f32, f16, complex64, and everything that is differentiated): two f16 pieces per operand, three products.
//   half (bf16 results): one f16 piece per operand.  Directions with small singular values are the ones a step amplifies
//   (by a per step, a^5 = 485 for the default), and B is small on them: rounding X before B X costs 2^-11 of |B X| and
//   does not reach them, where rounding the carried X would (1e-3 against 2e-2 of the result, five steps, random and
//   low-rank-plus-noise matrices, against 64 bits; a bf16 result is itself rounded at 1.7e-3).
// Complex matrices are real ones of twice the size, E(X) = [[Re, Im], [-Im, Re]], E(X Y) = E(X) E(Y), E(X)^T = E(X^H):
// the two symmetric products run on E directly, the updates compute the upper block row only.
#include <hip/hip_runtime.h>
#include <math.h>

#include "../../include/tcmi.h"
#include "tcmi_mm16.h"

extern "C" int tcmi_set_error_(int code, const char* msg);

namespace tcmi {
namespace orth {

using namespace mm16;

enum { SRC_F32 = 0, SRC_F16 = 1, SRC_BF16 = 2, SRC_C64 = 3, SRC_PLANAR = 4 };

struct Mat {                    // a batch of matrices as the caller holds them; strides in elements
  const void* p;
  long long rs, cs, bs;
};

template <int SRC>
__device__ __forceinline__ float2 fetch(const void* p, long long at) {
  if constexpr (SRC == SRC_F32 || SRC == SRC_PLANAR) return make_float2(((const float*)p)[at], 0.f);
  if constexpr (SRC == SRC_F16) return make_float2((float)((const f16*)p)[at], 0.f);
  if constexpr (SRC == SRC_BF16) return make_float2((float)((const __bf16*)p)[at], 0.f);
  if constexpr (SRC == SRC_C64) return ((const float2*)p)[at];
  return make_float2(0.f, 0.f);
}

// four neighbours, the address aligned for one load
template <int SRC>
__device__ __forceinline__ f32x4 fetch4(const void* p, long long at) {
  if constexpr (SRC == SRC_F16) return __builtin_convertvector(*reinterpret_cast<const f16x4*>((const f16*)p + at), f32x4);
  else if constexpr (SRC == SRC_BF16) return __builtin_convertvector(*reinterpret_cast<const bf16x4*>((const __bf16*)p + at), f32x4);
  else return *reinterpret_cast<const f32x4*>((const float*)p + at);
}

__device__ __forceinline__ void put(void* p, int dtype, long long at, float v) {
  if (dtype == TCMI_F32) ((float*)p)[at] = v;
  else if (dtype == TCMI_F16) ((f16*)p)[at] = (f16)v;
  else ((__bf16*)p)[at] = (__bf16)v;
}

__device__ __forceinline__ double block_sum(double v, double* red) {        // 256 threads, fixed order
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0] + red[1] + red[2] + red[3];
  __syncthreads();
  return v;
}

// Partial sums of squares (MODE 0), of x y (MODE 1: <D, G>), or the momentum update with the squares of its direction u
// (MODE 2), in f64: an f32 square overflows from 1.8e19 on.  One read of the data; partial sums in a fixed order, so the
// result does not depend on the order of the workgroups.  lanes: threads along the contiguous axis.
struct SumArgs {
  Mat x, y;
  int outer, inner, lanes, vec;            // vec: four neighbours can be read (and the momentum updated) at once
  double* part;               // [batch][gridDim.x]
  float* buf;                 // MODE 2: momentum, strides below
  long long brs, bcs, bbs;
  float rest;
  int nesterov;
};

// `rest` = 1 - momentum, formed in f64: as 1 - 0.95f it would be off by 2^-22 of itself
__device__ __forceinline__ float direction(float g, float v, float rest, int nesterov) {
  return nesterov ? fmaf(rest, g - v, v) : v;
}

template <int SRC, int MODE>
__device__ __forceinline__ double sums_one(const SumArgs& a, long long o, int i, long long bx, long long by) {
  const float2 v = fetch<SRC>(a.x.p, bx + o * a.x.rs + i * a.x.cs);
  if constexpr (MODE == 1) {              // y: planar f32 D, imaginary parts brs further on
    const float* d = (const float*)a.y.p + by + o * a.y.rs + i * a.y.cs;
    double s = (double)v.x * d[0];
    if constexpr (SRC == SRC_C64) s += (double)v.y * d[a.brs];
    return s;
  } else if constexpr (MODE == 2) {
    float* m = a.buf + by + o * a.brs + i * a.bcs;
    const float nv = fmaf(a.rest, v.x - m[0], m[0]);
    m[0] = nv;
    const float u = direction(v.x, nv, a.rest, a.nesterov);
    return (double)u * u;
  } else {
    return (double)v.x * v.x + (double)v.y * v.y;
  }
}

template <int SRC, int MODE>
__global__ __launch_bounds__(256) void sums_kernel(SumArgs a) {
  __shared__ double red[4];
  const int per = 256 / a.lanes, r0 = threadIdx.x / a.lanes, c0 = threadIdx.x % a.lanes;
  const long long bx = (long long)blockIdx.y * a.x.bs, by = (long long)blockIdx.y * (MODE == 2 ? a.bbs : a.y.bs);
  double s = 0.0;
  for (long long o = blockIdx.x * per + r0; o < a.outer; o += gridDim.x * per) {
    int i = c0;
    if constexpr (SRC != SRC_C64 && MODE != 1) {
      if (a.vec) {                        // four neighbours a thread; f32 sums of four squares would overflow, so f64 at once
        i = 4 * c0;
#pragma unroll 2
        for (; i + 3 < a.inner; i += 4 * a.lanes) {
          const f32x4 v = fetch4<SRC>(a.x.p, bx + o * a.x.rs + i);
          f32x4 u = v;
          if constexpr (MODE == 2) {
            f32x4* m = reinterpret_cast<f32x4*>(a.buf + by + o * a.brs + i);
            f32x4 w = *m;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              w[k] = fmaf(a.rest, v[k] - w[k], w[k]);
              u[k] = direction(v[k], w[k], a.rest, a.nesterov);
            }
            *m = w;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) s += (double)u[k] * u[k];
        }
        for (const int e = min(i + 4, a.inner); i < e; ++i) s += sums_one<SRC, MODE>(a, o, i, bx, by);
        continue;
      }
    }
    for (; i < a.inner; i += a.lanes) s += sums_one<SRC, MODE>(a, o, i, bx, by);
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) a.part[(long long)blockIdx.y * gridDim.x + blockIdx.x] = s;
}

// A factor m 2^e, 0.5 <= |m| <= 1: norms and their inverses leave f32's range long before the entries that they scale.
struct Factor {
  float m;
  int e;
};
__device__ __forceinline__ float times(float x, Factor f) { return ldexpf(x, f.e) * f.m; }
__device__ __forceinline__ Factor factor_of(double d) {
  if (!(fabs(d) < INFINITY)) return {(float)d, 0};
  int k;
  const double f = frexp(d, &k);
  return {(float)f, k};
}
// 1 / d; 0 for 0
__device__ __forceinline__ Factor inverse(double d) {
  if (d == 0.0 || !(d < INFINITY)) return {d == 0.0 ? 0.f : (float)(1.0 / d), 0};
  int k;
  const double f = frexp(d, &k);
  return {(float)(0.5 / f), 1 - k};
}

// Operand layout: a 64 x 64 tile of the source becomes f16 pieces, row-major and transposed (both k-contiguous for the
// products that read them), zero beyond the matrix up to the padded length, and the f32 carry.  Bound by its writes.
// part: the tile is divided by (sqrt(sum of part) + eps); every workgroup adds the partial sums itself.
struct PackArgs {
  Mat src;
  int m, n, tx, ty, fast_rows, vec;        // logical size, tiles, 1: the source is contiguous along its columns; vec: four at once
  const double* part;
  int npart;
  float eps, scale;                        // pieces = value * scale
  double* norm_out;                        // [batch] the norm without eps (may be null)
  const float* buf;                        // momentum (null: none)
  long long brs, bcs, bbs;
  float rest;
  int nesterov;
  f16 *x, *t;                              // X [mr][ld], X^T [nc][ldt]
  long long ld, os, ldt, ts;               // row strides and batch strides
  float* carry;                            // f32 [m][ldc] (null: none); complex: im at column n + j
  int carry_raw;                           // 1: the carry is not divided by the norm
  long long ldc, cbs;
  int embed;                               // complex as a real matrix of twice the size
};

template <int SRC, int P>
__global__ __launch_bounds__(256) void pack_kernel(PackArgs a) {
  constexpr bool MAYBE_COMPLEX = SRC == SRC_C64 || SRC == SRC_PLANAR;
  __shared__ float tr[64][65], tim[MAYBE_COMPLEX ? 64 : 1][65];
  __shared__ double red[4];
  const unsigned tiles = (unsigned)a.tx * a.ty;
  const int bz = blockIdx.x / tiles, t = blockIdx.x % tiles, i0 = (t / a.tx) * 64, j0 = (t % a.tx) * 64;
  Factor inv = {1.f, 0};
  if (a.part) {
    double s = 0.0;
    for (int k = threadIdx.x; k < a.npart; k += 256) s += a.part[(long long)bz * a.npart + k];
    const double nrm = sqrt(block_sum(s, red));
    if (a.norm_out && t == 0 && threadIdx.x == 0) a.norm_out[bz] = nrm;
    inv = inverse(nrm + (double)a.eps);
  }
  // 16 threads along an axis, four elements each, 16 lines at a time
  const long long base = (long long)bz * a.src.bs;
  const int u = (threadIdx.x & 15) * 4, w = threadIdx.x >> 4;
  const int flen = a.fast_rows ? a.m : a.n;
#pragma unroll
  for (int k = w; k < 64; k += 16) {
    const int line = (a.fast_rows ? j0 : i0) + k, f0 = (a.fast_rows ? i0 : j0) + u;
    const long long ls = a.fast_rows ? a.src.cs : a.src.rs, fs = a.fast_rows ? a.src.rs : a.src.cs;
    f32x4 re = {0.f, 0.f, 0.f, 0.f}, im = {0.f, 0.f, 0.f, 0.f};
    if (line < (a.fast_rows ? a.n : a.m)) {
      const long long at = base + line * ls + f0 * fs;
      if (SRC != SRC_C64 && a.vec && f0 + 3 < flen) {
        re = fetch4<SRC>(a.src.p, at);
        if (SRC == SRC_PLANAR && a.embed) {
          const float* q = (const float*)a.src.p + at + a.n;
#pragma unroll
          for (int e = 0; e < 4; ++e) im[e] = q[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (f0 + e < flen) {
            const float2 v = fetch<SRC>(a.src.p, at + e * fs);
            re[e] = v.x;
            im[e] = SRC == SRC_PLANAR && a.embed ? ((const float*)a.src.p)[at + e * fs + a.n] : v.y;
          }
      }
      if (a.buf) {
        const long long bt = (long long)bz * a.bbs + (a.fast_rows ? line * a.bcs + f0 * a.brs : line * a.brs + f0 * a.bcs);
        const long long bf = a.fast_rows ? a.brs : a.bcs;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (f0 + e < flen) re[e] = direction(re[e], a.buf[bt + e * bf], a.rest, a.nesterov);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int il = a.fast_rows ? u + e : k, jl = a.fast_rows ? k : u + e;
      tr[il][jl] = re[e];
      if (MAYBE_COMPLEX) tim[MAYBE_COMPLEX ? il : 0][jl] = im[e];
    }
  }
  __syncthreads();
  const Factor cinv = a.carry_raw ? Factor{1.f, 0} : inv;
  const bool twice = MAYBE_COMPLEX && a.embed;
  const int mrows = twice ? a.m : (int)kpad(a.m, P), ncols = twice ? a.n : (int)kpad(a.n, P);
  f16 *px = a.x + (long long)bz * a.os, *pt = a.t + (long long)bz * a.ts;
  // four values at k .. k + 3 of a row, as far as `len` reaches (`len` - k in 1 .. 4)
  auto store = [&](f16* row, int k, int len, f32x4 v) {
    f16x4 hi, lo;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f16 h, l;
      two_pieces(times(v[e], inv) * a.scale, h, l);
      hi[e] = h;
      lo[e] = l;
    }
    if (k + 3 < len && (k & 3) == 0) {
      store_four<P>(row, k, hi, lo);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k + e < len) {
          row[kpos<P>(k + e)] = hi[e];
          if (P == 2) row[kpos<P>(k + e) + 32] = lo[e];
        }
    }
  };
  auto carry = [&](float* q, int left, f32x4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = times(v[e], cinv);
    if (left > 3 && ((uintptr_t)q & 15) == 0) {
      *reinterpret_cast<f32x4*>(q) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (e < left) q[e] = v[e];
    }
  };
#pragma unroll
  for (int k = w; k < 64; k += 16) {
    {                                      // rows of X
      const int i = i0 + k, j = j0 + u;
      if (i < a.m && j < ncols) {
        const f32x4 re = {tr[k][u], tr[k][u + 1], tr[k][u + 2], tr[k][u + 3]};
        store(px + i * a.ld, j, ncols, re);
        float* c = a.carry ? a.carry + (long long)bz * a.cbs + i * a.ldc + j : nullptr;
        if (c && j < a.n) carry(c, a.n - j, re);
        if (twice) {
          const int q = MAYBE_COMPLEX ? k : 0;
          const f32x4 im = {tim[q][u], tim[q][u + 1], tim[q][u + 2], tim[q][u + 3]};
          store(px + i * a.ld, j + a.n, 2 * a.n, im);
          store(px + (i + a.m) * a.ld, j, a.n, -im);
          store(px + (i + a.m) * a.ld, j + a.n, 2 * a.n, re);
          if (c) carry(c + a.n, a.n - j, im);
        }
      }
    }
    {                                      // rows of X^T
      const int i = i0 + u, j = j0 + k;
      if (j < a.n && i < mrows) {
        const f32x4 re = {tr[u][k], tr[u + 1][k], tr[u + 2][k], tr[u + 3][k]};
        store(pt + j * a.ldt, i, mrows, re);
        if (twice) {
          const f32x4 im = MAYBE_COMPLEX ? f32x4{tim[MAYBE_COMPLEX ? u : 0][k], tim[MAYBE_COMPLEX ? u + 1 : 0][k],
                                                 tim[MAYBE_COMPLEX ? u + 2 : 0][k], tim[MAYBE_COMPLEX ? u + 3 : 0][k]}
                                         : re;
          store(pt + (j + a.n) * a.ldt, i, a.m, im);
          store(pt + j * a.ldt, i + a.m, 2 * a.m, -im);
          store(pt + (j + a.n) * a.ldt, i + a.m, 2 * a.m, re);
        }
      }
    }
  }
}

__global__ __launch_bounds__(256) void clear_kernel(uint4* p, long long n) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) p[i] = make_uint4(0, 0, 0, 0);
}

// A symmetric result as f16 pieces: value = alpha acc + beta src, stored times `scale`; a tile below the diagonal also
// writes its mirror image (through LDS where the product is not split: two bytes a lane took 15 us of 85 at 4096 x 4096).
// Columns up to the padded width get zeros.
template <int P>
struct EpiSym {
  static constexpr bool TILE = true, FOUR = true;
  f16* out;
  const f16* src;
  long long ld, bs;
  float alpha, beta, scale;
  template <class T>
  static constexpr int lds() { return Transposed<T, P>::BYTES; }
  // the real part of a doubled hermitian result stands in it twice (g.half is a multiple of 64)
  __device__ __forceinline__ bool twice(const Args& g, int row, int col) const { return row < g.half && col < g.half; }
  __device__ __forceinline__ long long second(const Args& g) const { return g.half * ld + kpos<P>(g.half); }
  __device__ __forceinline__ void put_row(const Args& g, int bz, int wide, int row, int col, f32x4 v, f16x4& vh, f16x4& vl) const {
    const bool in = row < g.M && col < wide;
    const long long at = bz * bs + row * ld + kpos<P>(col);
    f16x4 s4 = {}, t4 = {};
    if (src && in) {
      s4 = *reinterpret_cast<const f16x4*>(src + at);
      if (P == 2) t4 = *reinterpret_cast<const f16x4*>(src + at + 32);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x = fmaf(v[r], alpha, beta * ((float)s4[r] + (float)t4[r]));
      x = row < g.M && col + r < g.M ? x * scale : 0.f;
      f16 a, b;
      two_pieces(x, a, b);
      vh[r] = a;
      vl[r] = b;
    }
    if (in) {
      *reinterpret_cast<f16x4*>(out + at) = vh;
      if (P == 2) *reinterpret_cast<f16x4*>(out + at + 32) = vl;
      if (twice(g, row, col)) {
        *reinterpret_cast<f16x4*>(out + at + second(g)) = vh;
        if (P == 2) *reinterpret_cast<f16x4*>(out + at + second(g) + 32) = vl;
      }
    }
  }
  __device__ __forceinline__ void four(const Args& g, int bz, bool mirror, int row, int col, f32x4 v) const {
    const int wide = (int)kpad(g.M, P);
    f16x4 vh, vl;
    put_row(g, bz, wide, row, col, v, vh, vl);
    if (mirror && row < wide) {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < g.M) {
          f16* p = out + bz * bs + (col + r) * ld + kpos<P>(row);
          p[0] = vh[r];
          if (P == 2) p[32] = vl[r];
          if (twice(g, row, col)) {
            p[second(g)] = vh[r];
            if (P == 2) p[second(g) + 32] = vl[r];
          }
        }
    }
  }
  template <class T>
  __device__ __forceinline__ void tile(const Args& g, int m0, int n0, int bz, bool mirror, char* mem, f32x4 (&acc)[T::MI][T::NI]) const {
    const int wide = (int)kpad(g.M, P);
    const Transposed<T, P> turned{reinterpret_cast<f16*>(mem)};
    __syncthreads();
    each<T>(m0, n0, acc, [&](int row, int col, f32x4 v) {
      f16x4 vh, vl;
      put_row(g, bz, wide, row, col, v, vh, vl);
      if (mirror) turned.stage(row - m0, col - n0, vh, vl);
    });
    if (!mirror) return;
    __syncthreads();
    turned.flush(out + bz * bs, ld, n0, g.M, m0, wide);
    if (twice(g, m0, n0)) turned.flush(out + bz * bs + second(g), ld, n0, g.half, m0, g.half);
  }
};

// carry <- beta carry + alpha acc (f32, in place: a thread reads and writes the same element)
struct EpiCarry {
  static constexpr bool TILE = false, FOUR = true;
  float* carry;
  long long ld, bs;
  float alpha, beta;
  const double* dev;             // [batch] further factor of acc held on the device (null: none)
  __device__ __forceinline__ void four(const Args& g, int bz, bool, int row, int col, f32x4 v) const {
    if (row >= g.M) return;
    const float al = dev ? (float)(alpha * dev[bz]) : alpha;
    float* p = carry + bz * bs + row * ld + col;
    if (col + 3 < g.N) {
      f32x4 x = *reinterpret_cast<f32x4*>(p);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = fmaf(al, v[r], beta * x[r]);
      *reinterpret_cast<f32x4*>(p) = x;
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (col + r < g.N) p[r] = fmaf(al, v[r], beta * p[r]);
    }
  }
};

// A step's result as the next step's operands: x = beta carry + alpha acc stays in the carry and goes out as pieces, row-major
// and (through LDS) transposed.  Saves the pass that would read the carry again (27 us a step of 4096 x 4096).  Complex
// matrices (n > 0: columns of the imaginary part start there) need sides that are multiples of 16: the product forms the
// upper half [Re, Im], and the lower one [-Im, Re] is written beside it.
template <int P>
struct EpiNext {
  static constexpr bool TILE = true, FOUR = true;
  float* carry;
  long long ldc, cs;
  float alpha, beta, scale;
  f16 *x, *t;
  long long ld, xs, ldt, ts;
  int n;
  template <class T>
  static constexpr int lds() { return Transposed<T, P>::BYTES; }
  // rows of X^T that hold values or their padding
  __device__ __forceinline__ int tall(const Args& g) const { return n ? g.M : (int)kpad(g.M, P); }
  __device__ __forceinline__ void put_row(const Args& g, int bz, int row, int col, f32x4 v, f16x4& vh, f16x4& vl) const {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (row < g.M && col < g.N) {                    // rows of the carry are padded to four columns
      f32x4* c = reinterpret_cast<f32x4*>(carry + bz * cs + row * ldc + col);
      const f32x4 old = *c;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = col + r < g.N ? fmaf(alpha, v[r], beta * old[r]) : 0.f;
      *c = o;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      f16 a, b;
      two_pieces(o[r] * scale, a, b);
      vh[r] = a;
      vl[r] = b;
    }
    if (row < g.M && col < (int)kpad(g.N, P)) {
      f16* o = x + bz * xs + row * ld;
      store_four<P>(o, col, vh, vl);
      if (n) {
        if (col < n) store_four<P>(o + g.M * ld, col + n, vh, vl);
        else store_four<P>(o + g.M * ld, col - n, -vh, -vl);
      }
    }
  }
  __device__ __forceinline__ void four(const Args& g, int bz, bool, int row, int col, f32x4 v) const {
    f16x4 vh, vl;
    put_row(g, bz, row, col, v, vh, vl);
    if (row >= tall(g)) return;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (col + r < g.N) {
        f16* o = t + bz * ts + (col + r) * ldt + kpos<P>(row);
        o[0] = vh[r];
        if (P == 2) o[32] = vl[r];
        if (n) {
          const bool im = col >= n;
          o = t + bz * ts + (col + r + (im ? -n : n)) * ldt + kpos<P>(row + g.M);
          o[0] = im ? -vh[r] : vh[r];
          if (P == 2) o[32] = im ? -vl[r] : vl[r];
        }
      }
  }
  template <class T>
  __device__ __forceinline__ void tile(const Args& g, int m0, int n0, int bz, bool, char* mem, f32x4 (&acc)[T::MI][T::NI]) const {
    const Transposed<T, P> turned{reinterpret_cast<f16*>(mem)};
    __syncthreads();
    each<T>(m0, n0, acc, [&](int row, int col, f32x4 v) {
      f16x4 vh, vl;
      put_row(g, bz, row, col, v, vh, vl);
      turned.stage(row - m0, col - n0, vh, vl);
    });
    __syncthreads();
    turned.flush(t + bz * ts, ldt, n0, g.N, m0, tall(g));
    if (n) turned.flush_twin(t + bz * ts, ldt, n0, g.N, m0, g.M, n);
  }
};

// The last step: x = beta X + alpha acc goes to the caller's matrix (out = x) or into a weight (out = keep out + rate x).
// P = 0: X is the f32 carry.  P > 0: the product is the transposed one, T B, so that a matrix taller than wide is written along
// its rows too, and X comes from T's pieces (one piece, 2^-11 of X in the last step, is below what one-piece products cost).
template <int P, int DT>
struct EpiOut {
  static constexpr bool TILE = false, FOUR = true;
  const void* src;               // f32 carry, or T
  long long ld, bs;
  float alpha, beta;
  void* out;
  long long rs, cs, os;
  int n;                         // columns; complex: columns of the imaginary part start there
  int update;
  float keep, rate;
  int vec;                       // rows contiguous and aligned for four elements
  __device__ __forceinline__ float old_x(long long row, int j) const {
    if constexpr (P == 0) return ((const float*)src)[row + j];
    const f16* p = (const f16*)src + row + kpos<P>(j);
    return P == 2 ? (float)p[0] + (float)p[32] : (float)p[0];
  }
  __device__ __forceinline__ void four(const Args& g, int bz, bool, int row, int col, f32x4 v) const {
    if (row >= g.M) return;
    const long long line = bz * bs + row * ld;
    if (DT != TCMI_C64 && vec && col + 3 < g.N) {                    // four neighbours of a row-major matrix at once
      f32x4 x;
      if constexpr (P == 0) {
        x = *reinterpret_cast<const f32x4*>((const float*)src + line + col);
      } else {
        const f16* p = (const f16*)src + line + kpos<P>(col);
        x = __builtin_convertvector(*reinterpret_cast<const f16x4*>(p), f32x4);
        if (P == 2) x += __builtin_convertvector(*reinterpret_cast<const f16x4*>(p + 32), f32x4);
      }
      const long long at = bz * os + row * rs + col;
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = fmaf(alpha, v[r], beta * x[r]);
      if constexpr (DT == TCMI_F32) out4<f32x4>((float*)out + at, x);
      else if constexpr (DT == TCMI_F16) out4<f16x4>((f16*)out + at, x);
      else if constexpr (DT == TCMI_BF16) out4<bf16x4>((__bf16*)out + at, x);
      return;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = col + r;
      if (j >= g.N) continue;
      const float x = fmaf(alpha, v[r], beta * old_x(line, j));
      if constexpr (DT == TCMI_C64) {
        const int im = j >= n;
        ((float*)out)[2 * (bz * os + row * rs + (j - im * n) * cs) + im] = x;
      } else {
        const long long at = bz * os + row * rs + j * cs;
        if (update) {
          const float old = DT == TCMI_F32 ? ((float*)out)[at] : DT == TCMI_F16 ? (float)((f16*)out)[at] : (float)((__bf16*)out)[at];
          put(out, DT, at, fmaf(rate, x, keep * old));
        } else {
          put(out, DT, at, x);
        }
      }
    }
  }
  template <class V4, class E>
  __device__ __forceinline__ void out4(E* p, f32x4 x) const {
    if (update) {
      const f32x4 old = __builtin_convertvector(*reinterpret_cast<const V4*>(p), f32x4);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = fmaf(rate, x[r], keep * old[r]);
    }
    *reinterpret_cast<V4*>(p) = __builtin_convertvector(x, V4);
  }
};

// dG = (D - X_0 <D, G> / |G|) / N, X_0 = G / N; d holds D, or D / dnorm
template <int SRC>
__global__ __launch_bounds__(256) void grad_out_kernel(Mat gm, const float* d, long long ldd, long long dbs, int m, int n,
                                                       const double* part, int npart, const double* norm, const double* dnorm, float eps, void* out,
                                                       long long rs, long long cs, long long os, int dtype) {
  __shared__ double red[4];
  const int bz = blockIdx.y;
  double s = 0.0;
  for (int k = threadIdx.x; k < npart; k += 256) s += part[(long long)bz * npart + k];
  const double inner = block_sum(s, red), nr = norm[bz], full = nr + (double)eps;
  const Factor inv = inverse(full), f1 = factor_of(full == 0.0 ? 0.0 : (dnorm ? dnorm[bz] : 1.0) / full);
  const float f2 = nr == 0.0 ? 0.f : (float)(inner / nr);
  const long long total = (long long)m * n;
  for (long long k = blockIdx.x * 256ll + threadIdx.x; k < total; k += gridDim.x * 256ll) {
    // the source decides the order: consecutive threads along its contiguous axis
    const long long i = gm.cs <= gm.rs ? k / n : k % m, j = gm.cs <= gm.rs ? k % n : k / m;
    const float2 g = fetch<SRC>(gm.p, bz * gm.bs + i * gm.rs + j * gm.cs);
    const float* dd = d + bz * dbs + i * ldd + j;
    const long long at = bz * os + i * rs + j * cs;
    if (SRC == SRC_C64) {
      ((float2*)out)[at] = make_float2(times(dd[0] - times(g.x, inv) * f2, f1), times(dd[n] - times(g.y, inv) * f2, f1));
    } else {
      put(out, dtype, at, times(dd[0] - times(g.x, inv) * f2, f1));
    }
  }
}

// The same two steps, <D, G> and dG, for a G that is contiguous along its columns (a matrix taller than wide): D lies across
// it, so 64 x 64 tiles of D pass through LDS (62 x 256 x 128 complex64: 17 + 15 us; read across 36 + 29).
struct TurnedArgs {
  Mat g;
  const float* d;
  long long ldd, dbs;
  int m, n, tx, tiles, npart;
  double* part;                  // [batch][npart]; the sums write it, one value a workgroup
  const double *norm, *dnorm;
  float eps;
  void* out;
  long long rs, cs, os;
  int dtype;
};

template <int SRC, bool OUT>
__global__ __launch_bounds__(256) void turned_kernel(TurnedArgs a) {
  __shared__ float re[64][65], im[SRC == SRC_C64 ? 64 : 1][65];
  __shared__ double red[4];
  const int bz = blockIdx.y, u = threadIdx.x & 63, w = threadIdx.x >> 6;
  double s = 0.0;
  Factor inv = {0.f, 0}, f1 = {0.f, 0};
  float f2 = 0.f;
  if (OUT) {
    for (int k = threadIdx.x; k < a.npart; k += 256) s += a.part[(long long)bz * a.npart + k];
    const double inner = block_sum(s, red), nr = a.norm[bz], full = nr + (double)a.eps;
    inv = inverse(full);
    f1 = factor_of(full == 0.0 ? 0.0 : (a.dnorm ? a.dnorm[bz] : 1.0) / full);
    f2 = nr == 0.0 ? 0.f : (float)(inner / nr);
  }
  for (int t = blockIdx.x; t < a.tiles; t += gridDim.x) {
    const int i0 = t / a.tx * 64, j0 = t % a.tx * 64;
    __syncthreads();
#pragma unroll 4
    for (int k = w; k < 64; k += 4)
      if (i0 + k < a.m && j0 + u < a.n) {
        const float* p = a.d + bz * a.dbs + (i0 + k) * a.ldd + j0 + u;
        re[k][u] = p[0];
        if (SRC == SRC_C64) im[SRC == SRC_C64 ? k : 0][u] = p[a.n];
      }
    __syncthreads();
#pragma unroll 4
    for (int k = w; k < 64; k += 4) {
      const int i = i0 + u, j = j0 + k;
      if (i >= a.m || j >= a.n) continue;
      const float2 g = fetch<SRC>(a.g.p, bz * a.g.bs + i * a.g.rs + j * a.g.cs);
      const float x = re[u][k], y = SRC == SRC_C64 ? im[SRC == SRC_C64 ? u : 0][k] : 0.f;
      if constexpr (OUT) {
        const long long at = bz * a.os + i * a.rs + j * a.cs;
        if constexpr (SRC == SRC_C64) ((float2*)a.out)[at] = make_float2(times(x - times(g.x, inv) * f2, f1), times(y - times(g.y, inv) * f2, f1));
        else put(a.out, a.dtype, at, times(x - times(g.x, inv) * f2, f1));
      } else {
        s += (double)g.x * x + (double)g.y * y;
      }
    }
  }
  if (!OUT) {
    s = block_sum(s, red);
    if (threadIdx.x == 0) a.part[(long long)bz * gridDim.x + blockIdx.x] = s;
  }
}

// ------------------------------------------------------------------------------------------- matrices that fit one CU
// One workgroup per matrix, everything in LDS, f32 matrix instructions (exact products): one launch instead of four per
// step.  Taken when a step's operands fit 160 KB of LDS and the columns are few (small_bytes).  Bound by the latency of the chain
// load -> norm -> 3 products a step -> store: five steps of a 24 x 28 matrix are 15 dependent products, 10.6 us of kernel
// (with branches around all eight tiles a wave could have, and the tiles' places kept per lane: 14.3).
// Fragments: of 16 consecutive k, lane group g = lane >> 4 takes k = 4 g .. 4 g + 3 (the sum does not care which lane holds
// which k), so a row operand is one 16-byte LDS read and a column operand four 4-byte reads; with rows 4 (mod 8) floats
// apart neither has bank conflicts.
struct SmallShape {
  int m, n, cx, R, C, R16, C16, ldx, lda;
};

__host__ __device__ inline SmallShape small_shape(int m, int n, int cx) {
  SmallShape s;
  s.m = m;
  s.n = n;
  s.cx = cx;
  s.R = cx * m;
  s.C = cx * n;
  s.R16 = (s.R + 15) & ~15;
  s.C16 = (s.C + 15) & ~15;
  s.ldx = s.C16 + 4;
  s.lda = s.R16 + 4;
  return s;
}

constexpr int SMALL_THREADS = 512, SMALL_WAVES = 8, SMALL_TILES = 8;        // 16 x 16 tiles per wave in the update, at most

struct SmallArgs {
  Mat src, dy;
  int m, n, cx, steps, flat;               // flat: 1 when the source is contiguous along n
  float coef[3 * TCMI_NS_MAX_STEPS];
  float eps;
  float* buf;
  long long brs, bcs, bbs;
  float rest;
  int nesterov;
  void* out;
  long long ors, ocs, obs;
  int dtype, update;
  float keep, rate;
  float* saved;                            // [batch][steps][m][C] iterates, then the norm: [batch] (null: not kept)
  double* norm;
};

__device__ __forceinline__ f32x4 mfma4(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
  for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
  return c;
}

// sum_k p[i][k] q[j][k] for one 16 x 16 tile; lane holds rows 4 (lane >> 4) + r, column lane & 15
__device__ __forceinline__ f32x4 rows_rows(const float* p, const float* q, int ld, int K, f32x4 c) {
  const int at = (threadIdx.x & 15) * ld + 4 * ((threadIdx.x & 63) >> 4);
  p += at;
  q += at;
  f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(q);
  for (int k = 16; k < K; k += 16) {                 // the next reads go out before the products that wait for these
    const f32x4 na = *reinterpret_cast<const f32x4*>(p + k), nb = *reinterpret_cast<const f32x4*>(q + k);
    __builtin_amdgcn_sched_barrier(0);
    c = mfma4(a, b, c);
    a = na;
    b = nb;
  }
  return mfma4(a, b, c);
}

// sum_k p[i][k] x[k][j]
__device__ __forceinline__ f32x4 rows_cols(const float* p, int ldp, const float* x, int ldx, int K, f32x4 c) {
  const int l = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
  p += l * ldp + 4 * g;
  x += 4 * g * ldx + l;
  f32x4 a = *reinterpret_cast<const f32x4*>(p), b = {x[0], x[ldx], x[2 * ldx], x[3 * ldx]};
  for (int k = 16; k < K; k += 16) {
    x += 16 * ldx;
    const f32x4 na = *reinterpret_cast<const f32x4*>(p + k), nb = {x[0], x[ldx], x[2 * ldx], x[3 * ldx]};
    __builtin_amdgcn_sched_barrier(0);
    c = mfma4(a, b, c);
    a = na;
    b = nb;
  }
  return mfma4(a, b, c);
}

__device__ __forceinline__ int small_wave() { return __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6); }

// f(i0, j0) for the tiles on and below the diagonal, dealt to the waves
template <class F>
__device__ __forceinline__ void lower_tiles(int R16, F f) {
  const int t = R16 / 16;
  int i = 0, j = small_wave();
  while (true) {
    while (j > i) j -= ++i;                          // a row of tiles holds one more than the one above
    if (i >= t) return;
    f(i * 16, j * 16);
    j += SMALL_WAVES;
  }
}

__device__ __forceinline__ void put_both(float* a, int lda, int i0, int j0, f32x4 v) {
  const int j = j0 + (threadIdx.x & 15), i = i0 + 4 * ((threadIdx.x & 63) >> 4);
#pragma unroll
  for (int r = 0; r < 4; ++r) a[(i + r) * lda + j] = v[r];
  *reinterpret_cast<f32x4*>(a + j * lda + i) = v;
}

__device__ __forceinline__ f32x4 get_tile(const float* a, int ld, int i0, int j0) {
  const float* p = a + (i0 + 4 * ((threadIdx.x & 63) >> 4)) * ld + j0 + (threadIdx.x & 15);
  return f32x4{p[0], p[ld], p[2 * ld], p[3 * ld]};
}

__device__ __forceinline__ double small_sum(double v, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int k = 0; k < SMALL_WAVES; ++k) v += red[k];
  return v;
}

__device__ __forceinline__ void embed(float* x, int ldx, const SmallShape& s, int i, int j, float2 v) {
  x[i * ldx + j] = v.x;
  if (s.cx == 2) {
    x[i * ldx + j + s.n] = v.y;
    x[(i + s.m) * ldx + j] = -v.y;
    x[(i + s.m) * ldx + j + s.n] = v.x;
  }
}

// element k of an m x n matrix, consecutive k along its contiguous axis
__device__ __forceinline__ void place(int k, int m, int n, int flat, int& i, int& j) {
  if (flat) {
    i = k / n;
    j = k - i * n;
  } else {
    j = k / m;
    i = k - j * m;
  }
}

__device__ __forceinline__ void gram(const float* X, float* A, const SmallShape& s) {
  lower_tiles(s.R16, [&](int i0, int j0) {
    put_both(A, s.lda, i0, j0, rows_rows(X + i0 * s.ldx, X + j0 * s.ldx, s.ldx, s.C16, f32x4{0.f, 0.f, 0.f, 0.f}));
  });
}

__device__ __forceinline__ void poly(const float* A, float* Bm, const SmallShape& s, float b, float c) {
  lower_tiles(s.R16, [&](int i0, int j0) {
    const f32x4 a = get_tile(A, s.lda, i0, j0);
    const f32x4 v = rows_rows(A + i0 * s.lda, A + j0 * s.lda, s.lda, s.R16, f32x4{0.f, 0.f, 0.f, 0.f});
    f32x4 o;
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = fmaf(c, v[r], b * a[r]);
    put_both(Bm, s.lda, i0, j0, o);
  });
}

// X <- a X + B X (+ Q Y): all waves finish reading before any writes
template <bool TWO, int SLOTS>
__device__ __forceinline__ void update(float* X, const float* Bm, const float* Q, const float* Y, const SmallShape& s, float a) {
  const int wave = small_wave(), tc = s.C16 / 16, tiles = tc * (s.R16 / 16);
  f32x4 res[SLOTS];
#pragma unroll
  for (int u = 0; u < SLOTS; ++u) {
    const int t = wave + u * SMALL_WAVES;
    if (t < tiles) {
      const int i0 = t / tc * 16, j0 = t % tc * 16;
      const f32x4 x = get_tile(X, s.ldx, i0, j0);
      f32x4 v = rows_cols(Bm + i0 * s.lda, s.lda, X + j0, s.ldx, s.R16, f32x4{0.f, 0.f, 0.f, 0.f});
      if (TWO) v = rows_cols(Q + i0 * s.lda, s.lda, Y + j0, s.ldx, s.R16, v);
#pragma unroll
      for (int r = 0; r < 4; ++r) res[u][r] = fmaf(a, x[r], v[r]);
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < SLOTS; ++u) {
    const int t = wave + u * SMALL_WAVES;
    if (t < tiles) {
      float* p = X + (t / tc * 16 + 4 * ((threadIdx.x & 63) >> 4)) * s.ldx + t % tc * 16 + (threadIdx.x & 15);
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r * s.ldx] = res[u][r];
    }
  }
  __syncthreads();
}

template <int SRC, int SLOTS>
__global__ __launch_bounds__(SMALL_THREADS) void small_kernel(SmallArgs a) {
  extern __shared__ __attribute__((aligned(16))) float mem[];
  __shared__ double red[SMALL_WAVES];
  const SmallShape s = small_shape(a.m, a.n, a.cx);
  float *X = mem, *A = X + s.R16 * s.ldx, *Bm = A + s.R16 * s.lda;
  const long long bz = blockIdx.x;
  for (int k = threadIdx.x; k < s.R16 * s.ldx; k += SMALL_THREADS) X[k] = 0.f;
  __syncthreads();
  double sum = 0.0;
  for (int k = threadIdx.x; k < s.m * s.n; k += SMALL_THREADS) {
    int i, j;
    place(k, s.m, s.n, a.flat, i, j);
    float2 v = fetch<SRC>(a.src.p, bz * a.src.bs + i * a.src.rs + j * a.src.cs);
    if (a.buf) {
      float* m = a.buf + bz * a.bbs + i * a.brs + j * a.bcs;
      const float nv = fmaf(a.rest, v.x - m[0], m[0]);
      m[0] = nv;
      v.x = direction(v.x, nv, a.rest, a.nesterov);
    }
    sum += (double)v.x * v.x + (double)v.y * v.y;
    embed(X, s.ldx, s, i, j, v);
  }
  const double nrm = sqrt(small_sum(sum, red)), full = nrm + (double)a.eps;
  if (a.norm && threadIdx.x == 0) a.norm[bz] = nrm;
  const Factor inv = inverse(full);
  for (int k = threadIdx.x; k < s.R16 * s.ldx; k += SMALL_THREADS) X[k] = times(X[k], inv);
  __syncthreads();
  for (int t = 0; t < a.steps; ++t) {
    if (a.saved) {
      float* w = a.saved + (bz * a.steps + t) * s.m * s.C;
      for (int k = threadIdx.x; k < s.m * s.C; k += SMALL_THREADS) w[k] = X[k / s.C * s.ldx + k % s.C];
    }
    const float ca = a.coef[3 * t], cb = a.coef[3 * t + 1], cc = a.coef[3 * t + 2];
    gram(X, A, s);
    __syncthreads();
    poly(A, Bm, s, cb, cc);
    __syncthreads();
    update<false, SLOTS>(X, Bm, nullptr, nullptr, s, ca);
  }
  for (int k = threadIdx.x; k < s.m * s.n; k += SMALL_THREADS) {
    int i, j;
    place(k, s.m, s.n, a.ocs <= a.ors, i, j);
    const float x = X[i * s.ldx + j];
    const long long at = bz * a.obs + i * a.ors + j * a.ocs;
    if (SRC == SRC_C64) {
      ((float2*)a.out)[at] = make_float2(x, X[i * s.ldx + j + s.n]);
    } else if (a.update) {
      const float old = SRC == SRC_F32 ? ((float*)a.out)[at] : SRC == SRC_F16 ? (float)((f16*)a.out)[at] : (float)((__bf16*)a.out)[at];
      put(a.out, a.dtype, at, fmaf(a.rate, x, a.keep * old));
    } else {
      put(a.out, a.dtype, at, x);
    }
  }
}

template <int SRC, int SLOTS>
__global__ __launch_bounds__(SMALL_THREADS) void small_grad_kernel(SmallArgs a) {
  extern __shared__ __attribute__((aligned(16))) float mem[];
  __shared__ double red[SMALL_WAVES];
  const SmallShape s = small_shape(a.m, a.n, a.cx);
  const int xs = s.R16 * s.ldx, as = s.R16 * s.lda;
  float *X = mem, *D = X + xs, *A = D + xs, *Bm = A + as, *S = Bm + as, *Q = S + as;
  const long long bz = blockIdx.x;
  for (int k = threadIdx.x; k < 2 * xs; k += SMALL_THREADS) X[k] = 0.f;
  __syncthreads();
  for (int k = threadIdx.x; k < s.m * s.n; k += SMALL_THREADS) {
    int i, j;
    place(k, s.m, s.n, a.dy.cs <= a.dy.rs, i, j);
    embed(D, s.ldx, s, i, j, fetch<SRC>(a.dy.p, bz * a.dy.bs + i * a.dy.rs + j * a.dy.cs));
  }
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  for (int t = a.steps - 1; t >= 0; --t) {
    const float *w = a.saved + (bz * a.steps + t) * s.m * s.C, ca = a.coef[3 * t], b = a.coef[3 * t + 1], c = a.coef[3 * t + 2];
    for (int k = threadIdx.x; k < s.m * s.n; k += SMALL_THREADS) {
      const int i = k / s.n, j = k % s.n;
      embed(X, s.ldx, s, i, j, make_float2(w[i * s.C + j], s.cx == 2 ? w[i * s.C + j + s.n] : 0.f));
    }
    __syncthreads();
    gram(X, A, s);
    lower_tiles(s.R16, [&](int i0, int j0) {
      f32x4 v = rows_rows(D + i0 * s.ldx, X + j0 * s.ldx, s.ldx, s.C16, zero);
      put_both(S, s.lda, i0, j0, rows_rows(X + i0 * s.ldx, D + j0 * s.ldx, s.ldx, s.C16, v));
    });
    __syncthreads();
    poly(A, Bm, s, b, c);
    lower_tiles(s.R16, [&](int i0, int j0) {
      f32x4 v = rows_rows(A + i0 * s.lda, S + j0 * s.lda, s.lda, s.R16, zero);
      v = rows_rows(S + i0 * s.lda, A + j0 * s.lda, s.lda, s.R16, v);
      const f32x4 g = get_tile(S, s.lda, i0, j0);
      f32x4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = fmaf(c, v[r], b * g[r]);
      put_both(Q, s.lda, i0, j0, o);
    });
    __syncthreads();
    update<true, SLOTS>(D, Bm, Q, X, s, ca);
  }
  double sum = 0.0;
  for (int k = threadIdx.x; k < s.m * s.n; k += SMALL_THREADS) {
    int i, j;
    place(k, s.m, s.n, a.flat, i, j);
    const float2 g = fetch<SRC>(a.src.p, bz * a.src.bs + i * a.src.rs + j * a.src.cs);
    sum += (double)g.x * D[i * s.ldx + j];
    if (SRC == SRC_C64) sum += (double)g.y * D[i * s.ldx + j + s.n];
  }
  const double inner = small_sum(sum, red), nr = a.norm[bz], full = nr + (double)a.eps;
  const Factor f1 = inverse(full);
  const float f2 = nr == 0.0 ? 0.f : (float)(inner / nr);
  for (int k = threadIdx.x; k < s.m * s.n; k += SMALL_THREADS) {
    int i, j;
    place(k, s.m, s.n, a.flat, i, j);
    const float2 g = fetch<SRC>(a.src.p, bz * a.src.bs + i * a.src.rs + j * a.src.cs);
    const long long at = bz * a.obs + i * a.ors + j * a.ocs;
    const float x = times(D[i * s.ldx + j] - times(g.x, f1) * f2, f1);
    if (SRC == SRC_C64) ((float2*)a.out)[at] = make_float2(x, times(D[i * s.ldx + j + s.n] - times(g.y, f1) * f2, f1));
    else put(a.out, a.dtype, at, x);
  }
}

// ------------------------------------------------------------------------------- few rows, long columns: two reads of G
// Every X of the iteration is a polynomial M of A_0 = X_0 X_0^H times X_0, so for a short side up to 64 (embedded) the steps
// run on m x m matrices alone: one pass forms G G^H, one workgroup iterates
//     P = a + b A + c A A,  M <- P M,  A <- P A P
// and a second pass writes M X_0.  A_k is no longer formed from X_k: an error of A_0 in a direction of small singular
// value grows by a^2 a step, 2e4 in five, so everything m x m is f64 (G G^H too: its products are exact, its sums f64).
// The gradient alike: D_k = U_k dY + V_k X_0 with U <- P U, V <- P V + Q M,
//     T = (U dY X_0^H + V A_0) M,  S = T + T^H,  Q = b S + c (A S + S A),
// from one pass for dY G^H and one for U dY + V X_0.
// In directions that G does not have M is the product of the steps' a, and what cancels there in M X_0 leaves its rounding
// behind: f32 sums hold while that product is small (steep), f64 ones (the second pass from 2^-53, 16 products for 1) until the
// rounding of A_0, which grows by its square, is felt; from there on the iterated forms take over, whose noise the steps
// themselves keep down.  Rows that occur twice, 32 x 1000, against 64 bits, 5 / 8 / 10 / 12 / 16 steps of the default: f32
// 9e-6 / 3e-4 / 3e-3 / 3e-2 / 5, f64 1e-13 / 2e-12 / 4e-11 / 6e-10 / 1e-7; of rank one, f64: 4e-13 / 1e-11 / 3e-9 / 5e-6 / 3.
// Bound by the reads of G for long sides, by the chain of small f64
// products (17 forward, 55 for the gradient) for short ones.  33 x 1088 x 9 f32: 28 us a call (large form: 325); gradient of 38 x 14 x 5789
// bf16: 157 us, most of it autograd's (3.0 ms).
typedef double f64x4 __attribute__((ext_vector_type(4)));
typedef double f64x2 __attribute__((ext_vector_type(2)));

constexpr int THIN_R = 64, THIN_GRAD_R = 32, THIN_COLS = 64, THIN_MAX_PART = 128;

struct ThinArgs {
  Mat g, dy;                     // rows = the short side
  int m, n, cx, steps, flat, dflat, chunks, parts;
  double coef[3 * TCMI_NS_MAX_STEPS];
  double eps;
  float* buf;
  long long brs, bcs, bbs;
  float rest;
  int nesterov;
  void* out;
  long long ors, ocs, obs;
  int dtype, update, oflat;
  float keep, rate;
  double* part;                  // [batch][parts][R16 R16]
  double* norm;                  // [batch]
  double* a0;                    // [batch][R16 R16], kept for the gradient (null: not kept)
  double* steps_mem;             // gradient: [batch][steps][3][R16 R16] P, M, A
  double *m1, *m2;               // [batch][R16 R16]: out = m1 X_0, or (m1 dY + m2 X_0) / N
};

__device__ __forceinline__ f64x4 mfma64(double a, double b, f64x4 c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }

// loads columns [j0, j0 + 64) of a matrix into LDS rows of ld floats, embedded, zero outside
template <int SRC, bool BUF>
__device__ __forceinline__ void thin_load(float* x, int ld, const ThinArgs& a, const Mat& src, int flat, long long bz, int j0, bool momentum) {
  const int R16 = (a.cx * a.m + 15) & ~15;
  for (int k = threadIdx.x; k < R16 * ld; k += 256) x[k] = 0.f;
  __syncthreads();
  const int cols = min(THIN_COLS, a.n - j0);
  for (int k = threadIdx.x; k < a.m * THIN_COLS; k += 256) {
    int i, j;
    if (flat) {
      i = k / THIN_COLS;
      j = k % THIN_COLS;
    } else {
      j = k / a.m;
      i = k - j * a.m;
    }
    if (j >= cols) continue;
    float2 v = fetch<SRC>(src.p, bz * src.bs + i * src.rs + (long long)(j0 + j) * src.cs);
    if (BUF && a.buf) {
      float* m = a.buf + bz * a.bbs + i * a.brs + (long long)(j0 + j) * a.bcs;
      float nv = m[0];
      if (momentum) {
        nv = fmaf(a.rest, v.x - nv, nv);
        m[0] = nv;
      }
      v.x = direction(v.x, nv, a.rest, a.nesterov);
    }
    x[i * ld + j] = v.x;
    if (a.cx == 2) {
      x[i * ld + j + THIN_COLS] = v.y;
      x[(i + a.m) * ld + j] = -v.y;
      x[(i + a.m) * ld + j + THIN_COLS] = v.x;
    }
  }
  __syncthreads();
}

// partial sums of G G^H (lower tiles), or of G dY^H (all tiles)
template <int SRC, bool GRAD>
__global__ __launch_bounds__(256) void thin_gram_kernel(ThinArgs a) {
  extern __shared__ __attribute__((aligned(16))) float mem[];
  const int R16 = (a.cx * a.m + 15) & ~15, w = a.cx * THIN_COLS, ld = w + 4, tr = R16 / 16;
  const long long bz = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  float *X = mem, *D = mem + R16 * ld;
  f64x4 acc[4] = {};
  for (int c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    thin_load<SRC, !GRAD>(X, ld, a, a.g, a.flat, bz, c * THIN_COLS, true);
    if (GRAD) thin_load<SRC, false>(D, ld, a, a.dy, a.dflat, bz, c * THIN_COLS, false);
    int t = 0, u = 0;
#pragma unroll
    for (int q = 0; q < 16; ++q) {
      const int i = q / 4, j = q % 4;
      if (i >= tr || j >= tr || (!GRAD && j > i)) continue;
      if (t++ % 4 != wave) continue;
      const float* p = X + (i * 16 + l) * ld + 4 * g;
      const float* s = (GRAD ? D : X) + (j * 16 + l) * ld + 4 * g;
      f64x4 v = u == 0 ? acc[0] : u == 1 ? acc[1] : u == 2 ? acc[2] : acc[3];
      for (int k = 0; k < w; k += 16) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(p + k), y = *reinterpret_cast<const f32x4*>(s + k);
#pragma unroll
        for (int r = 0; r < 4; ++r) v = mfma64((double)x[r], (double)y[r], v);
      }
      if (u == 0) acc[0] = v;
      else if (u == 1) acc[1] = v;
      else if (u == 2) acc[2] = v;
      else acc[3] = v;
      ++u;
    }
    __syncthreads();
  }
  double* out = a.part + (bz * gridDim.x + blockIdx.x) * R16 * R16;
  int t = 0, u = 0;
#pragma unroll
  for (int q = 0; q < 16; ++q) {
    const int i = q / 4, j = q % 4;
    if (i >= tr || j >= tr || (!GRAD && j > i)) continue;
    if (t++ % 4 != wave) continue;
    const f64x4 v = u == 0 ? acc[0] : u == 1 ? acc[1] : u == 2 ? acc[2] : acc[3];
    ++u;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = i * 16 + g + 4 * r, col = j * 16 + l;
      out[row * R16 + col] = v[r];
      if (!GRAD && i != j) out[col * R16 + row] = v[r];
    }
  }
}

constexpr int THIN_THREADS = 512;

// c += sum_k p[i][k] q[j][k], rows ld doubles apart
__device__ __forceinline__ f64x4 rows64(const double* p, const double* q, int ld, int R16, f64x4 c) {
  const int l = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
  p += l * ld + 2 * g;
  q += l * ld + 2 * g;
  f64x2 x = *reinterpret_cast<const f64x2*>(p), y = *reinterpret_cast<const f64x2*>(q);
  for (int k = 8; k < R16; k += 8) {                 // the next reads go out before the products that wait for these
    const f64x2 nx = *reinterpret_cast<const f64x2*>(p + k), ny = *reinterpret_cast<const f64x2*>(q + k);
    __builtin_amdgcn_sched_barrier(0);
    c = mfma64(x[0], y[0], c);
    c = mfma64(x[1], y[1], c);
    x = nx;
    y = ny;
  }
  c = mfma64(x[0], y[0], c);
  return mfma64(x[1], y[1], c);
}

// f(i0, j0) for the tiles dealt to the waves; LOWER: on and below the diagonal
template <bool LOWER, class F>
__device__ __forceinline__ void tiles64(int R16, F f) {
  const int wave = threadIdx.x >> 6, t = R16 / 16;
  int k = 0;
  for (int i = 0; i < t; ++i)
    for (int j = 0; j < (LOWER ? i + 1 : t); ++j, ++k)
      if (k % (THIN_THREADS / 64) == wave) f(i * 16, j * 16);
}

template <class F>
__device__ __forceinline__ void cells64(int i0, int j0, f64x4 v, F f) {        // f(row, col, value) of a tile's four cells
  const int l = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int r = 0; r < 4; ++r) f(i0 + g + 4 * r, j0 + l, v[r]);
}

// A cell on or below the diagonal and its mirror image.  Cells above it in a tile on the diagonal are left out: the rounding of
// p q and of its transpose differ, and a matrix that holds some of each is not symmetric, which the next products multiply by
// the square of what M grows to (8 x 1000 of rank 4, ten steps: 6e-5 of the result instead of 3e-9).
__device__ __forceinline__ void put_sym(double* out, int ld, int i, int j, double x) {
  if (j > i) return;
  out[i * ld + j] = x;
  out[j * ld + i] = x;
}

// out = sym(p q) for commuting symmetric p, q: lower tiles, written twice
__device__ __forceinline__ void sym64(const double* p, const double* q, double* out, int ld, int R16) {
  tiles64<true>(R16, [&](int i0, int j0) {
    cells64(i0, j0, rows64(p + i0 * ld, q + j0 * ld, ld, R16, f64x4{0, 0, 0, 0}), [&](int i, int j, double x) { put_sym(out, ld, i, j, x); });
  });
}

__device__ __forceinline__ void poly64(const double* A, double* P, int ld, int R16, double a, double b, double c) {
  tiles64<true>(R16, [&](int i0, int j0) {
    cells64(i0, j0, rows64(A + i0 * ld, A + j0 * ld, ld, R16, f64x4{0, 0, 0, 0}), [&](int i, int j, double x) {
      put_sym(P, ld, i, j, c * x + b * A[i * ld + j] + (i == j ? a : 0.0));
    });
  });
}

// the iteration on m x m matrices; STEPS: P, M (before the step) and A of every step go to memory for the gradient
template <bool STEPS>
__device__ __forceinline__ void thin_iterate(const ThinArgs& a, double* A, double* P, double* M, double* T, int ld, int R16, long long bz) {
  for (int k = threadIdx.x; k < R16 * R16; k += THIN_THREADS) M[k / R16 * ld + k % R16] = k / R16 == k % R16 ? 1.0 : 0.0;
  for (int t = 0; t < a.steps; ++t) {
    __syncthreads();
    poly64(A, P, ld, R16, a.coef[3 * t], a.coef[3 * t + 1], a.coef[3 * t + 2]);
    __syncthreads();
    if (STEPS) {
      double* w = a.steps_mem + (bz * a.steps + t) * 3 * R16 * R16;
      for (int k = threadIdx.x; k < R16 * R16; k += THIN_THREADS) {
        const int at = k / R16 * ld + k % R16;
        w[k] = P[at];
        w[R16 * R16 + k] = M[at];
        w[2 * R16 * R16 + k] = A[at];
      }
      if (t + 1 == a.steps) break;
    }
    sym64(P, M, T, ld, R16);
    __syncthreads();
    double* x = M;
    M = T;
    T = x;
    if (t + 1 < a.steps) {
      sym64(P, A, T, ld, R16);
      __syncthreads();
      sym64(P, T, A, ld, R16);
    }
  }
  __syncthreads();
  if (!STEPS) {
    for (int k = threadIdx.x; k < R16 * R16; k += THIN_THREADS) a.m1[bz * R16 * R16 + k] = M[k / R16 * ld + k % R16];
  }
}

// sum of the parts of a pass, in a fixed order
__device__ __forceinline__ double part_sum(const ThinArgs& a, long long bz, int R16, int k) {
  double s = 0.0;
  const double* p = a.part + bz * a.parts * R16 * R16 + k;
#pragma unroll 4
  for (int i = 0; i < a.parts; ++i) s += p[(long long)i * R16 * R16];
  return s;
}

__global__ __launch_bounds__(THIN_THREADS) void thin_poly_kernel(ThinArgs a) {
  extern __shared__ __attribute__((aligned(16))) double mem64[];
  __shared__ double nrm;
  const int R = a.cx * a.m, R16 = (R + 15) & ~15, ld = R16 + 2, sz = R16 * ld;
  const long long bz = blockIdx.x;
  double *A = mem64, *P = A + sz, *M = P + sz, *T = M + sz;
  for (int k = threadIdx.x; k < R16 * R16; k += THIN_THREADS) A[k / R16 * ld + k % R16] = part_sum(a, bz, R16, k);
  __syncthreads();
  if (threadIdx.x < 64) {                     // |G|^2 is the trace (of the upper block)
    double s = threadIdx.x < a.m ? A[threadIdx.x * ld + threadIdx.x] : 0.0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (threadIdx.x == 0) {
      nrm = sqrt(s);
      a.norm[bz] = nrm;
    }
  }
  __syncthreads();
  const double n = nrm + a.eps, inv = n == 0.0 ? 0.0 : 1.0 / (n * n);
  for (int k = threadIdx.x; k < R16 * R16; k += THIN_THREADS) {
    double& x = A[k / R16 * ld + k % R16];
    x *= inv;
    if (a.a0) a.a0[bz * R16 * R16 + k] = x;
  }
  thin_iterate<false>(a, A, P, M, T, ld, R16, bz);
}

__global__ __launch_bounds__(THIN_THREADS) void thin_grad_poly_kernel(ThinArgs a) {
  extern __shared__ __attribute__((aligned(16))) double mem64[];
  __shared__ double tr;
  const int R = a.cx * a.m, R16 = (R + 15) & ~15, ld = R16 + 2, sz = R16 * ld, q2 = R16 * R16;
  const long long bz = blockIdx.x;
  double *A0 = mem64, *Wt = A0 + sz, *U = Wt + sz, *V = U + sz, *Vt = V + sz, *P = Vt + sz, *M = P + sz, *A = M + sz, *Z = A + sz, *S = Z + sz,
         *Q = S + sz;
  const double nr = a.norm[bz], n = nr + a.eps, inv = n == 0.0 ? 0.0 : 1.0 / n;
  for (int k = threadIdx.x; k < q2; k += THIN_THREADS) {
    const int i = k / R16, j = k % R16, at = i * ld + j;
    A0[at] = A[at] = a.a0[bz * q2 + k];
    Wt[at] = part_sum(a, bz, R16, k) * inv;        // G dY^H / N = (dY X_0^H)^H
    U[at] = i == j ? 1.0 : 0.0;
    V[at] = Vt[at] = 0.0;
  }
  __syncthreads();
  thin_iterate<true>(a, A, P, M, Z, ld, R16, bz);
  const f64x4 zero = {0, 0, 0, 0};
  for (int t = a.steps - 1; t >= 0; --t) {
    const double* w = a.steps_mem + (bz * a.steps + t) * 3 * q2;
    const double b = a.coef[3 * t + 1], c = a.coef[3 * t + 2];
    __syncthreads();
    for (int k = threadIdx.x; k < q2; k += THIN_THREADS) {
      const int at = k / R16 * ld + k % R16;
      P[at] = w[k];
      M[at] = w[q2 + k];
      A[at] = w[2 * q2 + k];
    }
    __syncthreads();
    tiles64<false>(R16, [&](int i0, int j0) {      // Z = U W + V A_0
      f64x4 v = rows64(U + i0 * ld, Wt + j0 * ld, ld, R16, zero);
      v = rows64(V + i0 * ld, A0 + j0 * ld, ld, R16, v);
      cells64(i0, j0, v, [&](int i, int j, double x) { Z[i * ld + j] = x; });
    });
    __syncthreads();
    tiles64<false>(R16, [&](int i0, int j0) {      // Q holds T = Z M for the moment
      cells64(i0, j0, rows64(Z + i0 * ld, M + j0 * ld, ld, R16, zero), [&](int i, int j, double x) { Q[i * ld + j] = x; });
    });
    __syncthreads();
    for (int k = threadIdx.x; k < q2; k += THIN_THREADS) {
      const int i = k / R16, j = k % R16;
      S[i * ld + j] = Q[i * ld + j] + Q[j * ld + i];
    }
    __syncthreads();
    tiles64<true>(R16, [&](int i0, int j0) {       // Q = b S + c (A S + S A)
      f64x4 v = rows64(A + i0 * ld, S + j0 * ld, ld, R16, zero);
      v = rows64(S + i0 * ld, A + j0 * ld, ld, R16, v);
      cells64(i0, j0, v, [&](int i, int j, double x) { put_sym(Q, ld, i, j, c * x + b * S[i * ld + j]); });
    });
    __syncthreads();
    sym64(P, U, Z, ld, R16);                       // U <- P U
    tiles64<false>(R16, [&](int i0, int j0) {      // V <- P V + Q M, kept with its transpose
      f64x4 v = rows64(P + i0 * ld, Vt + j0 * ld, ld, R16, zero);
      v = rows64(Q + i0 * ld, M + j0 * ld, ld, R16, v);
      cells64(i0, j0, v, [&](int i, int j, double x) { S[i * ld + j] = x; });
    });
    __syncthreads();
    for (int k = threadIdx.x; k < q2; k += THIN_THREADS) {
      const int i = k / R16, j = k % R16;
      V[i * ld + j] = S[i * ld + j];
      Vt[j * ld + i] = S[i * ld + j];
      U[i * ld + j] = Z[i * ld + j];
    }
  }
  __syncthreads();
  // <D, X_0> = trace of U W + V A_0 (half of the embedded one)
  double s = 0.0;
  for (int k = threadIdx.x; k < q2; k += THIN_THREADS) {
    const int i = k / R16, j = k % R16;
    s += U[i * ld + j] * Wt[i * ld + j] + V[i * ld + j] * A0[i * ld + j];
  }
  __shared__ double red[THIN_THREADS / 64];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int k = 0; k < THIN_THREADS / 64; ++k) s += red[k];
    tr = s / a.cx;
  }
  __syncthreads();
  // dG = (D - G <D, G> / (N |G|)) / N, D = U dY + V X_0, <D, G> = N <D, X_0>, G = N X_0
  const double f = nr == 0.0 ? 0.0 : tr * n / nr;
  for (int k = threadIdx.x; k < q2; k += THIN_THREADS) {
    const int i = k / R16, j = k % R16;
    a.m1[bz * q2 + k] = U[i * ld + j];
    a.m2[bz * q2 + k] = V[i * ld + j] - (i == j ? f : 0.0);
  }
}

// c += sum_k p[i][k] x[k][j], p in f64, x exact f32
__device__ __forceinline__ f64x4 rows_cols64(const double* p, int ldp, const float* x, int ldx, int K, f64x4 c) {
  const int l = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
  p += l * ldp + g;
  x += g * ldx + l;
  for (int k = 0; k < K; k += 4) c = mfma64(p[k], (double)x[k * ldx], c);
  return c;
}

// out = m1 X_0, or (m1 dY + m2 X_0) / N, X_0 = G / N, 64 columns a workgroup.  S: the type of the products and sums; in f64
// G is divided behind them, as rounding G / N would already cost what f64 is there to save.
template <int SRC, bool GRAD, class S>
__global__ __launch_bounds__(256) void thin_apply_kernel(ThinArgs a) {
  extern __shared__ __attribute__((aligned(16))) float mem[];
  constexpr bool WIDE = std::is_same<S, double>::value;
  const int R16 = (a.cx * a.m + 15) & ~15, M16 = (a.m + 15) & ~15, w = a.cx * THIN_COLS, ld = w + 4, ldm = R16 + (WIDE ? 2 : 4);
  const long long bz = blockIdx.y;
  const int j0 = blockIdx.x * THIN_COLS, wave = threadIdx.x >> 6, tc = w / 16, tiles = tc * (M16 / 16);
  const int l = threadIdx.x & 15, q = (threadIdx.x & 63) >> 4;
  float *X = mem, *D = X + R16 * ld;
  S *M1 = reinterpret_cast<S*>(mem + (GRAD ? 2 : 1) * R16 * ld), *M2 = M1 + R16 * ldm;
  for (int k = threadIdx.x; k < R16 * R16; k += 256) {
    M1[k / R16 * ldm + k % R16] = (S)a.m1[bz * R16 * R16 + k];
    if (GRAD) M2[k / R16 * ldm + k % R16] = (S)a.m2[bz * R16 * R16 + k];
  }
  thin_load<SRC, !GRAD>(X, ld, a, a.g, a.flat, bz, j0, false);
  if (GRAD) thin_load<SRC, false>(D, ld, a, a.dy, a.dflat, bz, j0, false);
  const double full = a.norm[bz] + a.eps;
  const Factor inv = inverse(full);
  const double inv64 = full == 0.0 ? 0.0 : 1.0 / full;
  if constexpr (!WIDE) {
    for (int k = threadIdx.x; k < R16 * ld; k += 256) X[k] = times(X[k], inv);
    __syncthreads();
  }
  f32x4 res[8];                                    // at most 64 x 128 results: 32 tiles, 8 a wave
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int t = wave + u * 4;
    if (t >= tiles) continue;
    const int i0 = t / tc * 16, c0 = t % tc * 16;
    if constexpr (WIDE) {
      f64x4 v = rows_cols64((GRAD ? M2 : M1) + i0 * ldm, ldm, X + c0, ld, R16, f64x4{0.0, 0.0, 0.0, 0.0});
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] *= inv64;
      if (GRAD) v = rows_cols64(M1 + i0 * ldm, ldm, D + c0, ld, R16, v);
#pragma unroll
      for (int r = 0; r < 4; ++r) res[u][r] = (float)v[r];
    } else {
      f32x4 v = rows_cols((GRAD ? M2 : M1) + i0 * ldm, ldm, X + c0, ld, R16, f32x4{0.f, 0.f, 0.f, 0.f});
      if (GRAD) v = rows_cols(M1 + i0 * ldm, ldm, D + c0, ld, R16, v);
      res[u] = v;
    }
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < 8; ++u) {
    const int t = wave + u * 4;
    if (t >= tiles) continue;
    float* p = X + t / tc * 16 * ld + t % tc * 16 + l;        // rows 4 q + r of the tile; q + 4 r from the f64 instruction
#pragma unroll
    for (int r = 0; r < 4; ++r) p[(WIDE ? q + 4 * r : 4 * q + r) * ld] = res[u][r];
  }
  __syncthreads();
  const int cols = min(THIN_COLS, a.n - j0);
  for (int k = threadIdx.x; k < a.m * THIN_COLS; k += 256) {
    int i, j;
    if (a.oflat) {
      i = k / THIN_COLS;
      j = k % THIN_COLS;
    } else {
      j = k / a.m;
      i = k - j * a.m;
    }
    if (j >= cols) continue;
    const Factor by = GRAD ? inv : Factor{1.f, 0};
    const float x = times(X[i * ld + j], by);
    const long long at = bz * a.obs + i * a.ors + (long long)(j0 + j) * a.ocs;
    if (SRC == SRC_C64) {
      ((float2*)a.out)[at] = make_float2(x, times(X[i * ld + j + THIN_COLS], by));
    } else if (!GRAD && a.update) {
      const float old = SRC == SRC_F32 ? ((float*)a.out)[at] : SRC == SRC_F16 ? (float)((f16*)a.out)[at] : (float)((__bf16*)a.out)[at];
      put(a.out, a.dtype, at, fmaf(a.rate, x, a.keep * old));
    } else {
      put(a.out, a.dtype, at, x);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- host side
struct Shape {
  int m, n;                       // min, max of the caller's two dimensions
  bool flip;                      // the caller's matrix is taller than wide: X is its transpose
  int cx;                         // 2 for complex
  int mr, nc;                     // size of the (embedded) real matrix
  int P;                          // pieces per operand
  long long mp, np;               // stored row lengths over mr and nc: padded, times the pieces
  long long ldc;                  // f32 rows of the carry
  int batch;
};

Shape shape_of(int rows, int cols, int batch, int dtype, bool full) {
  Shape s;
  s.flip = rows > cols;
  s.m = s.flip ? cols : rows;
  s.n = s.flip ? rows : cols;
  s.cx = dtype == TCMI_C64 ? 2 : 1;
  s.mr = s.cx * s.m;
  s.nc = s.cx * s.n;
  s.P = full ? 2 : 1;
  s.mp = s.P * kpad(s.mr, s.P);
  s.np = s.P * kpad(s.nc, s.P);
  s.ldc = (s.nc + 3ll) & ~3ll;
  s.batch = batch;
  return s;
}

struct Arena {                    // hands out 256-byte aligned pieces of a caller's buffer (base null: only counts)
  char* base;
  long long used = 0;
  template <class P>
  P* take(long long count) {
    P* p = base ? reinterpret_cast<P*>(base + used) : nullptr;
    used += (count * (long long)sizeof(P) + 255) & ~255ll;
    return p;
  }
};

struct Pieces {                   // one step's operands
  f16 *x, *t, *a, *b;
};

Pieces take_pieces(Arena& w, const Shape& s) {
  Pieces p;
  p.x = w.take<f16>(s.mr * s.np * s.batch);
  p.t = w.take<f16>(s.nc * s.mp * s.batch);
  p.a = w.take<f16>(s.mr * s.mp * s.batch);
  p.b = w.take<f16>(s.mr * s.mp * s.batch);
  return p;
}

constexpr int MAX_PART = 1024;

struct Work {
  double *part, *norm;
  float *carry, *split;
  Pieces p;
  f16* t2;                        // X^T changes places with this: a step's product reads one while it writes the other
};

Work take_work(Arena& w, const Shape& s, bool saved) {
  Work k{};
  k.part = w.take<double>((long long)s.batch * MAX_PART);
  k.norm = w.take<double>(s.batch);
  k.carry = w.take<float>(s.m * s.ldc * s.batch);
  k.split = w.take<float>(PART_BYTES / 4);
  if (!saved) {
    k.p = take_pieces(w, s);
    k.t2 = w.take<f16>(s.nc * s.mp * s.batch);
  }
  return k;
}

struct Saved {
  double* norm;
  Pieces p[TCMI_NS_MAX_STEPS];
};

Saved take_saved(Arena& w, const Shape& s, int steps) {
  Saved v{};
  v.norm = w.take<double>(s.batch);
  for (int i = 0; i < steps; ++i) v.p[i] = take_pieces(w, s);
  return v;
}

struct GradWork {
  double *part, *norm;
  float *carry, *split;
  f16 *d, *t, *t2, *s, *q;
};

GradWork take_grad(Arena& w, const Shape& s) {
  GradWork k{};
  k.part = w.take<double>((long long)s.batch * MAX_PART);
  k.norm = w.take<double>(s.batch);
  k.carry = w.take<float>(s.m * s.ldc * s.batch);
  k.split = w.take<float>(PART_BYTES / 4);
  k.d = w.take<f16>(s.mr * s.np * s.batch);
  k.t = w.take<f16>(s.nc * s.mp * s.batch);
  k.t2 = w.take<f16>(s.nc * s.mp * s.batch);
  k.s = w.take<f16>(s.mr * s.mp * s.batch);
  k.q = w.take<f16>(s.mr * s.mp * s.batch);
  return k;
}

// What bounds the operands of a step whose X has singular values in [0, s]: x for X, A = s^2, B = max |b t + c t^2|, next = max |p|,
// slope = max |p'|, by which a step can lengthen a derivative: its gains are divided differences of the odd p,
// factor = max |p(t) / t|, what it can multiply a direction by.
struct Bound {
  double x, A, B, next, slope, factor;
};

Bound bound_of(double s, const double* co) {
  const double a = co[0], b = co[1], c = co[2], t1 = s * s;
  Bound r{s, t1, fabs(b * t1 + c * t1 * t1), 0.0, 0.0, fmax(fabs(a), fabs(a + b * t1 + c * t1 * t1))};
  if (c != 0.0) {
    const double t = -b / (2 * c);
    if (t > 0 && t < t1) {
      r.B = fmax(r.B, fabs(b * t + c * t * t));
      r.factor = fmax(r.factor, fabs(a + b * t + c * t * t));
    }
  }
  auto p = [&](double t) { return fabs(sqrt(t) * (a + b * t + c * t * t)); };
  auto slope = [&](double t) { return fabs(a + 3 * b * t + 5 * c * t * t); };
  r.slope = fmax(slope(0.0), slope(t1));
  if (c != 0.0 && -0.3 * b / c > 0 && -0.3 * b / c < t1) r.slope = fmax(r.slope, slope(-0.3 * b / c));
  r.next = p(t1);
  const double disc = 9 * b * b - 20 * a * c;
  if (c != 0.0 && disc >= 0) {
    const double u = (-3 * b + sqrt(disc)) / (10 * c), v = (-3 * b - sqrt(disc)) / (10 * c);
    if (u > 0 && u < t1) r.next = fmax(r.next, p(u));
    if (v > 0 && v < t1) r.next = fmax(r.next, p(v));
  } else if (c == 0.0 && b != 0.0) {
    const double u = -a / (3 * b);
    if (u > 0 && u < t1) r.next = fmax(r.next, p(u));
  }
  return r;
}

// the largest power of two that keeps values up to `bound` below 2^15
float scale_for(double bound) {
  if (!(bound > 0)) return 1.f;
  int e;
  frexp(bound, &e);               // bound < 2^e
  e = 15 - e;
  return (float)ldexp(1.0, e > 30 ? 30 : e);
}

constexpr double SLACK = 1.02;    // rounding may carry a singular value past its bound
constexpr double MAX_S = 64.0;

struct Scales {
  float x, A, B;
};

bool scales_of(int steps, const double* coef, Scales* out) {
  double s = 1.0;
  for (int i = 0; i < steps; ++i) {
    const Bound b = bound_of(s * SLACK, coef + 3 * i);
    if (!(b.x <= MAX_S) || !(b.B <= 1024.0) || !isfinite(b.next)) return false;
    out[i] = {scale_for(b.x), scale_for(b.A), scale_for(b.B)};
    s = b.next;
  }
  return s * SLACK <= MAX_S;
}

// what the steps together can multiply a direction by; infinite without coefficients
double growth_of(int steps, const double* coef) {
  if (!coef) return INFINITY;
  double s = 1.0, g = 1.0;
  for (int i = 0; i < steps; ++i) {
    const Bound b = bound_of(s * SLACK, coef + 3 * i);
    g *= fmax(1.0, b.factor);
    s = b.next;
  }
  return g == g ? g : INFINITY;
}

template <int P, class Epi>
hipError_t run(Args& g, bool tri, const Epi& e, hipStream_t st) {
  return launch_best<f16x8, P>(g, tri, e, st);
}

int sum_blocks(const Shape& s) {
  long long n = (long long)s.m * s.n / 1024;
  const int cap = s.batch >= 64 ? 16 : s.batch >= 8 ? 64 : s.batch > 1 ? 256 : MAX_PART;
  return (int)(n < 1 ? 1 : n > cap ? cap : n);
}

// whether four neighbours along the contiguous axis (stride cs) form one aligned load
bool aligned4(const void* p, long long rs, long long cs, long long bs, int size) {
  return cs == 1 && rs % 4 == 0 && bs % 4 == 0 && ((uintptr_t)p & (4 * size - 1)) == 0;
}

template <int MODE>
hipError_t launch_sums(int src, SumArgs a, int blocks, int batch, hipStream_t st) {
  // the contiguous axis inside; the sum does not care which of the two is called rows
  if (a.x.rs < a.x.cs && a.outer > 0) {
    long long t = a.x.rs; a.x.rs = a.x.cs; a.x.cs = t;
    t = a.y.rs; a.y.rs = a.y.cs; a.y.cs = t;
    if (MODE == 2) { t = a.brs; a.brs = a.bcs; a.bcs = t; }
    const int o = a.outer; a.outer = a.inner; a.inner = o;
  }
  a.vec = src != SRC_C64 && aligned4(a.x.p, a.x.rs, a.x.cs, a.x.bs, src == SRC_F32 ? 4 : 2) &&
          (MODE != 2 || aligned4(a.buf, a.brs, a.bcs, a.bbs, 4));
  const int wide = a.vec ? (a.inner + 3) / 4 : a.inner;
  a.lanes = wide > 128 ? 256 : wide > 64 ? 128 : wide > 32 ? 64 : wide > 16 ? 32 : 16;
  const dim3 grid(blocks, batch);
  if (src == SRC_F32) hipLaunchKernelGGL((sums_kernel<SRC_F32, MODE>), grid, dim3(256), 0, st, a);
  else if (src == SRC_F16) hipLaunchKernelGGL((sums_kernel<SRC_F16, MODE>), grid, dim3(256), 0, st, a);
  else if (src == SRC_BF16) hipLaunchKernelGGL((sums_kernel<SRC_BF16, MODE>), grid, dim3(256), 0, st, a);
  else if constexpr (MODE != 2) hipLaunchKernelGGL((sums_kernel<SRC_C64, MODE>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <int P>
hipError_t launch_pack(int src, PackArgs a, const Shape& s, hipStream_t st) {
  a.m = s.m;
  a.n = s.n;
  a.tx = (s.n + 63) / 64;
  a.ty = (s.m + 63) / 64;
  a.embed = s.cx == 2;
  a.fast_rows = a.src.rs < a.src.cs;
  a.vec = src != SRC_C64 && aligned4(a.src.p, a.fast_rows ? a.src.cs : a.src.rs, a.fast_rows ? a.src.rs : a.src.cs, a.src.bs,
                                     src == SRC_F32 || src == SRC_PLANAR ? 4 : 2);
  a.ld = s.np;
  a.os = s.mr * s.np;
  a.ldt = s.mp;
  a.ts = s.nc * s.mp;
  a.ldc = s.ldc;
  a.cbs = s.m * s.ldc;
  const long long blocks = (long long)a.tx * a.ty * s.batch;
  if (blocks >= (1ll << 31)) return hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks);
  if (src == SRC_F32) hipLaunchKernelGGL((pack_kernel<SRC_F32, P>), grid, dim3(256), 0, st, a);
  else if (src == SRC_F16) hipLaunchKernelGGL((pack_kernel<SRC_F16, P>), grid, dim3(256), 0, st, a);
  else if (src == SRC_BF16) hipLaunchKernelGGL((pack_kernel<SRC_BF16, P>), grid, dim3(256), 0, st, a);
  else if (src == SRC_C64) hipLaunchKernelGGL((pack_kernel<SRC_C64, P>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((pack_kernel<SRC_PLANAR, P>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t clear(void* p, long long bytes, hipStream_t st) {
  const long long n = bytes / 16;
  const long long b = (n + 255) / 256;
  hipLaunchKernelGGL(clear_kernel, dim3((unsigned)(b > 4096 ? 4096 : b < 1 ? 1 : b)), dim3(256), 0, st, (uint4*)p, n);
  return hipGetLastError();
}

Args base_args(const Shape& s, float* split, int M, int N, long long K, long long ld, long long sa, long long sb) {
  Args g{};
  g.M = M;
  g.N = N;
  g.K = (int)K;
  g.lda = g.ldb = ld;
  g.sa = sa;
  g.sb = sb;
  g.batch = s.batch;
  g.doubled = s.cx == 2 ? s.m : 0;
  g.part = split;
  return g;
}

void pair(Args& g, const f16* a, const f16* b) {
  g.a[g.nseg] = a;
  g.b[g.nseg] = b;
  ++g.nseg;
}

constexpr int SMALL_LDS = 156 * 1024;        // of 160 KB: the reductions take a little

// The two-pass form's results are off by the growth times the rounding of its last product, 2^-24 in f32 (600 holds five steps
// of the default, 485, at 9e-6 to 6e-5), and by the growth's square times 2^-53 times the root of the columns: 2^18, ten
// steps of the default, leaves 1e-3 of its margin at 2^24 columns.
constexpr double GROWTH_F32 = 600.0, THIN_GROWTH = 262144.0;

bool thin_fits(const Shape& s, bool grad, double growth) { return growth <= THIN_GROWTH && s.mr <= (grad ? THIN_GRAD_R : THIN_R); }

// Where the two-pass form could take the matrix too, the one-workgroup form stops here: its time grows with the columns, the
// other's chain of m x m products does not.  Result / gradient of one f32 matrix in us, one workgroup and two passes:
// 8 x 192 17 / 33 and 20 / 37, 8 x 320 25 / 49 and 20 / 38, 24 x 192 29 / 54 and 31 / 66, 24 x 320 43 / 80 and 31 / 67,
// 56 x 192 61 and 81, 56 x 320 80 and 80; 2000 x 8 x 300 101 / 252 and 97 / 200.
constexpr int SMALL_COLS = 240;

// bytes of LDS of the one-workgroup form; 0: it does not fit, or another is quicker
int small_bytes(const Shape& s, bool grad, double growth) {
  if (s.mr > 512 || s.nc > 4096 || (thin_fits(s, grad, growth) && s.nc > SMALL_COLS)) return 0;
  const SmallShape q = small_shape(s.m, s.n, s.cx);
  if ((q.R16 / 16) * (q.C16 / 16) > SMALL_WAVES * SMALL_TILES) return 0;
  const long long b = 4ll * ((grad ? 2 : 1) * q.R16 * q.ldx + (grad ? 4 : 2) * q.R16 * q.lda);
  return b <= SMALL_LDS ? (int)b : 0;
}

// the saved block of the one-workgroup form: norms, then the iterates
struct SmallSaved {
  double* norm;
  float* x;
};

SmallSaved take_small(Arena& w, const Shape& s, int steps) {
  SmallSaved v;
  v.norm = w.take<double>(s.batch);
  v.x = w.take<float>((long long)s.batch * steps * s.m * s.nc);
  return v;
}

template <int SRC, bool GRAD, int SLOTS>
hipError_t small_launch(const SmallArgs& a, int bytes, int batch, hipStream_t st) {
  const void* f = GRAD ? reinterpret_cast<const void*>(small_grad_kernel<SRC, SLOTS>) : reinterpret_cast<const void*>(small_kernel<SRC, SLOTS>);
  static std::atomic<unsigned long long> done{0};
  const hipError_t e = raise_lds(f, SMALL_LDS, done);
  if (e != hipSuccess) return e;
  if (GRAD) hipLaunchKernelGGL((small_grad_kernel<SRC, SLOTS>), dim3(batch), dim3(SMALL_THREADS), bytes, st, a);
  else hipLaunchKernelGGL((small_kernel<SRC, SLOTS>), dim3(batch), dim3(SMALL_THREADS), bytes, st, a);
  return hipGetLastError();
}

// as many tiles a wave as the matrix needs: the branches around those that it lacks are what a step of a small one waits for
template <int SRC, bool GRAD>
hipError_t small_slots(const SmallArgs& a, int bytes, int batch, hipStream_t st) {
  const SmallShape q = small_shape(a.m, a.n, a.cx);
  const int tiles = (q.R16 / 16) * (q.C16 / 16);
  if (tiles <= SMALL_WAVES) return small_launch<SRC, GRAD, 1>(a, bytes, batch, st);
  if (tiles <= 2 * SMALL_WAVES) return small_launch<SRC, GRAD, 2>(a, bytes, batch, st);
  return small_launch<SRC, GRAD, SMALL_TILES>(a, bytes, batch, st);
}

template <bool GRAD>
hipError_t small_by_type(int src, const SmallArgs& a, int bytes, int batch, hipStream_t st) {
  if (src == SRC_F32) return small_slots<SRC_F32, GRAD>(a, bytes, batch, st);
  if (src == SRC_F16) return small_slots<SRC_F16, GRAD>(a, bytes, batch, st);
  if (src == SRC_BF16) return small_slots<SRC_BF16, GRAD>(a, bytes, batch, st);
  return small_slots<SRC_C64, GRAD>(a, bytes, batch, st);
}

#define TRY(x)                                   \
  do {                                           \
    const hipError_t e_ = (x);                   \
    if (e_ != hipSuccess) return e_;             \
  } while (0)

// A, B of one step from the pieces of X.  tri: tiles above the diagonal are copies of those below.  Two-piece products add
// hi lo' before lo hi', so a copy's rounding is that of x y where its neighbours' is that of y x, and rows of G that are equal stop
// being so: 2^-24 in a direction that G does not have, times a in every step after.  Steps that grow it past 600 (six of the
// default) compute every tile: 128 x 200 f32 with rows that occur twice, 10 / 16 steps: 5e-4 / 0.8 of the result -> 4e-6 / 7e-6.
template <int P>
hipError_t ns_factor(const Shape& s, const Pieces& p, const Scales& c, const double* co, bool tri, float* split, hipStream_t st) {
  const long long xs = s.mr * s.np, qs = s.mr * s.mp;
  Args g = base_args(s, split, s.mr, s.mr, s.np, s.np, xs, xs);
  pair(g, p.x, p.x);
  TRY(run<P>(g, tri, EpiSym<P>{p.a, nullptr, s.mp, qs, 1.f / (c.x * c.x), 0.f, c.A}, st));
  g = base_args(s, split, s.mr, s.mr, s.mp, s.mp, qs, qs);
  pair(g, p.a, p.a);
  return run<P>(g, tri, EpiSym<P>{p.b, p.a, s.mp, qs, (float)co[2] / (c.A * c.A), (float)co[1] / c.A, c.B}, st);
}

struct Problem {
  Mat g;                          // caller's matrix with rows = the shorter axis
  void* out;
  long long ors, ocs, obs;
  int src, dtype, steps;
  const double* coef;
  double eps;
  // optimiser step
  float* buf;
  long long brs, bcs, bbs;
  float rest, keep, rate;
  int nesterov;
};

SmallArgs small_args(const Shape& s, const Problem& q) {
  SmallArgs a{};
  a.src = q.g;
  a.m = s.m;
  a.n = s.n;
  a.cx = s.cx;
  a.steps = q.steps;
  a.flat = q.g.cs <= q.g.rs;
  for (int i = 0; i < 3 * q.steps; ++i) a.coef[i] = (float)q.coef[i];
  a.eps = (float)q.eps;
  a.buf = q.buf;
  a.brs = q.brs;
  a.bcs = q.bcs;
  a.bbs = q.bbs;
  a.rest = q.rest;
  a.nesterov = q.nesterov;
  a.out = q.out;
  a.ors = q.ors;
  a.ocs = q.ocs;
  a.obs = q.obs;
  a.dtype = q.dtype;
  a.update = q.buf != nullptr;
  a.keep = q.keep;
  a.rate = q.rate;
  return a;
}

// the doubled matrix of a complex one has padding that no product writes; else products leave the next step's operands
bool padded(const Shape& s) { return s.cx == 2 && (s.mp != s.P * s.mr || s.np != s.P * s.nc); }

template <int P>
hipError_t forward(const Shape& s, const Problem& q, const Scales* sc, Work& w, Saved* sv, hipStream_t st) {
  const int nb = sum_blocks(s);
  const bool fuse = !padded(s), tri = P == 1 || growth_of(q.steps, q.coef) <= GROWTH_F32;
  SumArgs sa{};
  sa.x = q.g;
  sa.outer = s.m;
  sa.inner = s.n;
  sa.part = w.part;
  if (q.buf) {
    sa.buf = q.buf;
    sa.brs = q.brs;
    sa.bcs = q.bcs;
    sa.bbs = q.bbs;
    sa.rest = q.rest;
    sa.nesterov = q.nesterov;
    TRY(launch_sums<2>(q.src, sa, nb, s.batch, st));
  } else {
    TRY(launch_sums<0>(q.src, sa, nb, s.batch, st));
  }
  for (int i = 0; i < q.steps; ++i) {
    Pieces p = sv ? sv->p[i] : w.p;
    if (!sv && fuse && i % 2) p.t = w.t2;
    const bool fused = i > 0 && fuse;                // the step before left this one's operands
    if (padded(s) && (sv || i == 0)) {               // the doubled matrix's padding
      TRY(clear(p.x, s.mr * s.np * s.batch * 2, st));
      TRY(clear(p.t, s.nc * s.mp * s.batch * 2, st));
    }
    PackArgs a{};
    a.scale = sc[i].x;
    a.x = p.x;
    a.t = p.t;
    if (i == 0) {
      a.src = q.g;
      a.part = w.part;
      a.npart = nb;
      a.eps = (float)q.eps;
      a.norm_out = sv ? sv->norm : w.norm;
      a.carry = w.carry;
      a.buf = q.buf;
      a.brs = q.brs;
      a.bcs = q.bcs;
      a.bbs = q.bbs;
      a.rest = q.rest;
      a.nesterov = q.nesterov;
      TRY(launch_pack<P>(q.src, a, s, st));
    } else if (!fused) {
      a.src = Mat{w.carry, s.ldc, 1, s.m * s.ldc};
      TRY(launch_pack<P>(SRC_PLANAR, a, s, st));
    }
    TRY(ns_factor<P>(s, p, sc[i], q.coef + 3 * i, tri, w.split, st));
    const float alpha = 1.f / (sc[i].B * sc[i].x), beta = (float)q.coef[3 * i];
    const long long ts = s.nc * s.mp, qs = s.mr * s.mp, cs = s.m * s.ldc;
    if (i + 1 < q.steps) {
      Args g = base_args(s, w.split, s.m, s.nc, s.mp, s.mp, qs, ts);
      pair(g, p.b, p.t);
      if (fuse) {
        const Pieces& n = sv ? sv->p[i + 1] : w.p;
        f16* t = !sv && i % 2 == 0 ? w.t2 : n.t;
        TRY(run<P>(g, false, EpiNext<P>{w.carry, s.ldc, cs, alpha, beta, sc[i + 1].x, n.x, t, s.np, s.mr * s.np, s.mp, ts,
                                               s.cx == 2 ? s.n : 0}, st));
      } else {
        TRY(run<P>(g, false, EpiCarry{w.carry, s.ldc, cs, alpha, beta, nullptr}, st));
      }
      continue;
    }
    const int size = q.dtype == TCMI_F32 ? 4 : 2, up = q.buf != nullptr;
    hipError_t e = hipSuccess;
#define LAST(DT)                                                                                                              \
  if (q.dtype == DT) {                                                                                                        \
    if (s.flip && DT != TCMI_C64) {                                                                                           \
      Args g = base_args(s, w.split, s.nc, s.m, s.mp, s.mp, ts, qs);                                                          \
      pair(g, p.t, p.b);                                                                                                      \
      e = run<P>(g, false, EpiOut<P, DT>{p.t, s.mp, ts, alpha, beta / sc[i].x, q.out, q.ocs, q.ors, q.obs, s.n, up, q.keep, q.rate, \
                                         aligned4(q.out, q.ocs, q.ors, q.obs, size)}, st);                                    \
    } else {                                                                                                                  \
      Args g = base_args(s, w.split, s.m, s.nc, s.mp, s.mp, qs, ts);                                                          \
      pair(g, p.b, p.t);                                                                                                      \
      e = run<P>(g, false, EpiOut<0, DT>{w.carry, s.ldc, cs, alpha, beta, q.out, q.ors, q.ocs, q.obs, s.n, up, q.keep, q.rate, \
                                         aligned4(q.out, q.ors, q.ocs, q.obs, size)}, st);                                    \
    }                                                                                                                         \
  }
    LAST(TCMI_BF16)
    if constexpr (P == 2) {                          // one piece serves bf16 results only
      LAST(TCMI_F32)
      LAST(TCMI_F16)
      LAST(TCMI_C64)
    }
#undef LAST
    TRY(e);
  }
  return hipSuccess;
}

// ---- few rows, long columns
int thin_r16(const Shape& s) { return (s.mr + 15) & ~15; }

int thin_chunks(const Shape& s) { return (s.n + THIN_COLS - 1) / THIN_COLS; }

// workgroups of a pass over the columns: enough for the card, few enough that one workgroup adds their sums quickly
int thin_parts(const Shape& s) {
  const int r = thin_r16(s);
  int most = r <= 16 ? THIN_MAX_PART : r <= 32 ? 64 : 32;
  const int room = (512 + s.batch - 1) / s.batch, c = thin_chunks(s);
  if (most > room) most = room < 4 ? 4 : room;
  return c < most ? c : most;
}

struct ThinWork {
  double *part, *norm, *steps, *m1, *m2;
};

ThinWork take_thin(Arena& w, const Shape& s, bool grad, int steps) {
  ThinWork k{};
  const long long q = (long long)thin_r16(s) * thin_r16(s) * s.batch;
  k.part = w.take<double>(q * thin_parts(s));
  k.norm = w.take<double>(s.batch);
  k.m1 = w.take<double>(q);
  if (grad) {
    k.m2 = w.take<double>(q);
    k.steps = w.take<double>(3 * q * steps);
  }
  return k;
}

struct ThinSaved {
  double *norm, *a0;
};

ThinSaved take_thin_saved(Arena& w, const Shape& s) {
  ThinSaved v;
  v.norm = w.take<double>(s.batch);
  v.a0 = w.take<double>((long long)thin_r16(s) * thin_r16(s) * s.batch);
  return v;
}

ThinArgs thin_args(const Shape& s, const Problem& q, const ThinWork& w) {
  ThinArgs a{};
  a.g = q.g;
  a.m = s.m;
  a.n = s.n;
  a.cx = s.cx;
  a.steps = q.steps;
  a.flat = q.g.cs <= q.g.rs;
  a.oflat = q.ocs <= q.ors;
  a.chunks = thin_chunks(s);
  a.parts = thin_parts(s);
  for (int i = 0; i < 3 * q.steps; ++i) a.coef[i] = q.coef[i];
  a.eps = q.eps;
  a.buf = q.buf;
  a.brs = q.brs;
  a.bcs = q.bcs;
  a.bbs = q.bbs;
  a.rest = q.rest;
  a.nesterov = q.nesterov;
  a.out = q.out;
  a.ors = q.ors;
  a.ocs = q.ocs;
  a.obs = q.obs;
  a.dtype = q.dtype;
  a.update = q.buf != nullptr;
  a.keep = q.keep;
  a.rate = q.rate;
  a.part = w.part;
  a.norm = w.norm;
  a.m1 = w.m1;
  a.m2 = w.m2;
  a.steps_mem = w.steps;
  return a;
}

template <int SRC, bool GRAD, class S>
hipError_t thin_apply(const Shape& s, const ThinArgs& a, hipStream_t st) {
  constexpr int pad = 16 / sizeof(S), size = sizeof(S);
  const int r = thin_r16(s), ld = s.cx * THIN_COLS + 4, bytes = (GRAD ? 2 : 1) * r * (4 * ld + size * (r + pad));
  static std::atomic<unsigned long long> done{0};
  const hipError_t e = raise_lds(reinterpret_cast<const void*>(thin_apply_kernel<SRC, GRAD, S>),
                                 THIN_R * (4 * (2 * THIN_COLS + 4) + size * (THIN_R + pad)), done);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((thin_apply_kernel<SRC, GRAD, S>), dim3(a.chunks, s.batch), dim3(256), bytes, st, a);
  return hipGetLastError();
}

template <int SRC, bool GRAD>
hipError_t thin_launch(const Shape& s, const ThinArgs& a, double growth, hipStream_t st) {
  const int r = thin_r16(s), gram = (GRAD ? 2 : 1) * r * (s.cx * THIN_COLS + 4) * 4, poly = (GRAD ? 11 : 4) * r * (r + 2) * 8;
  static std::atomic<unsigned long long> done[2] = {};
  hipError_t e = raise_lds(reinterpret_cast<const void*>(thin_gram_kernel<SRC, GRAD>), THIN_R * (2 * THIN_COLS + 4) * 4, done[0]);
  if (e == hipSuccess)
    e = raise_lds(GRAD ? reinterpret_cast<const void*>(thin_grad_poly_kernel) : reinterpret_cast<const void*>(thin_poly_kernel), SMALL_LDS, done[1]);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((thin_gram_kernel<SRC, GRAD>), dim3(a.parts, s.batch), dim3(256), gram, st, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (GRAD) hipLaunchKernelGGL(thin_grad_poly_kernel, dim3(s.batch), dim3(THIN_THREADS), poly, st, a);
  else hipLaunchKernelGGL(thin_poly_kernel, dim3(s.batch), dim3(THIN_THREADS), poly, st, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  return growth <= GROWTH_F32 ? thin_apply<SRC, GRAD, float>(s, a, st) : thin_apply<SRC, GRAD, double>(s, a, st);
}

template <bool GRAD>
hipError_t thin(const Shape& s, int src, const ThinArgs& a, double growth, hipStream_t st) {
  if (src == SRC_F32) return thin_launch<SRC_F32, GRAD>(s, a, growth, st);
  if (src == SRC_F16) return thin_launch<SRC_F16, GRAD>(s, a, growth, st);
  if (src == SRC_BF16) return thin_launch<SRC_BF16, GRAD>(s, a, growth, st);
  return thin_launch<SRC_C64, GRAD>(s, a, growth, st);
}

hipError_t forward(const Shape& s, const Problem& q, const Scales* sc, Work& w, Saved* sv, hipStream_t st) {
  return s.P == 2 ? forward<2>(s, q, sc, w, sv, st) : forward<1>(s, q, sc, w, sv, st);
}

hipError_t backward(const Shape& s, const Problem& q, const Mat& dy, const Scales* sc, GradWork& w, const Saved& sv, hipStream_t st) {
  const long long xs = s.mr * s.np, ts = s.nc * s.mp, qs = s.mr * s.mp;
  const int nb = sum_blocks(s);
  if (padded(s)) {
    TRY(clear(w.d, xs * s.batch * 2, st));
    TRY(clear(w.t, ts * s.batch * 2, st));
  }
  // The pieces of D are taken under a bound.  Where the steps can lengthen D by 2^10 at most (the default coefficients: 566),
  // that is |dY| times what the steps allow, and a step leaves the next one's pieces.  Of the 39 binades between f16's largest
  // value and its smallest step 22 are the pieces' own, so D may stay 2^7 below the bound before an entry of D's mean size
  // in a 1000 x 1000 matrix loses bits; in fact its part outside G's symmetric directions grows as X does, 2 to 9 times.  A
  // larger bound would leave too few bits: there D is measured and divided by its norm at every step.
  double bound[TCMI_NS_MAX_STEPS], dn[TCMI_NS_MAX_STEPS];
  double sig = 1.0, grown = 1.0;
  for (int i = 0; i < q.steps; ++i) {
    bound[i] = sig * SLACK;
    sig = bound_of(bound[i], q.coef + 3 * i).next;
  }
  for (int i = q.steps - 1; i >= 0; --i) {
    dn[i] = grown;
    grown *= fmax(1.0, bound_of(bound[i], q.coef + 3 * i).slope);
  }
  const bool fuse = !padded(s) && dn[0] <= 1024.0;
  float sD[TCMI_NS_MAX_STEPS], sQ[TCMI_NS_MAX_STEPS], sS[TCMI_NS_MAX_STEPS];
  for (int i = 0; i < q.steps; ++i) {
    // |S|_F <= 2 x |D|, |Q|_F <= (2 x b + 4 x^3 c) |D|.  B D and Q X share an accumulator, so their scales have to agree:
    // sB sD = sQ sX.
    const double x = bound[i], b = fabs(q.coef[3 * i + 1]), c = fabs(q.coef[3 * i + 2]), d = (fuse ? dn[i] : 1.0) * SLACK;
    const float qmax = scale_for((2 * x * b + 4 * x * x * x * c) * d);
    sS[i] = scale_for(2 * x * d);
    sD[i] = scale_for(d);
    sQ[i] = sc[i].B * sD[i] / sc[i].x;
    if (sQ[i] > qmax) {
      sD[i] *= qmax / sQ[i];
      sQ[i] = qmax;
    }
  }
  for (int i = q.steps - 1; i >= 0; --i) {
    const Pieces& p = sv.p[i];
    const bool first = i == q.steps - 1;
    if (first || !fuse) {                            // |D| and D's pieces
      SumArgs sa{};
      sa.outer = s.m;
      sa.part = w.part;
      PackArgs a{};
      a.part = w.part;
      a.npart = nb;
      a.norm_out = w.norm;
      a.scale = sD[i];
      a.x = w.d;
      a.t = w.t;
      if (first) {
        sa.x = a.src = dy;
        sa.inner = s.n;
        a.carry = w.carry;
        a.carry_raw = !fuse;                         // else only its pieces are divided, the epilogue multiplies
        TRY(launch_sums<0>(q.src, sa, nb, s.batch, st));
        TRY(launch_pack<2>(q.src, a, s, st));
      } else {
        sa.x = a.src = Mat{w.carry, s.ldc, 1, s.m * s.ldc};
        sa.inner = s.nc;
        TRY(launch_sums<0>(SRC_F32, sa, nb, s.batch, st));
        TRY(launch_pack<2>(SRC_PLANAR, a, s, st));
      }
    }
    // S = D X^T + X D^T
    Args g = base_args(s, w.split, s.mr, s.mr, s.np, s.np, xs, xs);
    pair(g, w.d, p.x);
    pair(g, p.x, w.d);
    TRY(run<2>(g, true, EpiSym<2>{w.s, nullptr, s.mp, qs, 1.f / (sD[i] * sc[i].x), 0.f, sS[i]}, st));
    // Q = b S + c (A S + S A)
    g = base_args(s, w.split, s.mr, s.mr, s.mp, s.mp, qs, qs);
    pair(g, p.a, w.s);
    pair(g, w.s, p.a);
    TRY(run<2>(g, true, EpiSym<2>{w.q, w.s, s.mp, qs, (float)q.coef[3 * i + 2] / (sc[i].A * sS[i]), (float)q.coef[3 * i + 1] / sS[i], sQ[i]}, st));
    // D <- a D + B D + Q X (not fused: the products hold D / |D|)
    g = base_args(s, w.split, s.m, s.nc, s.mp, s.mp, qs, ts);
    pair(g, p.b, w.t);
    pair(g, w.q, p.t);
    const float alpha = 1.f / (sc[i].B * sD[i]), beta = (float)q.coef[3 * i];
    if (fuse && i > 0) {
      TRY(run<2>(g, false, EpiNext<2>{w.carry, s.ldc, s.m * s.ldc, alpha, beta, sD[i - 1], w.d, w.t2, s.np, xs, s.mp, ts,
                                      s.cx == 2 ? s.n : 0}, st));
      f16* t = w.t;
      w.t = w.t2;
      w.t2 = t;
    } else {
      TRY(run<2>(g, false, EpiCarry{w.carry, s.ldc, s.m * s.ldc, alpha, beta, fuse ? nullptr : w.norm}, st));
    }
  }
  // dG
  if (q.g.rs < q.g.cs) {
    TurnedArgs a{};
    a.g = q.g;
    a.d = w.carry;
    a.ldd = s.ldc;
    a.dbs = s.m * s.ldc;
    a.m = s.m;
    a.n = s.n;
    a.tx = (s.n + 63) / 64;
    a.tiles = a.tx * ((s.m + 63) / 64);
    a.npart = a.tiles < nb ? a.tiles : nb;
    a.part = w.part;
    a.norm = sv.norm;
    a.dnorm = fuse ? w.norm : nullptr;
    a.eps = (float)q.eps;
    a.out = q.out;
    a.rs = q.ors;
    a.cs = q.ocs;
    a.os = q.obs;
    a.dtype = q.dtype;
    const dim3 sums(a.npart, s.batch), outs(a.tiles < 4096 ? a.tiles : 4096, s.batch);
#define GO(SRC)                                                                          \
  {                                                                                      \
    hipLaunchKernelGGL((turned_kernel<SRC, false>), sums, dim3(256), 0, st, a);          \
    TRY(hipGetLastError());                                                              \
    hipLaunchKernelGGL((turned_kernel<SRC, true>), outs, dim3(256), 0, st, a);           \
  }
    if (q.src == SRC_F32) GO(SRC_F32)
    else if (q.src == SRC_F16) GO(SRC_F16)
    else if (q.src == SRC_BF16) GO(SRC_BF16)
    else GO(SRC_C64)
#undef GO
    return hipGetLastError();
  }
  SumArgs sa{};
  sa.x = q.g;
  sa.y = Mat{w.carry, s.ldc, 1, s.m * s.ldc};
  sa.brs = s.n;
  sa.outer = s.m;
  sa.inner = s.n;
  sa.part = w.part;
  TRY(launch_sums<1>(q.src, sa, nb, s.batch, st));
  const long long total = (long long)s.m * s.n;
  const unsigned gx = (unsigned)((total + 1023) / 1024 > 4096 ? 4096 : (total + 1023) / 1024);
  const dim3 grid(gx, s.batch);
#define GO(SRC)                                                                                                            \
  hipLaunchKernelGGL(grad_out_kernel<SRC>, grid, dim3(256), 0, st, q.g, w.carry, s.ldc, s.m * s.ldc, s.m, s.n, w.part, nb, \
                     sv.norm, fuse ? w.norm : nullptr, (float)q.eps, q.out, q.ors, q.ocs, q.obs, q.dtype)
  if (q.src == SRC_F32) GO(SRC_F32);
  else if (q.src == SRC_F16) GO(SRC_F16);
  else if (q.src == SRC_BF16) GO(SRC_BF16);
  else GO(SRC_C64);
#undef GO
  return hipGetLastError();
}

int src_of(int dtype) {
  return dtype == TCMI_F32 ? SRC_F32 : dtype == TCMI_F16 ? SRC_F16 : dtype == TCMI_BF16 ? SRC_BF16 : dtype == TCMI_C64 ? SRC_C64 : -1;
}

bool sizes_ok(int rows, int cols, int batch, int steps, int dtype) {
  return rows >= 1 && cols >= 1 && batch >= 1 && batch <= 65535 && rows <= (1 << 24) && cols <= (1 << 24) && steps >= 1 &&
         steps <= TCMI_NS_MAX_STEPS && src_of(dtype) >= 0;
}

// the large form's rows have to stay within a product's offsets
bool rows_ok(const Shape& s) { return s.np <= MAX_ROW && s.mp <= MAX_ROW; }

// a matrix with its shorter axis as rows
Mat oriented(const void* p, long long rs, long long cs, long long bs, bool flip) { return flip ? Mat{p, cs, rs, bs} : Mat{p, rs, cs, bs}; }

}  // namespace orth
}  // namespace tcmi

using namespace tcmi::orth;

extern "C" {

long long tcmi_ns_work_bytes_coef(int rows, int cols, int batch, int steps, const double* coef_host, int full, int dtype, int what) {
  if (!sizes_ok(rows, cols, batch, steps, dtype) || what < 0 || what > 3) return -1;
  const Shape s = shape_of(rows, cols, batch, dtype, full != 0 || what != TCMI_NS_WORK);
  const bool grad = what != TCMI_NS_WORK;
  auto bytes = [&](double growth) -> long long {
    Arena a{nullptr};
    if (small_bytes(s, grad, growth)) {
      if (what == TCMI_NS_SAVED) take_small(a, s, steps);
      else a.take<char>(1);
    } else if (thin_fits(s, grad, growth)) {
      if (what == TCMI_NS_SAVED) take_thin_saved(a, s);
      else take_thin(a, s, what == TCMI_NS_WORK_GRAD, steps);
    } else {
      if (!rows_ok(s)) return -1;
      if (what == TCMI_NS_WORK) take_work(a, s, false);
      else if (what == TCMI_NS_WORK_SAVING) take_work(a, s, true);
      else if (what == TCMI_NS_SAVED) take_saved(a, s, steps);
      else take_grad(a, s);
    }
    return a.used;
  };
  const long long most = bytes(growth_of(steps, coef_host));
  if (coef_host) return most;
  const long long least = bytes(1.0);              // any coefficients: whichever form they lead to
  return most > least ? most : least;
}

long long tcmi_ns_work_bytes(int rows, int cols, int batch, int steps, int full, int dtype, int what) {
  return tcmi_ns_work_bytes_coef(rows, cols, batch, steps, nullptr, full, dtype, what);
}

int tcmi_newton_schulz(const void* g, long long g_rs, long long g_cs, long long g_bs, void* out, int rows, int cols, int batch,
                       int steps, const double* coef_host, double eps, int full, void* saved, long long saved_bytes, void* work,
                       long long work_bytes, int dtype, void* stream) {
  if (!sizes_ok(rows, cols, batch, steps, dtype) || !g || !out || !coef_host || !work || !(eps >= 0) || (saved && !full) ||
      (!full && dtype != TCMI_BF16))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_newton_schulz: bad argument");
  const Shape s = shape_of(rows, cols, batch, dtype, full != 0);
  // three forms: one workgroup per matrix; two passes around m x m matrices; a sequence of large products
  const double growth = growth_of(steps, coef_host);
  const int small = small_bytes(s, saved != nullptr, growth);
  const bool narrow = !small && thin_fits(s, saved != nullptr, growth);
  Arena aw{(char*)work}, av{(char*)saved};
  Work w{};
  Saved sv{};
  SmallSaved ss{};
  ThinWork tw{};
  ThinSaved ts{};
  if (small) {
    if (saved) ss = take_small(av, s, steps);
  } else if (narrow) {
    tw = take_thin(aw, s, false, steps);
    if (saved) ts = take_thin_saved(av, s);
  } else {
    if (!rows_ok(s)) return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_newton_schulz: a side is too long");
    w = take_work(aw, s, saved != nullptr);
    if (saved) sv = take_saved(av, s, steps);
  }
  if (aw.used > work_bytes || (saved && av.used > saved_bytes) || ((uintptr_t)work & 255) || ((uintptr_t)saved & 255))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_newton_schulz: workspace too small or not 256-byte aligned");
  Scales sc[TCMI_NS_MAX_STEPS];
  if (!scales_of(steps, coef_host, sc))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_newton_schulz: these coefficients let a singular value grow past 64");
  Problem q{};
  q.g = oriented(g, g_rs, g_cs, g_bs, s.flip);
  q.out = out;
  q.ors = s.flip ? 1 : cols;
  q.ocs = s.flip ? cols : 1;
  q.obs = (long long)rows * cols;
  q.src = src_of(dtype);
  q.dtype = dtype;
  q.steps = steps;
  q.coef = coef_host;
  q.eps = eps;
  hipError_t e;
  if (small) {
    SmallArgs a = small_args(s, q);
    a.saved = ss.x;
    a.norm = ss.norm;
    e = small_by_type<false>(q.src, a, small, batch, reinterpret_cast<hipStream_t>(stream));
  } else if (narrow) {
    ThinArgs a = thin_args(s, q, tw);
    a.a0 = ts.a0;
    if (saved) a.norm = ts.norm;
    e = thin<false>(s, q.src, a, growth, reinterpret_cast<hipStream_t>(stream));
  } else {
    e = forward(s, q, sc, w, saved ? &sv : nullptr, reinterpret_cast<hipStream_t>(stream));
  }
  return e == hipSuccess ? TCMI_OK : tcmi_set_error_(TCMI_ERR_HIP, hipGetErrorString(e));
}

int tcmi_newton_schulz_grad(const void* g, long long g_rs, long long g_cs, long long g_bs, const void* dout, long long d_rs,
                            long long d_cs, long long d_bs, void* dg, int rows, int cols, int batch, int steps,
                            const double* coef_host, double eps, const void* saved, long long saved_bytes, void* work,
                            long long work_bytes, int dtype, void* stream) {
  if (!sizes_ok(rows, cols, batch, steps, dtype) || !g || !dout || !dg || !coef_host || !saved || !work || !(eps >= 0))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_newton_schulz_grad: bad argument");
  const Shape s = shape_of(rows, cols, batch, dtype, true);
  Arena aw{(char*)work}, av{(char*)const_cast<void*>(saved)};
  const double growth = growth_of(steps, coef_host);
  const int small = small_bytes(s, true, growth);
  const bool narrow = !small && thin_fits(s, true, growth);
  GradWork w{};
  Saved sv{};
  SmallSaved ss{};
  ThinWork tw{};
  ThinSaved ts{};
  if (small) {
    ss = take_small(av, s, steps);
  } else if (narrow) {
    tw = take_thin(aw, s, true, steps);
    ts = take_thin_saved(av, s);
  } else {
    if (!rows_ok(s)) return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_newton_schulz_grad: a side is too long");
    w = take_grad(aw, s);
    sv = take_saved(av, s, steps);
  }
  if (aw.used > work_bytes || av.used > saved_bytes || ((uintptr_t)work & 255) || ((uintptr_t)saved & 255))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_newton_schulz_grad: workspace too small or not 256-byte aligned");
  Scales sc[TCMI_NS_MAX_STEPS];
  if (!scales_of(steps, coef_host, sc))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_newton_schulz_grad: these coefficients let a singular value grow past 64");
  Problem q{};
  q.g = oriented(g, g_rs, g_cs, g_bs, s.flip);
  q.out = dg;
  q.ors = s.flip ? 1 : cols;
  q.ocs = s.flip ? cols : 1;
  q.obs = (long long)rows * cols;
  q.src = src_of(dtype);
  q.dtype = dtype;
  q.steps = steps;
  q.coef = coef_host;
  q.eps = eps;
  hipError_t e;
  if (small) {
    SmallArgs a = small_args(s, q);
    a.dy = oriented(dout, d_rs, d_cs, d_bs, s.flip);
    a.saved = ss.x;
    a.norm = ss.norm;
    e = small_by_type<true>(q.src, a, small, batch, reinterpret_cast<hipStream_t>(stream));
  } else if (narrow) {
    ThinArgs a = thin_args(s, q, tw);
    a.dy = oriented(dout, d_rs, d_cs, d_bs, s.flip);
    a.dflat = a.dy.cs <= a.dy.rs;
    a.a0 = ts.a0;
    a.norm = ts.norm;
    e = thin<true>(s, q.src, a, growth, reinterpret_cast<hipStream_t>(stream));
  } else {
    e = backward(s, q, oriented(dout, d_rs, d_cs, d_bs, s.flip), sc, w, sv, reinterpret_cast<hipStream_t>(stream));
  }
  return e == hipSuccess ? TCMI_OK : tcmi_set_error_(TCMI_ERR_HIP, hipGetErrorString(e));
}

int tcmi_muon_step(void* param, long long p_rs, long long p_cs, long long p_bs, const void* grad, long long g_rs, long long g_cs,
                   long long g_bs, float* buf, long long b_rs, long long b_cs, long long b_bs, int rows, int cols, int batch,
                   double momentum, int nesterov, double keep, double rate, int steps, const double* coef_host, double eps,
                   int full, void* work, long long work_bytes, int dtype, void* stream) {
  if (!sizes_ok(rows, cols, batch, steps, dtype) || dtype == TCMI_C64 || !param || !grad || !buf || !coef_host || !work || !(eps >= 0) ||
      !(momentum >= 0) || !(momentum < 1) || (!full && dtype != TCMI_BF16))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_muon_step: bad argument");
  const Shape s = shape_of(rows, cols, batch, dtype, full != 0);
  const double growth = growth_of(steps, coef_host);
  const int small = small_bytes(s, false, growth);
  const bool narrow = !small && thin_fits(s, false, growth);
  Arena aw{(char*)work};
  Work w{};
  ThinWork tw{};
  if (!small && !narrow && !rows_ok(s)) return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_muon_step: a side is too long");
  if (narrow) tw = take_thin(aw, s, false, steps);
  else if (!small) w = take_work(aw, s, false);
  if (aw.used > work_bytes || ((uintptr_t)work & 255))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_muon_step: workspace too small or not 256-byte aligned");
  Scales sc[TCMI_NS_MAX_STEPS];
  if (!scales_of(steps, coef_host, sc))
    return tcmi_set_error_(TCMI_ERR_ARG, "tcmi_muon_step: these coefficients let a singular value grow past 64");
  Problem q{};
  q.g = oriented(grad, g_rs, g_cs, g_bs, s.flip);
  q.out = param;
  q.ors = s.flip ? p_cs : p_rs;
  q.ocs = s.flip ? p_rs : p_cs;
  q.obs = p_bs;
  q.src = src_of(dtype);
  q.dtype = dtype;
  q.steps = steps;
  q.coef = coef_host;
  q.eps = eps;
  q.buf = buf;
  q.brs = s.flip ? b_cs : b_rs;
  q.bcs = s.flip ? b_rs : b_cs;
  q.bbs = b_bs;
  q.rest = (float)(1.0 - momentum);
  q.nesterov = nesterov;
  q.keep = (float)keep;
  q.rate = (float)rate;
  const hipError_t e = small    ? small_by_type<false>(q.src, small_args(s, q), small, batch, reinterpret_cast<hipStream_t>(stream))
                       : narrow ? thin<false>(s, q.src, thin_args(s, q, tw), growth, reinterpret_cast<hipStream_t>(stream))
                                : forward(s, q, sc, w, nullptr, reinterpret_cast<hipStream_t>(stream));
  return e == hipSuccess ? TCMI_OK : tcmi_set_error_(TCMI_ERR_HIP, hipGetErrorString(e));
}

}  // extern "C"
