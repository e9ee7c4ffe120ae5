// Matrix core of the training operators: C[m][n] = sum_s sum_k A_s[m][k] B_s[n][k] on the f16 / bf16 matrix pipe with f32
// accumulators, up to six pairs ("segments") of k-contiguous operands per product, and an epilogue functor per use.
//
// Segments carry the precision: an f32 operand x is held as two f16 pieces x = hi + lo (11 + 11 significand bits), and
// x y ~= hi hi' + hi lo' + lo hi' is three segments of one accumulation; what is dropped is below 2^-22 |x y|, the size of
// an f32 rounding.  Sums of several products (P D + Q X) are segments too.
//
// Operand contract (checked by the callers on the host): rows are k-contiguous and 16-byte aligned, K is a multiple of
// 64 with everything beyond the true length zero, row indices past the end are clamped (never read outside), and the
// epilogue masks what the clamped rows produce.
#ifndef TCMI_MM16_H
#define TCMI_MM16_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tcmi {
namespace mm16 {

using f16 = _Float16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int MAX_SEG = 6;

struct Args {
  const void* a[MAX_SEG];
  const void* b[MAX_SEG];
  int nseg;
  int M, N, K;                 // K a multiple of 64
  long long lda, ldb;          // elements between rows
  long long sa, sb;            // elements between batch members
  int tm, tn;                  // tiles per matrix
  int tri;                     // 1: C is symmetric, only tiles with row tile >= column tile are computed
  int tiles;                   // tiles per batch member (tm * tn, or the triangle)
};

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Which tile a workgroup computes.  Workgroups go to the eight XCDs in turn; renumbered so that each XCD (its own L2) gets
// one contiguous range, in bands of 8 row tiles, whose operand rows it then reads from its L2.
__device__ __forceinline__ void tile_of(const Args& g, int& ti, int& tj, int& bz) {
  const unsigned total = gridDim.x, id = blockIdx.x;
  const unsigned q = total >> 3, r = total & 7, x = id & 7;
  const unsigned w = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
  bz = (int)(w / (unsigned)g.tiles);
  const unsigned t = w % (unsigned)g.tiles;
  if (g.tri) {
    unsigned i = (unsigned)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while (i * (i + 1) / 2 > t) --i;
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    ti = (int)i;
    tj = (int)(t - i * (i + 1) / 2);
  } else {
    const unsigned band = t / (8u * g.tn), in = t % (8u * g.tn);
    const unsigned rows = min(8u, (unsigned)g.tm - band * 8u);
    ti = (int)(band * 8u + in % rows);
    tj = (int)(in / rows);
  }
}

template <int BM_, int BN_, int WM_, int WN_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  static constexpr int STAGE = (BM + BN) * 128;            // bytes of one 64-deep k step of both operands
};

using LdsPtr = __attribute__((address_space(3))) void*;

// One product tile.  `acc[mi][ni]` holds C[row][col .. col + 3] with row = m0 + wm * BM / WM + 16 mi + (lane & 15) and
// col = n0 + wn * BN / WN + 16 ni + 4 (lane >> 4): the B fragment is the first MFMA operand, so a lane ends with four
// neighbouring columns of one row.
// LDS: a row's 64 k values are eight 16-byte chunks; chunk c of row r lies at position c ^ (r & 7), which spreads the 16
// rows a fragment read touches over all banks.  Global -> LDS goes without registers (buffer_load ... lds), two stages.
#ifdef __HIP_DEVICE_COMPILE__          // the host pass does not know the buffer resource type
template <class V, class T>
__device__ __forceinline__ void product(const Args& g, int m0, int n0, int bz, char* lds, f32x4 (&acc)[T::MI][T::NI]) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / T::WN, wn = wave % T::WN;
  constexpr int LA = T::BM / 8 / T::WAVES, LB = T::BN / 8 / T::WAVES;      // loads per wave: 8 rows of 128 bytes each
  static_assert(LA >= 1 && LB >= 1, "tile too small for its waves");
  unsigned va[LA], vb[LB];
  const unsigned chunk = (unsigned)((lane & 7) ^ (lane >> 3)) * 16u;
#pragma unroll
  for (int j = 0; j < LA; ++j) {
    const int r = min((j * T::WAVES + wave) * 8 + (lane >> 3), g.M - 1 - m0);
    va[j] = (unsigned)r * (unsigned)g.lda * 2u + chunk;
  }
#pragma unroll
  for (int j = 0; j < LB; ++j) {
    const int r = min((j * T::WAVES + wave) * 8 + (lane >> 3), g.N - 1 - n0);
    vb[j] = (unsigned)r * (unsigned)g.ldb * 2u + chunk;
  }
  const long long offa = ((long long)bz * g.sa + (long long)m0 * g.lda) * 2;
  const long long offb = ((long long)bz * g.sb + (long long)n0 * g.ldb) * 2;
  const int ksteps = g.K >> 6, steps = ksteps * g.nseg;
  int ls = 0, lk = 0;                                                   // segment and k step of the next load

  auto load = [&](int stage) {
    char* base = lds + stage * T::STAGE;
    auto ra = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)g.a[ls] + offa), 0, 0xffffffffu, 0x00027000);
    auto rb = __builtin_amdgcn_make_buffer_rsrc((void*)((const char*)g.b[ls] + offb), 0, 0xffffffffu, 0x00027000);
    const unsigned so = (unsigned)lk * 128u;
#pragma unroll
    for (int j = 0; j < LA; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (LdsPtr)(base + (j * T::WAVES + wave) * 1024), 16, va[j], so, 0, 0);
#pragma unroll
    for (int j = 0; j < LB; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (LdsPtr)(base + T::BM * 128 + (j * T::WAVES + wave) * 1024), 16, vb[j], so, 0, 0);
    if (++lk == ksteps) {
      lk = 0;
      ++ls;
    }
  };

  load(0);
  for (int s = 0; s < steps; ++s) {
    __builtin_amdgcn_s_waitcnt(0);                 // this wave's loads of step s are in LDS, its reads of step s - 1 done
    __syncthreads();
    if (s + 1 < steps) load((s + 1) & 1);
    const char* pa = lds + (s & 1) * T::STAGE + (wm * T::MI * 16) * 128;
    const char* pb = lds + (s & 1) * T::STAGE + (T::BM + wn * T::NI * 16) * 128;
    const int r = lane & 15;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int c = ((k * 4 + (lane >> 4)) ^ (r & 7)) * 16 + r * 128;
      V fa[T::MI], fb[T::NI];
#pragma unroll
      for (int i = 0; i < T::MI; ++i) fa[i] = *reinterpret_cast<const V*>(pa + i * 2048 + c);
#pragma unroll
      for (int i = 0; i < T::NI; ++i) fb[i] = *reinterpret_cast<const V*>(pb + i * 2048 + c);
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int j = 0; j < T::NI; ++j) acc[i][j] = mfma(fb[j], fa[i], acc[i][j]);
    }
  }
}

#endif

// Epi: __device__ void tile(const Args&, int m0, int n0, int bz, bool mirror, char* lds, f32x4 (&acc)[MI][NI])
template <class V, class T, class Epi>
__global__ __launch_bounds__(T::THREADS) void product_kernel(Args g, Epi e) {
#ifdef __HIP_DEVICE_COMPILE__
  __shared__ __attribute__((aligned(128))) char lds[2 * T::STAGE];
  int ti, tj, bz;
  tile_of(g, ti, tj, bz);
  f32x4 acc[T::MI][T::NI];
#pragma unroll
  for (int i = 0; i < T::MI; ++i)
#pragma unroll
    for (int j = 0; j < T::NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  product<V, T>(g, ti * T::BM, tj * T::BN, bz, lds, acc);
  e.template tile<T>(g, ti * T::BM, tj * T::BN, bz, g.tri && ti != tj, lds, acc);
#endif
}

// calls f(row, col, value) for the lane's accumulators, four neighbouring columns a call
template <class T, class F>
__device__ __forceinline__ void each(int m0, int n0, const f32x4 (&acc)[T::MI][T::NI], F f) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / T::WN, wn = wave % T::WN;
#pragma unroll
  for (int i = 0; i < T::MI; ++i)
#pragma unroll
    for (int j = 0; j < T::NI; ++j)
      f(m0 + wm * T::MI * 16 + i * 16 + (lane & 15), n0 + wn * T::NI * 16 + j * 16 + 4 * (lane >> 4), acc[i][j]);
}

__device__ __forceinline__ void two_pieces(float x, f16& hi, f16& lo) {
  hi = (f16)x;
  lo = (f16)(x - (float)hi);
}

// host side: tile counts and launch
template <class T>
inline bool plan(Args& g, int batch, bool tri, unsigned* blocks) {
  g.tm = (g.M + T::BM - 1) / T::BM;
  g.tn = (g.N + T::BN - 1) / T::BN;
  g.tri = tri ? 1 : 0;
  const long long tiles = tri ? (long long)g.tm * (g.tm + 1) / 2 : (long long)g.tm * g.tn;
  if (tiles * batch >= (1ll << 31) || tiles < 1) return false;
  g.tiles = (int)tiles;
  *blocks = (unsigned)(tiles * batch);
  return true;
}

}  // namespace mm16
}  // namespace tcmi

#endif
