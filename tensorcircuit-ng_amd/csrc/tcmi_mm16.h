// Matrix core of the training operators: C[m][n] = sum_s sum_k A_s[m][k] B_s[n][k] on the f16 / bf16 matrix pipe with f32
// accumulators, up to two pairs ("segments") of k-contiguous operands per product (P D + Q X), and an epilogue functor per use.
//
// P pieces per operand carry the precision.  P = 1: the f16 / bf16 values.  P = 2: an f32 value x is held as two f16 pieces,
// x = hi + lo (11 + 11 significand bits), and x y ~= hi hi' + hi lo' + lo hi': three matrix products per fragment pair; what is
// dropped is below 2^-22 |x y|.  The pieces lie interleaved, 32 hi then 32 lo of the same 32 k, so that both forms have
// the same 128-byte k step in memory and in LDS and differ only in which fragments meet.
//
// Operand contract (checked by the callers on the host): rows are k-contiguous and 16-byte aligned, K (stored values a row)
// is a multiple of 64 with everything beyond the true length zero, row indices past the end are clamped (never read
// outside), and the epilogue masks what the clamped rows produce.
#ifndef TCMI_MM16_H
#define TCMI_MM16_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

namespace tcmi {
namespace mm16 {

using f16 = _Float16;
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

struct Args {
  const void* a[2];
  const void* b[2];
  int nseg;
  int M, N, K;                 // K: stored values of a row, a multiple of 64
  long long lda, ldb;          // elements between rows
  long long sa, sb;            // elements between batch members
  int tm, tn;                  // tiles per matrix
  int tri;                     // 1: C is symmetric, only tiles with row tile >= column tile are computed
  int doubled;                 // > 0: C = [[R, I], [-I, R]] from a hermitian R + iI of this size
  int half;                    // `doubled` where tiles end at it: the second R is not computed, the epilogue writes the first one twice
  int tiles;                   // tiles per batch member (tm * tn, or the triangle)
  int batch;
  int split;                   // > 1: the k steps are dealt to `split` workgroups, whose sums join_kernel adds
  float* part;                 // [split][batch * tiles][BM * BN]
  int wave_rows;               // rows of C that one wave holds: an epilogue may leave something per wave and column
};

// where logical k lies in a row of P pieces (the low piece 32 further), and the padded length of a row
template <int P>
__host__ __device__ constexpr long long kpos(long long k) {
  return P == 1 ? k : ((k >> 5) << 6) + (k & 31);
}
__host__ __device__ constexpr long long kpad(long long k, int P) { return P == 1 ? (k + 63) & ~63ll : (k + 31) & ~31ll; }

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// tile t of a batch member
__device__ __forceinline__ void tile_at(const Args& g, unsigned t, int& ti, int& tj) {
  if (g.tri) {
    const unsigned h = g.half ? (unsigned)g.tm / 2u : 0u, r = h * (h + 1) / 2;
    if (g.half && t >= r) {                           // below the triangle of R: the square of -I
      ti = (int)(h + (t - r) / h);
      tj = (int)((t - r) % h);
      return;
    }
    unsigned i = (unsigned)((sqrtf(8.f * (float)t + 1.f) - 1.f) * 0.5f);
    while (i * (i + 1) / 2 > t) --i;
    while ((i + 1) * (i + 2) / 2 <= t) ++i;
    ti = (int)i;
    tj = (int)(t - i * (i + 1) / 2);
  } else {                                          // bands of 8 row tiles: their operand rows stay in an L2
    const unsigned band = t / (8u * g.tn), in = t % (8u * g.tn);
    const unsigned rows = min(8u, (unsigned)g.tm - band * 8u);
    ti = (int)(band * 8u + in % rows);
    tj = (int)(in / rows);
  }
}

// Workgroups go to the eight XCDs in turn; renumbered so that each XCD (its own L2) gets one contiguous range.
__device__ __forceinline__ unsigned unit_of() {
  const unsigned total = gridDim.x, id = blockIdx.x;
  const unsigned q = total >> 3, r = total & 7, x = id & 7;
  return (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + (id >> 3);
}

template <int BM_, int BN_, int WM_, int WN_, int PER_CU_, int STAGES_>
struct Tile {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, PER_CU = PER_CU_;
  static constexpr int WAVES = WM * WN, THREADS = WAVES * 64;
  static constexpr int MI = BM / WM / 16, NI = BN / WN / 16;
  static constexpr int STAGE = (BM + BN) * 128;            // bytes of one k step of both operands
  static constexpr int STAGES = STAGES_, LDS = STAGES * STAGE;
  static constexpr int LOADS = (BM + BN) / 8 / WAVES;      // loads of a wave per step
  static_assert((STAGES - 1) * LOADS < 64, "vmcnt holds 6 bits");
  static constexpr int YOUNG = (STAGES - 2) * LOADS;       // loads that may still be under way in the middle of a step
};

using LdsPtr = __attribute__((address_space(3))) void*;

// Waits until all but this wave's YOUNG youngest loads have landed in LDS and none of its LDS reads is under way, then for the
// other waves; no memory operation moves across (the compiler's own barrier would wait for every load).
template <int YOUNG>
__device__ __forceinline__ void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(YOUNG) : "memory");
}

// Asks the scheduler to deal LDS reads (and loads) out between the matrix instructions of half a step.  Issued in one go they
// hold all eight waves of a 256 x 256 tile at the LDS queue while the matrix pipe idles: 8192^3 f16 880 -> 825 us, and
// 117 -> 110 us for 4096^3; the smaller tiles, which share a CU with other workgroups, do not change.
template <class T, bool LOADS>
__device__ __forceinline__ void mix() {
  constexpr int READS = T::MI + T::NI, MULS = T::MI * T::NI, MFMA = 0x8, VMEM = 0x20, DS = 0x100;
  if constexpr (LOADS) {
#pragma unroll
    for (int k = 0; k < T::LOADS; ++k) {
      __builtin_amdgcn_sched_group_barrier(DS, (READS + T::LOADS - 1) / T::LOADS, 0);
      __builtin_amdgcn_sched_group_barrier(VMEM, 1, 0);
      __builtin_amdgcn_sched_group_barrier(MFMA, MULS / T::LOADS, 0);
    }
  } else {
#pragma unroll
    for (int k = 0; k < READS; ++k) {
      __builtin_amdgcn_sched_group_barrier(DS, 1, 0);
      __builtin_amdgcn_sched_group_barrier(MFMA, MULS / READS, 0);
    }
  }
}

#ifdef __HIP_DEVICE_COMPILE__          // the host pass does not know the buffer resource type
// The k steps [s0, s1) of one product tile.  `acc[i][j]` holds C[row][col .. col + 3] with
// row = m0 + (wm MI + i) 16 + (lane & 15) and col = n0 + (wn NI + j) 16 + 4 (lane >> 4): the B fragment is the first
// matrix operand, so a lane ends with four neighbouring columns of one row.
//
// LDS: a row's k step is eight 16-byte chunks; chunk c of row r lies at position c ^ (r & 7), which spreads the 16 rows of a
// fragment read over all banks.  Global -> LDS goes without registers (buffer_load ... lds) into two stages; fragments go
// LDS -> registers half a step ahead of the matrix instructions that use them.  One barrier a step: when every wave has its
// stage in registers and its loads of the next stage have landed, the stage is free for the loads STAGES steps on.
template <class V, int P, class T>
__device__ __forceinline__ void product(const Args& g, int m0, int n0, int bz, int s0, int s1, char* lds, f32x4 (&acc)[T::MI][T::NI]) {
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
  const int ksteps = g.K >> 6;
  int ls = s0 / ksteps, lk = s0 % ksteps;                               // segment and k step of the next load

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
    const int wrap = lk + 1 == ksteps;
    lk = wrap ? 0 : lk + 1;
    ls += wrap;
  };

  const int r = lane & 15;
  const int at[2] = {(((lane >> 4)) ^ (r & 7)) * 16 + r * 128, ((4 + (lane >> 4)) ^ (r & 7)) * 16 + r * 128};
  const char* pa = lds + (wm * T::MI * 16) * 128;
  const char* pb = lds + (T::BM + wn * T::NI * 16) * 128;
  auto read_a = [&](V (&f)[T::MI], int stage, int half) {
#pragma unroll
    for (int i = 0; i < T::MI; ++i) f[i] = *reinterpret_cast<const V*>(pa + stage * T::STAGE + i * 2048 + at[half]);
  };
  auto read_b = [&](V (&f)[T::NI], int stage, int half) {
#pragma unroll
    for (int i = 0; i < T::NI; ++i) f[i] = *reinterpret_cast<const V*>(pb + stage * T::STAGE + i * 2048 + at[half]);
  };
  auto multiply = [&](const V (&fa)[T::MI], const V (&fb)[T::NI]) {
#pragma unroll
    for (int i = 0; i < T::MI; ++i)
#pragma unroll
      for (int j = 0; j < T::NI; ++j) acc[i][j] = mfma(fb[j], fa[i], acc[i][j]);
  };
  V a0[T::MI], a1[T::MI], b0[T::NI], b1[T::NI], b2[T::NI];
  // One k step: b holds the first half's B fragments, bn receives the next step's.  MORE: a next step exists, FILL: so does the
  // one whose loads take this stage (constants: no branches in the loop).
  int stage = 0;
  auto step = [&](auto more, auto fill, V (&b)[T::NI], V (&bn)[T::NI]) {
    const int next = stage + 1 == T::STAGES ? 0 : stage + 1;
    read_b(b1, stage, 1);
    read_a(a1, stage, 1);
    multiply(a0, b);
    if constexpr (T::PER_CU == 1) mix<T, false>();
    if constexpr (P == 2) multiply(a0, b1);
    if constexpr (more) {
      // this stage is in registers, the next one has landed (near the end, where fewer loads are under way: all have)
      wait_and_meet<fill ? T::YOUNG : 0>();
      if constexpr (fill) load(stage);
      read_b(bn, next, 0);
      read_a(a0, next, 0);
    }
    if constexpr (P == 1) multiply(a1, b1);
    else multiply(a1, b);
    if constexpr (fill && T::PER_CU == 1) mix<T, true>();
    stage = next;
  };
  constexpr std::true_type yes{};
  constexpr std::false_type no{};

  for (int k = 0; k < T::STAGES && s0 + k < s1; ++k) load(k);
  if (s0 + T::STAGES - 1 < s1) wait_and_meet<T::YOUNG + T::LOADS>();      // the first stage has landed
  else wait_and_meet<0>();
  read_b(b0, 0, 0);
  read_a(a0, 0, 0);
  int s = s0;
  if constexpr (P == 1) {
    for (; s + T::STAGES < s1; ++s) step(yes, yes, b0, b0);
    for (; s + 1 < s1; ++s) step(yes, no, b0, b0);
    step(no, no, b0, b0);
  } else {
    for (; s + T::STAGES + 1 < s1; s += 2) {
      step(yes, yes, b0, b2);
      step(yes, yes, b2, b0);
    }
    // at most STAGES + 1 steps left; the fragments change places with each
    for (; s + 1 < s1; ++s) {
      if (s + T::STAGES < s1) step(yes, yes, b0, b2);
      else step(yes, no, b0, b2);
#pragma unroll
      for (int i = 0; i < T::NI; ++i) b0[i] = b2[i];
    }
    step(no, no, b0, b2);
  }
}
#endif

// An epilogue works on whole tiles (TILE: void tile<T>(g, m0, n0, bz, mirror, lds, acc), with lds<T>() bytes of LDS), or on four
// neighbouring columns of a row at a time (FOUR: void four(g, bz, mirror, row, col, v); the product may then be split along
// k), or on both: tiles where it is not split.
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

template <class V, int P, class T, class Epi>
__global__ __launch_bounds__(T::THREADS, T::PER_CU * T::WAVES / 4) void product_kernel(Args g, Epi e) {
#ifdef __HIP_DEVICE_COMPILE__
  extern __shared__ __attribute__((aligned(128))) char lds[];
  const unsigned w = unit_of(), per = (unsigned)(g.tiles * g.batch), u = w % per, sp = w / per;
  const int bz = (int)(u / (unsigned)g.tiles);
  int ti, tj;
  tile_at(g, u % (unsigned)g.tiles, ti, tj);
  const int m0 = ti * T::BM, n0 = tj * T::BN, steps = (g.K >> 6) * g.nseg;
  const int s0 = (int)((long long)steps * sp / g.split), s1 = (int)((long long)steps * (sp + 1) / g.split);
  f32x4 acc[T::MI][T::NI];
#pragma unroll
  for (int i = 0; i < T::MI; ++i)
#pragma unroll
    for (int j = 0; j < T::NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  product<V, P, T>(g, m0, n0, bz, s0, s1, lds, acc);
  const bool mirror = g.tri && ti != tj;
  if constexpr (Epi::FOUR) {
    if (g.split > 1) {
      f32x4* p = reinterpret_cast<f32x4*>(g.part) + (long long)w * (T::BM * T::BN / 4) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < T::MI; ++i)
#pragma unroll
        for (int j = 0; j < T::NI; ++j) p[(i * T::NI + j) * T::THREADS] = acc[i][j];
      return;
    }
  }
  if constexpr (Epi::TILE) e.template tile<T>(g, m0, n0, bz, mirror, lds, acc);
  else each<T>(m0, n0, acc, [&](int row, int col, f32x4 v) { e.four(g, bz, mirror, row, col, v); });
#endif
}

// adds the parts of a split product in a fixed order and applies the epilogue: one workgroup per fragment column of a tile
template <class T, class Epi>
__global__ __launch_bounds__(T::THREADS) void join_kernel(Args g, Epi e) {
  constexpr unsigned F = T::MI * T::NI;
  const unsigned u = blockIdx.x / F, f = blockIdx.x % F, per = (unsigned)(g.tiles * g.batch);
  const int bz = (int)(u / (unsigned)g.tiles);
  int ti, tj;
  tile_at(g, u % (unsigned)g.tiles, ti, tj);
  const f32x4* p = reinterpret_cast<const f32x4*>(g.part) + (long long)u * (T::BM * T::BN / 4) + f * T::THREADS + threadIdx.x;
  const long long step = (long long)per * (T::BM * T::BN / 4);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < g.split; ++k) v += p[k * step];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int row = ti * T::BM + (wave / T::WN) * T::MI * 16 + (int)(f / T::NI) * 16 + (lane & 15);
  const int col = tj * T::BN + (wave % T::WN) * T::NI * 16 + (int)(f % T::NI) * 16 + 4 * (lane >> 4);
  e.four(g, bz, g.tri && ti != tj, row, col, v);
}

__device__ __forceinline__ void two_pieces(float x, f16& hi, f16& lo) {
  hi = (f16)x;
  lo = (f16)(x - (float)hi);
}

// four neighbouring values, stored as P pieces at logical column col (a multiple of 4)
template <int P>
__device__ __forceinline__ void store_four(f16* row, int col, const f16x4& hi, const f16x4& lo) {
  f16* p = row + kpos<P>(col);
  *reinterpret_cast<f16x4*>(p) = hi;
  if (P == 2) *reinterpret_cast<f16x4*>(p + 32) = lo;
}

// A tile's transpose through LDS: lines BM + 8 elements long (16-byte aligned, no bank conflicts), the low pieces behind the
// high ones.  stage() takes a lane's four values, flush() stores eight neighbours a thread: row c of the transpose at
// base + c * ld, its logical columns m0 .. , rows below `rows` and columns below `cols` (a multiple of 8).
template <class T, int P>
struct Transposed {
  static constexpr int LINE = T::BM + 8, BYTES = P * T::BN * LINE * 2;
  f16* lds;
  __device__ __forceinline__ void stage(int rl, int cl, const f16x4& hi, const f16x4& lo) const {
    f16* o = lds + cl * LINE + rl;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      o[r * LINE] = hi[r];
      if (P == 2) o[(T::BN + r) * LINE] = lo[r];
    }
  }
  __device__ __forceinline__ void flush(f16* base, long long ld, int n0, int rows, int m0, int cols) const {
    for (int k = threadIdx.x; k < T::BN * (T::BM / 8); k += T::THREADS) {
      const int c = k / (T::BM / 8), rl = k % (T::BM / 8) * 8;
      if (n0 + c >= rows || m0 + rl >= cols) continue;
      f16* o = base + (long long)(n0 + c) * ld + kpos<P>(m0 + rl);
      *reinterpret_cast<f16x8*>(o) = *reinterpret_cast<const f16x8*>(lds + c * LINE + rl);
      if (P == 2) *reinterpret_cast<f16x8*>(o + 32) = *reinterpret_cast<const f16x8*>(lds + (T::BN + c) * LINE + rl);
    }
  }
  // the other half of a doubled complex matrix: row c of the transpose goes to row c + n (the real part, c < n), or negated to
  // row c - n, `cols` columns further on (cols and n multiples of 16)
  __device__ __forceinline__ void flush_twin(f16* base, long long ld, int n0, int rows, int m0, int cols, int n) const {
    for (int k = threadIdx.x; k < T::BN * (T::BM / 8); k += T::THREADS) {
      const int c = k / (T::BM / 8), rl = k % (T::BM / 8) * 8;
      if (n0 + c >= rows || m0 + rl >= cols) continue;
      const bool im = n0 + c >= n;
      f16* o = base + (long long)(n0 + c + (im ? -n : n)) * ld + kpos<P>(m0 + rl + cols);
      f16x8 v = *reinterpret_cast<const f16x8*>(lds + c * LINE + rl);
      *reinterpret_cast<f16x8*>(o) = im ? -v : v;
      if (P == 2) {
        v = *reinterpret_cast<const f16x8*>(lds + (T::BN + c) * LINE + rl);
        *reinterpret_cast<f16x8*>(o + 32) = im ? -v : v;
      }
    }
  }
};

// ---- host side ----
using Big = Tile<256, 256, 2, 4, 1, 2>;
using Wide = Tile<192, 192, 2, 4, 1, 2>;
using Mid = Tile<128, 128, 2, 2, 2, 2>;
using Slim = Tile<128, 64, 4, 1, 2, 2>;
using Tiny = Tile<64, 64, 2, 2, 4, 2>;

constexpr long long PART_BYTES = 512ll * 128 * 128 * 4;       // workspace of a split product

// Which tile, and into how many parts along k.  Time of one k step of one round in microseconds, by the workgroups that share a
// CU, measured on products of 1000 .. 8192 rows (one / two pieces):
//   256 x 256   1.8                    one workgroup a CU; 1120 - 1180 TFLOP/s when the card is full
//   192 x 192   1.19                   one; 253 tiles of a 4096 x 4096 symmetric result: 76 us (256: 107, 128: 100)
//   128 x 128   0.72 / 0.73, two 1.02 / 1.2          1080 TFLOP/s; two pieces 446 (1340 on the pipe)
//   128 x 64    0.60, two 0.69 / 0.71                results up to 64 columns
//   64 x 64     0.38 / 0.48, two 0.56 / 0.58, three 0.68 / 0.70, four 0.79 / 0.80
// A product whose tiles do not fill the card takes smaller tiles (1000 x 1537 x 1000, two pieces: 18 us, 128 x 128: 27) or
// is split along k; its parts cost a second launch (4 us) and one write and one read of themselves (4 TB/s).
template <class T, int P>
inline double step_us(int per_cu) {
  const double one = P == 1;
  if (T::BM == 256) return 1.8;
  if (T::BM == 192) return 1.19;
  if (T::BM == 128 && T::BN == 128) return per_cu == 1 ? (one ? 0.72 : 0.73) : (one ? 1.02 : 1.2);
  if (T::BM == 128) return per_cu == 1 ? 0.60 : (one ? 0.69 : 0.71);
  return per_cu == 1 ? (one ? 0.38 : 0.48) : per_cu == 2 ? (one ? 0.56 : 0.58) : per_cu == 3 ? (one ? 0.68 : 0.70) : (one ? 0.79 : 0.80);
}

// whether a doubled hermitian result leaves out the second R (up to a quarter of the triangle's tiles): orthogonalising
// 2048 x 2048 complex64 3.41 -> 2.68 ms; 62 x 256 x 128, one round of tiles either way, 2 %
template <class T>
inline bool halves(const Args& g, bool tri) {
  return tri && T::BM == T::BN && g.doubled > 0 && g.doubled % T::BM == 0 && g.M == 2 * g.doubled;
}

template <class T>
inline long long tile_count(const Args& g, bool tri) {
  const long long tm = (g.M + T::BM - 1) / T::BM, tn = (g.N + T::BN - 1) / T::BN;
  return (halves<T>(g, tri) ? tm / 2 * (tm / 2 + 1) / 2 + tm / 2 * (tm / 2) : tri ? tm * (tm + 1) / 2 : tm * tn) * g.batch;
}

// the cheapest split of a product over tiles T, and its time
template <class T, int P>
inline double cost_of(const Args& g, bool tri, bool may_split, int* split) {
  const long long units = tile_count<T>(g, tri), steps = (long long)(g.K / 64) * g.nseg;
  double best = 1e30;
  for (const int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32}) {
    if (s > 1 && (!may_split || steps < 4 * s || units * s * T::BM * T::BN * 4 > PART_BYTES)) break;
    const long long u = units * s, round = 256 * T::PER_CU, rest = u % round, k = (steps + s - 1) / s;
    double t = k * ((u / round) * step_us<T, P>(T::PER_CU) + (rest ? step_us<T, P>((int)((rest + 255) / 256)) : 0.0));
    if (s > 1) t += 4.0 + u * T::BM * T::BN * 8.0 / 4e6;
    if (t < best) {
      best = t;
      *split = s;
    }
  }
  return best;
}

// Raises a kernel's limit of dynamic LDS, once per device (`done`: one bit each, up to 64; later devices every time).
inline hipError_t raise_lds(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return hipSuccess;
  e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == hipSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

constexpr long long MAX_ROW = 1ll << 22;       // elements between rows: 256 of them stay within 32-bit byte offsets

template <class V, int P, class T, class Epi>
hipError_t launch(Args& g, bool tri, int split, const Epi& e, hipStream_t st) {
  g.tm = (g.M + T::BM - 1) / T::BM;
  g.tn = (g.N + T::BN - 1) / T::BN;
  g.tri = tri ? 1 : 0;
  g.wave_rows = T::MI * 16;
  if (g.batch < 1) return hipErrorInvalidValue;
  g.half = halves<T>(g, tri) ? g.doubled : 0;
  const long long units = tile_count<T>(g, tri), tiles = units / g.batch;
  if (units < 1 || units >= (1ll << 24) || g.K < 64 || (g.K & 63) || g.nseg < 1 || g.lda > MAX_ROW || g.ldb > MAX_ROW) return hipErrorInvalidValue;
  g.tiles = (int)tiles;
  g.split = split;
  int lds = T::LDS;
  if constexpr (Epi::TILE) lds = lds > Epi::template lds<T>() ? lds : Epi::template lds<T>();
  static std::atomic<unsigned long long> done{0};
  hipError_t r = raise_lds(reinterpret_cast<const void*>(product_kernel<V, P, T, Epi>), lds, done);
  if (r != hipSuccess) return r;
  hipLaunchKernelGGL((product_kernel<V, P, T, Epi>), dim3((unsigned)(units * g.split)), dim3(T::THREADS), lds, st, g, e);
  r = hipGetLastError();
  if constexpr (Epi::FOUR) {
    if (r == hipSuccess && g.split > 1) {
      hipLaunchKernelGGL((join_kernel<T, Epi>), dim3((unsigned)(units * T::MI * T::NI)), dim3(T::THREADS), 0, st, g, e);
      r = hipGetLastError();
    }
  }
  return r;
}

template <class V, int P, class Epi>
hipError_t launch_best(Args& g, bool tri, const Epi& e, hipStream_t st) {
  const bool may = Epi::FOUR && g.part;
  int split[5] = {1, 1, 1, 1, 1};
  const double big = P == 1 ? cost_of<Big, P>(g, tri, may, split) : 1e30, wide = P == 1 ? cost_of<Wide, P>(g, tri, may, split + 1) : 1e30,
               mid = cost_of<Mid, P>(g, tri, may, split + 2), slim = tri ? 1e30 : cost_of<Slim, P>(g, tri, may, split + 3),
               tiny = cost_of<Tiny, P>(g, tri, may, split + 4);
  if constexpr (P == 1) {
    if (big <= wide && big <= mid && big <= slim && big <= tiny) return launch<V, P, Big>(g, tri, split[0], e, st);
    if (wide <= mid && wide <= slim && wide <= tiny) return launch<V, P, Wide>(g, tri, split[1], e, st);
  }
  if (mid <= slim && mid <= tiny) return launch<V, P, Mid>(g, tri, split[2], e, st);
  if (slim <= tiny) return launch<V, P, Slim>(g, tri, split[3], e, st);
  return launch<V, P, Tiny>(g, tri, split[4], e, st);
}

}  // namespace mm16
}  // namespace tcmi

#endif
