// Block-scaled e4m3 (gfx950): the activation quantiser and the matrix product, with one f32
// scale for each 128 elements of an activation row and each 128 x 128 block of a weight.
//
//   quant: group g of row m: s = max(amax |x| / 448, 2^-126) (pow2: the next power of two at
//          or above it), q = e4m3(x / s), s -> scale[g][m]
//   gemm:  C[m][n] = Σ_g sA[g][m] sB[n / 128][g] Σ_{k in g} A[m][k] B[n][k]  (+ bias, GELU, R)
#include <math.h>
#include <algorithm>
#include "vit_common.h"

namespace {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));

// ---- quantiser -------------------------------------------------------------------------
// HBM bound (one read, half to a quarter of it written).  16 lanes hold a group, 8 elements
// each; amax is the integer maximum of the magnitudes' bits, so an Inf or NaN in a group wins
// and makes the group's scale NaN (its products are NaN, not wrong numbers).  The quotient is
// the correctly rounded f32 one, so that q is a function of x and s alone: by the reciprocal of
// a power of two, else from the rounded reciprocal r as q0 = x r, q0 + (x - q0 s) r, which is
// the division's result wherever the remainder is exact (4 operations where a division takes
// about 12, half of the kernel's time; groups that small that the remainder would be denormal
// are scaled up first).  A block takes a group of 16 rows, whose scales lie side by side.
// 16,384 x 7,168 bf16: 65 us, 5.5 TB/s (79 with the division and 16 groups of a row in a
// block; no gain from 4 groups' loads in flight); 768 x 4,096: 3.5 us, a launch's latency.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  typedef T v8 __attribute__((ext_vector_type(8)));
  const v8 x = *reinterpret_cast<const v8*>(p);
#pragma unroll
  for (int i = 0; i < 8; i++) v[i] = (float)x[i];
}

template <typename T, bool POW2>
__global__ __launch_bounds__(256) void quant_block_kernel(const T* __restrict__ x, int64_t ldx,
                                                          uint8_t* __restrict__ q, int64_t ldq,
                                                          float* __restrict__ scale, int64_t lds_,
                                                          int64_t M, int K, uint32_t groups) {
  const uint32_t rt = blockIdx.x / groups, g = blockIdx.x - rt * groups;
  const int l = threadIdx.x & 15, k = (int)g * 128 + l * 8;
  const int64_t m = (int64_t)rt * 16 + (threadIdx.x >> 4);
  if (m >= M) return;
  float v[8] = {};
  if (k < K) load8(x + m * ldx + k, v);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; i++) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  float s = fmaxf(__uint_as_float(top) / 448.0f, 1.17549435e-38f);
  if (POW2) s = __uint_as_float((__float_as_uint(s) + 0x7fffffu) & 0x7f800000u);
  if (top >= 0x7f800000u) s = __uint_as_float(0x7fc00000u);
  if (l == 0) scale[(int64_t)g * lds_ + m] = s;
  if (k >= K) return;
  float y[8];
  if (POW2) {
    const float r = 1.0f / s;
#pragma unroll
    for (int i = 0; i < 8; i++) y[i] = v[i] * r;
  } else {
    const float up = s < 0x1p-64f ? 0x1p64f : 1.0f, z = s * up, r = 1.0f / z;
#pragma unroll
    for (int i = 0; i < 8; i++) {   // |y| <= 448 (1 + 2^-23): rounds to 448
      const float w = v[i] * up, q0 = w * r;
      y[i] = __builtin_fmaf(__builtin_fmaf(-q0, z, w), r, q0);
    }
  }
  int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
  int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
  *reinterpret_cast<uint2*>(q + m * ldq + k) = make_uint2(lo, hi);
}

// ---- product ---------------------------------------------------------------------------
struct GArgs {
  const uint8_t *A, *B;
  const float *sa, *sb, *bias, *R;
  void* C;
  int64_t lda, ldb, ld_sa, ld_sb, ldc, ldr;
  int M, N, K, groups, out_type, gelu, vec;
  int tiles_m, tiles_n;
};

constexpr uint32_t OOB = 0x80000000u;

template <int N>
__device__ __forceinline__ void vm_wait() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

__device__ __forceinline__ void block_sync_lds() {
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

__device__ __forceinline__ void glds16(__amdgpu_buffer_rsrc_t r, char* lds, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds), 16,
                                           voff, 0, 0, 0);
}

__device__ __forceinline__ void glds4(__amdgpu_buffer_rsrc_t r, char* lds, uint32_t voff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds), 4,
                                           voff, 0, 0, 0);
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, bytes, 0x00020000);
}

__device__ __forceinline__ void load8f(const float* p, float (&v)[8]) {
  const f32x4 x = *reinterpret_cast<const f32x4*>(p), y = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; i++) v[i] = x[i], v[4 + i] = y[i];
}

template <typename T>
__device__ __forceinline__ void store8h(void* c, int64_t at, const float (&v)[8]) {
  typedef T v8 __attribute__((ext_vector_type(8)));
  v8 o;
#pragma unroll
  for (int i = 0; i < 8; i++) o[i] = (T)v[i];
  *reinterpret_cast<v8*>(reinterpret_cast<T*>(c) + at) = o;
}

// Results leave through LDS: a lane's accumulators are 4 columns of one row each, stored
// directly they would be 32-B pieces of 16 rows.  cs: f32 [ROWS][COLS + 4]; a thread takes 8
// columns of every (NT / (COLS / 8))-th row, summed over KS such tiles.  Bias and residual are
// all read before the first store: a load's wait counts the stores in front of it too, a memory
// round trip for every row.
// The code is kept small (one rolled loop for rows without 16-B alignment, types chosen at run
// time): inlined for every case it was 250 KB, and its instruction fetches took 10 us a tile.
template <int ROWS, int COLS, int NT, int KS, bool RES>
__device__ __forceinline__ void store_wide(const GArgs& a, const float* cs, int m0, int n, int c,
                                           int r0) {
  constexpr int STEP = NT * 8 / COLS, IT = ROWS < STEP ? 1 : ROWS / STEP;
  static_assert(ROWS < STEP || IT * STEP == ROWS, "whole rows");
  if (ROWS < STEP && r0 >= ROWS) return;
  float bias[8] = {}, res[RES ? IT : 1][8];
  if (a.bias) load8f(a.bias + n, bias);
  if constexpr (RES) {
#pragma unroll
    for (int it = 0; it < IT; it++) {   // a row past the end: the last one again
      const int m = min(m0 + r0 + it * STEP, a.M - 1);
      load8f(a.R + m * a.ldr + n, res[it]);
    }
  }
#pragma unroll
  for (int it = 0; it < IT; it++) {
    const int r = r0 + it * STEP, m = m0 + r;
    if (m >= a.M) break;
    float v[8];
    load8f(cs + r * (COLS + 4) + c, v);
#pragma unroll
    for (int k = 1; k < KS; k++) {
      float w[8];
      load8f(cs + (k * ROWS + r) * (COLS + 4) + c, w);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] += w[i];
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] += bias[i];
    if (a.gelu) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = gelu_erf(v[i]);
    }
    if constexpr (RES) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] += res[it][i];
    }
    const int64_t at = m * a.ldc + n;
    if (a.out_type == M3S_BF16) {
      store8h<bf16_t>(a.C, at, v);
    } else if (a.out_type == M3S_F16) {
      store8h<_Float16>(a.C, at, v);
    } else {
      f32x4* o = reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.C) + at);
      o[0] = f32x4{v[0], v[1], v[2], v[3]};
      o[1] = f32x4{v[4], v[5], v[6], v[7]};
    }
  }
}

template <int ROWS, int COLS, int NT, int KS>
__device__ __forceinline__ void store_tile(const GArgs& a, const float* cs, int m0, int n0,
                                           int tid) {
  constexpr int TPR = COLS / 8;
  const int c = tid % TPR * 8, r0 = tid / TPR, n = n0 + c;
  if (a.vec && n + 8 <= a.N) {
    if (a.R) store_wide<ROWS, COLS, NT, KS, true>(a, cs, m0, n, c, r0);
    else store_wide<ROWS, COLS, NT, KS, false>(a, cs, m0, n, c, r0);
    return;
  }
  // the last columns, and rows without 16-B alignment: a thread keeps one column (its bias read
  // once) of every (NT / COLS)-th row; neighbours store neighbouring elements
  const bool all = !a.vec;
  const int edge = all ? 0 : (a.N - n0) / 8 * 8;
  const int width = min(a.N - n0, COLS) - edge;
  // with a.vec the threads of the cut chunk walk its columns themselves, and those whose chunks
  // lie behind it have none (R may be C: an element is read and written by one thread)
  const int c1 = all ? tid % COLS : edge, r1 = all ? tid / COLS : r0;
  const int step = all ? NT / COLS : NT / TPR;
  const int last = all ? c1 + 1 : edge + width;
  if (n0 + c1 >= a.N || (!all && c != edge)) return;
#pragma unroll 1
  for (int cc = c1; cc < last; cc++) {
    const float bias = a.bias ? a.bias[n0 + cc] : 0.f;
#pragma unroll 1
    for (int r = r1; r < ROWS && m0 + r < a.M; r += 8 * step) {
      float res[8];
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int m = min(m0 + r + i * step, a.M - 1);
        res[i] = a.R ? a.R[m * a.ldr + n0 + cc] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int rr = r + i * step, m = m0 + rr;
        if (rr >= ROWS || m >= a.M) break;
        float v = cs[rr * (COLS + 4) + cc];
#pragma unroll
        for (int k = 1; k < KS; k++) v += cs[(k * ROWS + rr) * (COLS + 4) + cc];
        v += bias;
        if (a.gelu) v = gelu_erf(v);
        v += res[i];
        const int64_t at = m * a.ldc + n0 + cc;
        if (a.out_type == M3S_BF16) ((bf16_t*)a.C)[at] = f2bf(v);
        else if (a.out_type == M3S_F16) ((_Float16*)a.C)[at] = (_Float16)v;
        else ((float*)a.C)[at] = v;
      }
    }
  }
}

// Block → tile.  Consecutive blocks go round the 8 XCDs; the remap gives an XCD a contiguous run
// of tiles, walked in groups of 8 row bands column by column, so that the run is a compact
// rectangle and its A bands and B columns are found in the XCD's L2.
__device__ __forceinline__ void tile_of(const GArgs& a, int& tm, int& tn) {
  const int total = gridDim.x, orig = blockIdx.x;
  int lin = orig;
  if (total >= 16) {
    const int qq = total / 8, rr = total % 8, xcd = orig % 8;
    lin = (xcd < rr ? xcd * (qq + 1) : rr * (qq + 1) + (xcd - rr) * qq) + orig / 8;
  }
  const int per = 8 * a.tiles_n, grp = lin / per, first = grp * 8;
  const int high = min(a.tiles_m - first, 8), in = lin - grp * per;
  tn = in / high;
  tm = first + in - tn * high;
}

// BM x BN tile, KS groups of WM x WN waves, each with a ring of NST stages of 128 K-bytes (one
// scale group) filled by LDS-DMA; group g takes the K-tiles g, g + KS, ... and the groups' sums
// join in LDS.  (A K-tile of one group is a chain of barrier, LDS reads, matrix instructions and
// FMAs.  With one block a CU a second group fills it, and the next K-tile's LDS reads run beside
// this one's matrix instructions; what is left is a CU's DMA rate: 768 x 1024 x K takes 0.205 us
// more for each K-tile of 64 + 64 rows, 80 B/ns or 35 a cycle.  With KS = 1 three blocks a CU do
// it, and the pipeline's registers would take one of them away.)
// The 16x16x128 matrix instruction takes a whole group: weights on the accumulator rows,
// activations on the lanes, so an accumulator quad belongs to one activation row and its group's
// factor sA sB is one value per lane and 16-row tile: acc += factor * partial, four FMAs beside
// the 32 cycles of the next matrix instruction.
// The instruction's own sums are f32 between groups of 8 products; the 8 are cut off 13 binary
// places behind the largest one's exponent.  On random e4m3 that is 1.5e-5 of the result
// (rms; a 32-bit product 1.1e-6), 1/2500 of what rounding random factors to e4m3 leaves in it
// (3.8e-2), and 16-bit results hide it; products through bf16, which would avoid it, run at half
// the rate.
template <int BM, int BN, int WM, int WN, int NST, int KS>
__global__ __launch_bounds__(WM* WN* KS * 64, 2) void gemm_block_kernel(GArgs a) {
  constexpr int GT = WM * WN * 64, NT = GT * KS;
  constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int AB = BM * 128, BB = BN * 128, STAGE = AB + BB + GT * 4;
  constexpr int CA = BM * 8 / GT, CB = BN * 8 / GT;   // DMA instructions per wave
  static_assert(CA * GT == BM * 8 && CB * GT == BN * 8 && BM < GT, "whole DMA instructions");
  static_assert(BN <= 128, "a tile's columns share one weight scale");
  static_assert(KS * BM * (BN + 4) * 4 <= KS * NST * STAGE, "the result tiles fit in the rings");
  static_assert(KS * NST * STAGE <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) char lds[KS * NST * STAGE];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wall = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wid = wall % (WM * WN), ksp = wall / (WM * WN);
  const int gtid = tid - ksp * GT;
  char* const ring = lds + ksp * NST * STAGE;
  const int wm = wid / WN, wn = wid % WN;
  int tm, tn;
  tile_of(a, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  // operand rows from the block's own base (no 32-bit limit on the matrices): rows past the
  // end lie behind the descriptor's size and read as zeros
  const int ma = min(a.M - m0, BM), nb = min(a.N - n0, BN);
  const __amdgpu_buffer_rsrc_t rA =
      rsrc(a.A + (int64_t)m0 * a.lda, (ma - 1) * (int)a.lda + a.K);
  const __amdgpu_buffer_rsrc_t rB =
      rsrc(a.B + (int64_t)n0 * a.ldb, (nb - 1) * (int)a.ldb + a.K);
  // DMA: thread chunk i GT + gtid is row i GT / 8 + gtid / 8, 16 B at kc (swizzled by the row;
  // the same for every i)
  static_assert(GT / 8 % 16 == 0, "one swizzle per thread");
  const int kc = ((gtid & 7) ^ ((gtid >> 4) & 7)) * 16;
  const uint32_t offa = (uint32_t)((gtid >> 3) * (int)a.lda + kc);
  const uint32_t offb = (uint32_t)((gtid >> 3) * (int)a.ldb + kc);
  const float* wscale = a.sb + (int64_t)(n0 / 128) * a.ld_sb;
  auto issue = [&](int j) {   // the group's j-th K-tile
    const int t = ksp + KS * j, k0 = t * 128;
    char* sb = ring + (j % NST) * STAGE;
    const bool in = kc < a.K - k0;   // past K lies the next row
#pragma unroll
    for (int i = 0; i < CA; i++)
      glds16(rA, sb + (i * GT + wid * 64) * 16,
             in ? offa + (uint32_t)(k0 + i * (GT / 8) * (int)a.lda) : OOB);
#pragma unroll
    for (int i = 0; i < CB; i++)
      glds16(rB, sb + AB + (i * GT + wid * 64) * 16,
             in ? offb + (uint32_t)(k0 + i * (GT / 8) * (int)a.ldb) : OOB);
    // scales: the tile's rows from the first BM / 64 waves, the weight block from the next
    const bool act = wid < (BM + 63) / 64;
    const __amdgpu_buffer_rsrc_t rS =
        rsrc(act ? a.sa + (int64_t)t * a.ld_sa + m0 : wscale + t, act ? ma * 4 : 4);
    glds4(rS, sb + AB + BB + wid * 64 * 4, act ? gtid * 4 : gtid == (BM + 63) / 64 * 64 ? 0 : OOB);
  };
  f32x4 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; j++)
#pragma unroll
    for (int i = 0; i < TM; i++) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int fr = lane & 15, fc = lane >> 4, sw = fr >> 1;
  const int lo0 = fr * 128 + ((fc ^ sw) << 4), lo1 = fr * 128 + (((fc ^ sw) ^ 4) << 4);
  const int nj = (a.groups + KS - 1) / KS;                                        // all groups
  const int nme = a.groups > ksp ? (a.groups - ksp + KS - 1) / KS : 0;   // this group
  struct Frag {
    i32x8 a[TM], b[TN];
    float s[TM], sb;
  };
  auto read = [&](int j, Frag& f) __attribute__((always_inline)) {
    const char* cur = ring + (j % NST) * STAGE;
    f.sb = *reinterpret_cast<const float*>(cur + AB + BB + (BM + 63) / 64 * 256);
#pragma unroll
    for (int i = 0; i < TM; i++) {
      const char* base = cur + (wm * (BM / WM) + i * 16) * 128;
      const i32x4 x = *reinterpret_cast<const i32x4*>(base + lo0);
      const i32x4 y = *reinterpret_cast<const i32x4*>(base + lo1);
      f.a[i] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
      f.s[i] = *reinterpret_cast<const float*>(cur + AB + BB +
                                               (wm * (BM / WM) + i * 16 + fr) * 4);
    }
#pragma unroll
    for (int jn = 0; jn < TN; jn++) {
      const char* base = cur + AB + (wn * (BN / WN) + jn * 16) * 128;
      const i32x4 x = *reinterpret_cast<const i32x4*>(base + lo0);
      const i32x4 y = *reinterpret_cast<const i32x4*>(base + lo1);
      f.b[jn] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  };
  auto mma = [&](const Frag& f) __attribute__((always_inline)) {
    float sc[TM];
#pragma unroll
    for (int i = 0; i < TM; i++) sc[i] = f.sb * f.s[i];
#pragma unroll
    for (int jn = 0; jn < TN; jn++)
#pragma unroll
      for (int i = 0; i < TM; i++) {
        const f32x4 p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            f.b[jn], f.a[i], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
        for (int e = 0; e < 4; e++)
          acc[jn][i][e] = __builtin_fmaf(p[e], sc[i], acc[jn][i][e]);
      }
  };
  constexpr int PER = CA + CB + 1;
  if constexpr (KS == 1) {
    // several blocks a CU fill each other's waits
#pragma unroll
    for (int st = 0; st < NST - 1; st++)
      if (st < nme) issue(st);
#pragma unroll 1
    for (int j = 0; j < nme; j++) {
      if (j + NST - 2 < nme) vm_wait<PER*(NST - 2)>();
      else vm_wait<0>();
      block_sync_lds();
      if (j + NST - 1 < nme) issue(j + NST - 1);
      Frag f;
      read(j, f);
      mma(f);
    }
  } else {
    // Trip j reads the next K-tile's operands into registers beside the matrix instructions of
    // its own, and issues DMA into the slot that trip j - 1 read, free behind the barrier: last,
    // since a wave waits about 100 cycles for each of its DMA instructions to go out
#pragma unroll
    for (int st = 0; st < NST; st++)
      if (st < nme) issue(st);
    if (NST <= nme) vm_wait<PER*(NST - 1)>();
    else vm_wait<0>();
    block_sync_lds();
    Frag even, odd;
    read(0, even);   // (a group without K-tiles reads what nothing uses)
    auto trip = [&](int j, const Frag& cur, Frag& next) __attribute__((always_inline)) {
      if (j + NST - 1 < nme) vm_wait<PER*(NST - 2)>();
      else vm_wait<0>();
      block_sync_lds();
      read(j + 1, next);
      mma(cur);
      __builtin_amdgcn_sched_barrier(0);
      if (j + NST < nme) issue(j + NST);
    };
    int j = 0;   // every group has nj - 1 K-tiles at least
#pragma unroll 1
    for (; j + 2 < nj; j += 2) {
      trip(j, even, odd);
      trip(j + 1, odd, even);
    }
    if (j + 1 < nj) {
      trip(j, even, odd);
      if (j + 1 < nme) mma(odd);
    } else if (j < nme) {
      mma(even);
    }
  }
  block_sync_lds();   // ring reads done, no DMA in flight
  float* cs = reinterpret_cast<float*>(lds) + ksp * BM * (BN + 4);
#pragma unroll
  for (int i = 0; i < TM; i++)
#pragma unroll
    for (int j = 0; j < TN; j++)
      *reinterpret_cast<f32x4*>(cs + (wm * (BM / WM) + i * 16 + fr) * (BN + 4) +
                                wn * (BN / WN) + j * 16 + fc * 4) = acc[j][i];
  block_sync_lds();
  store_tile<BM, BN, NT, KS>(a, reinterpret_cast<const float*>(lds), m0, n0, tid);
}

// Large grids: 256 x 256 tiles, 8 waves in two groups one barrier apart.  LDS holds half-tile
// slots of 128 rows x 128 B: two each of A rows 0-127 (A0), A rows 128-255 (A1) and B columns
// 0-127 (B0), three of B columns 128-255 (B1), and two of the K-tile's scales.  A K-tile (one
// scale group) is two phases, QM = 0, 1: each wave 64 rows of A half QM x 32 columns of both B
// halves, 16 matrix instructions and 64 FMAs.  Phase 0 reads A0, B0 and B1 (kept for phase 1)
// and issues A0, B0 and the scales of the next K-tile; phase 1 reads A1 and issues A1 of the
// next K-tile and B1 of the one behind it; each waits for what the phase before it issued.
// Group 1 runs one barrier behind, so that on each SIMD one wave's matrix instructions run
// beside the other's LDS reads and DMA issue.
//  * A slot issued in phase I is read in I + 2 or later: group 1's wait in phase I + 1 lies in
//    front of barrier 2I + 3, group 0 reads phase I + 2 behind it.  It is refilled two phases
//    or more after its last read Q: group 1's reads end before barrier 2Q + 2, which group 0
//    passes before it issues phase Q + 2.  (A0, B0, scales: issued 2t, read 2t + 2, refilled
//    2t + 4; A1: 2t + 1, 2t + 3, 2t + 5; B1: 2t + 1, 2t + 4, 2t + 7.)
//  * DMA issue is what a phase has to share out: a wave waits for each of its DMA instructions to
//    go out.  Hence B1 a K-tile ahead: 5 and 4 instructions a phase, not 7 and 2.
// Measured (8192 x 8192 x K, bf16): a K-tile takes 1.70 us, 3,230 cycles at the 1.9 GHz that random
// operands leave (zeros: 1.38 us, 3,040 at 2.2 GHz); its matrix instructions are 2,048 a SIMD.
// Prologue and result writes are 10-14 us a tile.  K = 4096: 255 us, 2.15 PF/s; K = 8192: 475 us,
// 2.31 PF/s.
__global__ __launch_bounds__(512, 1) void gemm_block_pp_kernel(GArgs a) {
  constexpr int HT = 128 * 128, BUFB = 3 * HT, B1 = 2 * BUFB, SC = B1 + 3 * HT;
  // 2 buffers of scales: 256 activation rows (waves 0-3), 2 weight blocks (wave 4), zeros
  __shared__ __attribute__((aligned(16))) char lds[SC + 2 * 2048];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wr = wid >> 2, wc = wid & 3;
  int tm, tn;
  tile_of(a, tm, tn);
  const int m0 = tm * 256, n0 = tn * 256;
  const int ma = min(a.M - m0, 256), nb = min(a.N - n0, 256);
  const __amdgpu_buffer_rsrc_t rA =
      rsrc(a.A + (int64_t)m0 * a.lda, (ma - 1) * (int)a.lda + a.K);
  const __amdgpu_buffer_rsrc_t rB =
      rsrc(a.B + (int64_t)n0 * a.ldb, (nb - 1) * (int)a.ldb + a.K);
  const int nk = a.groups;
  // DMA: thread chunk i * 512 + tid of a half-tile is row 64 i + tid / 8, 16 B at kc (swizzled;
  // the same for both i)
  const int kc = ((tid & 7) ^ ((tid >> 4) & 7)) * 16;
  const uint32_t offa = (uint32_t)((tid >> 3) * (int)a.lda + kc);
  const uint32_t offb = (uint32_t)((tid >> 3) * (int)a.ldb + kc);
  const float* sb = a.sb + (int64_t)(n0 / 128) * a.ld_sb;
  const int sb_bytes = (nb > 128 ? (int)a.ld_sb * 4 : 0) + 4;
  const uint32_t sb_off = wid == 4 && lane < 2 ? lane * (uint32_t)a.ld_sb * 4 : OOB;
  // half-tile h (A0 A1 B0 B1) of K-tile t
  auto slot = [&](int t, int h) { return h < 3 ? (t & 1) * BUFB + h * HT : B1 + t % 3 * HT; };
  auto issue = [&](int t, int h) {
    char* dst = lds + slot(t, h) + wid * 1024;
    const bool in = kc < a.K - t * 128;   // past K lies the next row
    const int ld = (int)(h < 2 ? a.lda : a.ldb);
#pragma unroll
    for (int i = 0; i < 2; i++)
      glds16(h < 2 ? rA : rB, dst + i * 8192,
             in ? (h < 2 ? offa : offb) + (uint32_t)(t * 128 + ((h & 1) * 128 + i * 64) * ld)
                : OOB);
    if (h == 0) {
      const bool act = wid < 4;
      const __amdgpu_buffer_rsrc_t rS =
          rsrc(act ? a.sa + (int64_t)t * a.ld_sa + m0 : sb + t, act ? ma * 4 : sb_bytes);
      glds4(rS, lds + SC + (t & 1) * 2048 + wid * 256, act ? tid * 4 : sb_off);
    }
  };
  const int fr = lane & 15, fc = lane >> 4, sw = fr >> 1;
  const int lo0 = fr * 128 + ((fc ^ sw) << 4), lo1 = fr * 128 + (((fc ^ sw) ^ 4) << 4);
  i32x8 af[4], bf[2][2];
  float sa[2][4];
  f32x4 acc[2][2][2][4];   // [QM][QN][column tile][row tile]
#pragma unroll
  for (int x = 0; x < 2; x++)
#pragma unroll
    for (int y = 0; y < 2; y++)
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[x][y][j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto frag = [&](const char* base) {
    const i32x4 x = *reinterpret_cast<const i32x4*>(base + lo0);
    const i32x4 y = *reinterpret_cast<const i32x4*>(base + lo1);
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
  };
  auto read_a = [&](int t, int qm) {
#pragma unroll
    for (int i = 0; i < 4; i++) af[i] = frag(lds + slot(t, qm) + (wr * 64 + i * 16) * 128);
  };
  // both halves' scales in phase 0: they are refilled in the next K-tile's
  auto read_scales = [&](int t) {
#pragma unroll
    for (int q = 0; q < 2; q++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        sa[q][i] = *reinterpret_cast<const float*>(lds + SC + (t & 1) * 2048 +
                                                   (q * 128 + wr * 64 + i * 16 + fr) * 4);
  };
  auto read_b = [&](int t, int qn) {
#pragma unroll
    for (int j = 0; j < 2; j++) bf[qn][j] = frag(lds + slot(t, 2 + qn) + (wc * 32 + j * 16) * 128);
  };
  // 8 partials a quadrant, in a ring of 4.  The FMAs of a partial go out 3 matrix instructions
  // behind it (its result takes 11 issue slots), those of the last three in the next quadrant:
  // every matrix instruction has 4 FMAs in its shadow and none waits for its own.
  f32x4 p[4] = {};
  float sc[4] = {};
  auto add = [&](f32x4 (&c)[2][4], int x) {
#pragma unroll
    for (int e = 0; e < 4; e++)
      c[x >> 2][x & 3][e] = __builtin_fmaf(p[x & 3][e], sc[x & 3], c[x >> 2][x & 3][e]);
    // keeps the FMAs here: sunk to the accumulators' next use, all partials would be live
    asm volatile("" : "+v"(c[x >> 2][x & 3]));
  };
  auto mfmas = [&](f32x4 (&prev)[2][4], int qm, int qn, float sb) {
    f32x4 (&c)[2][4] = acc[qm][qn];
#pragma unroll
    for (int x = 0; x < 8; x++) {
      p[x & 3] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
          bf[qn][x >> 2], af[x & 3], f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
      if (x < 3) add(prev, x + 5);
      else add(c, x - 3);
      if (x == 2) {
#pragma unroll
        for (int i = 0; i < 4; i++) sc[i] = sa[qm][i] * sb;
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto bar = []() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  };
  issue(0, 0);
  issue(0, 2);
  issue(0, 3);
  issue(0, 1);
  if (nk > 1) {
    issue(1, 3);
    vm_wait<4>();
  } else {
    vm_wait<2>();
  }
  bar();
  if (wr == 1) {
    bar();                          // the stagger
    __builtin_amdgcn_s_setprio(1);  // the younger group wins issue arbitration
  }
  // one loop body for all K-tiles (the last issues nothing and waits for everything): code
  // beside the loop is fetched anew in every block, a microsecond and more for each K-tile's
#pragma unroll 1
  for (int t = 0; t < nk; t++) {
    const int more = __builtin_amdgcn_readfirstlane(nk - 1 - t);   // K-tiles behind this one
    const f32x2 sbt = *reinterpret_cast<const f32x2*>(lds + SC + (t & 1) * 2048 + 1024);
    read_scales(t);
    read_a(t, 0);
    read_b(t, 0);
    read_b(t, 1);
    if (more) {
      issue(t + 1, 0);
      issue(t + 1, 2);
      vm_wait<5>();
    } else {
      vm_wait<0>();
    }
    bar();
    mfmas(acc[1][1], 0, 0, sbt[0]);
    mfmas(acc[0][0], 0, 1, sbt[1]);
    bar();
    read_a(t, 1);
    if (more > 1) {
      issue(t + 1, 1);
      issue(t + 2, 3);
      vm_wait<4>();
    } else if (more) {
      issue(t + 1, 1);
      vm_wait<2>();
    }
    bar();
    mfmas(acc[0][1], 1, 0, sbt[0]);
    mfmas(acc[1][0], 1, 1, sbt[1]);
    bar();
  }
#pragma unroll
  for (int x = 5; x < 8; x++) add(acc[1][1], x);
  if (wr == 1) __builtin_amdgcn_s_setprio(0);
  else bar();   // re-align the groups
  float* cs = reinterpret_cast<float*>(lds);
  static_assert(SC + 2 * 2048 <= 160 * 1024 && 128 * 260 * 4 <= SC, "half a result tile fits");
#pragma unroll 1
  for (int qm = 0; qm < 2; qm++) {
    block_sync_lds();
#pragma unroll
    for (int qn = 0; qn < 2; qn++)
#pragma unroll
      for (int j = 0; j < 2; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          *reinterpret_cast<f32x4*>(cs + (wr * 64 + i * 16 + fr) * 260 + qn * 128 + wc * 32 +
                                    j * 16 + fc * 4) = acc[0][qn][j][i];
          acc[0][qn][j][i] = acc[1][qn][j][i];
        }
    block_sync_lds();
    store_tile<128, 256, 512, 1>(a, cs, m0 + qm * 128, n0, tid);
  }
}

// Few rows (M <= 16): the weights are streamed once from memory to registers, one 16-column tile
// a block, K-tiles dealt to the block's W waves; no LDS but for the join of the waves' sums.
// HBM / latency bound: UN K-tiles of loads are in flight per wave before the first product
// (5 x 7168 x 1792: 5.9 us, 2.2 TB/s; 16 x 8192 x 4096: 11.1 us, 3.0 TB/s).
template <int W>
__global__ __launch_bounds__(W * 64) void gemm_block_rows_kernel(GArgs a) {
  constexpr int UN = 4;
  __shared__ __attribute__((aligned(16))) float part[W][16][20];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n0 = blockIdx.x * 16, nb = min(a.N - n0, 16);
  const int fr = lane & 15, fc = lane >> 4;
  const __amdgpu_buffer_rsrc_t rB =
      rsrc(a.B + (int64_t)n0 * a.ldb, (nb - 1) * (int)a.ldb + a.K);
  const __amdgpu_buffer_rsrc_t rA = rsrc(a.A, (a.M - 1) * (int)a.lda + a.K);
  const float* sbrow = a.sb + (int64_t)(n0 / 128) * a.ld_sb;
  const uint32_t ob = fr * (uint32_t)a.ldb + fc * 16, oa = fr * (uint32_t)a.lda + fc * 16;
  f32x4 acc = {};
  for (int t0 = wid; t0 < a.groups; t0 += W * UN) {
    i32x4 b[UN][2], x[UN][2];
    float s[UN];
#pragma unroll
    for (int u = 0; u < UN; u++) {
      const int t = t0 + u * W, k = t * 128 + fc * 16;
#pragma unroll
      for (int h = 0; h < 2; h++) {   // 16 B at k and k + 64; past K lies the next row
        const bool in = t < a.groups && k + h * 64 < a.K;
        const uint32_t at = t * 128 + h * 64;
        b[u][h] = __builtin_amdgcn_raw_buffer_load_b128(rB, in ? ob + at : OOB, 0, 0);
        x[u][h] = __builtin_amdgcn_raw_buffer_load_b128(rA, in ? oa + at : OOB, 0, 0);
      }
      s[u] = t < a.groups && fr < a.M ? a.sa[(int64_t)t * a.ld_sa + fr] * sbrow[t] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < UN; u++) {
      const f32x4 p = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
          __builtin_shufflevector(b[u][0], b[u][1], 0, 1, 2, 3, 4, 5, 6, 7),
          __builtin_shufflevector(x[u][0], x[u][1], 0, 1, 2, 3, 4, 5, 6, 7),
          f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] = __builtin_fmaf(p[e], s[u], acc[e]);
    }
  }
  *reinterpret_cast<f32x4*>(&part[wid][fr][fc * 4]) = acc;
  __syncthreads();
  if (tid >= 256) return;
  const int m = tid >> 4, c = tid & 15, n = n0 + c;
  if (m >= a.M || n >= a.N) return;
  float v = 0.f;
#pragma unroll
  for (int w = 0; w < W; w++) v += part[w][m][c];   // fixed order
  if (a.bias) v += a.bias[n];
  if (a.gelu) v = gelu_erf(v);
  if (a.R) v += a.R[m * a.ldr + n];
  const int64_t at = m * a.ldc + n;
  if (a.out_type == M3S_BF16) ((bf16_t*)a.C)[at] = f2bf(v);
  else if (a.out_type == M3S_F16) ((_Float16*)a.C)[at] = (_Float16)v;
  else ((float*)a.C)[at] = v;
}

int launch_pp(GArgs a, hipStream_t s) {
  a.tiles_m = (int)m3s_div_up(a.M, 256), a.tiles_n = (int)m3s_div_up(a.N, 256);
  const int64_t blocks = (int64_t)a.tiles_m * a.tiles_n;
  if (blocks >= (1ll << 23)) return M3S_ERR_TOO_LARGE;   // 2^32 threads
  hipLaunchKernelGGL(gemm_block_pp_kernel, dim3((unsigned)blocks), dim3(512), 0, s, a);
  M3S_LAUNCH_CHECK();
  return M3S_OK;
}

template <int W>
int launch_rows(const GArgs& a, hipStream_t s) {
  if (m3s_div_up(a.N, 16) >= (1ll << 32) / (W * 64)) return M3S_ERR_TOO_LARGE;   // threads
  hipLaunchKernelGGL((gemm_block_rows_kernel<W>), dim3(m3s_div_up(a.N, 16)), dim3(W * 64), 0, s, a);
  M3S_LAUNCH_CHECK();
  return M3S_OK;
}

template <int BM, int BN, int WM, int WN, int NST, int KS>
int launch_tile(GArgs a, hipStream_t s) {
  a.tiles_m = (int)m3s_div_up(a.M, BM), a.tiles_n = (int)m3s_div_up(a.N, BN);
  const int64_t blocks = (int64_t)a.tiles_m * a.tiles_n;
  if (blocks >= (1ll << 32) / (WM * WN * KS * 64)) return M3S_ERR_TOO_LARGE;   // threads
  hipLaunchKernelGGL((gemm_block_kernel<BM, BN, WM, WN, NST, KS>), dim3((unsigned)blocks),
                     dim3(WM * WN * KS * 64), 0, s, a);
  M3S_LAUNCH_CHECK();
  return M3S_OK;
}

}  // namespace

extern "C" int m3s_vit_quant_block(const void* d_x, int x_type, int64_t ldx, void* d_q,
                                   int64_t ldq, float* d_scale, int64_t ld_scale, int64_t M,
                                   int64_t K, int pow2, void* stream) {
  if (M < 0 || K < 0 || K % 16 || (x_type != M3S_BF16 && x_type != M3S_F32 && x_type != M3S_F16))
    return M3S_ERR_INVALID_ARG;
  if (M == 0 || K == 0) return M3S_OK;
  if (!d_x || !d_q || !d_scale || (uintptr_t)d_x % 16 || (uintptr_t)d_q % 16 ||
      (uintptr_t)d_scale % 4 || ldx < K || ldq < K || ld_scale < M || ldq % 16 ||
      ldx % (x_type == M3S_F32 ? 4 : 8))
    return M3S_ERR_INVALID_ARG;
  const int64_t groups = (K + 127) / 128, tiles = (M + 15) / 16;
  if (K >= (1ll << 31) - 128 || tiles >= (1ll << 24) / groups)   // 2^32 threads
    return M3S_ERR_TOO_LARGE;
  const dim3 grid((unsigned)(tiles * groups));
  hipStream_t s = m3s_stream(stream);
#define M3S_QUANT(T)                                                                         \
  do {                                                                                       \
    if (pow2)                                                                                \
      hipLaunchKernelGGL((quant_block_kernel<T, true>), grid, dim3(256), 0, s,               \
                         (const T*)d_x, ldx, (uint8_t*)d_q, ldq, d_scale, ld_scale, M,       \
                         (int)K, (uint32_t)groups);                                          \
    else                                                                                     \
      hipLaunchKernelGGL((quant_block_kernel<T, false>), grid, dim3(256), 0, s,              \
                         (const T*)d_x, ldx, (uint8_t*)d_q, ldq, d_scale, ld_scale, M,       \
                         (int)K, (uint32_t)groups);                                          \
  } while (0)
  if (x_type == M3S_BF16) M3S_QUANT(bf16_t);
  else if (x_type == M3S_F16) M3S_QUANT(_Float16);
  else M3S_QUANT(float);
#undef M3S_QUANT
  M3S_LAUNCH_CHECK();
  return M3S_OK;
}

extern "C" int m3s_vit_gemm_block(const m3s_gemm_block_desc* desc, void* stream) {
  if (!desc) return M3S_ERR_INVALID_ARG;
  const m3s_gemm_block_desc& d = *desc;
  if (d.M < 0 || d.N < 0 || d.K <= 0 || d.K % 16) return M3S_ERR_INVALID_ARG;
  if (d.out_type != M3S_BF16 && d.out_type != M3S_F32 && d.out_type != M3S_F16)
    return M3S_ERR_INVALID_ARG;
  if (d.M == 0 || d.N == 0) return M3S_OK;
  const int groups = (int)m3s_div_up(d.K, 128), size = d.out_type == M3S_F32 ? 4 : 2;
  if (!d.A || !d.B || !d.C || !d.scale_a || !d.scale_b ||
      ((uintptr_t)d.A | (uintptr_t)d.B) % 16 || d.lda % 16 || d.ldb % 16 || d.lda < d.K ||
      d.ldb < d.K || d.ldc < d.N || (uintptr_t)d.C % size || d.ld_sa < d.M || d.ld_sb < groups ||
      ((uintptr_t)d.scale_a | (uintptr_t)d.scale_b | (uintptr_t)d.bias | (uintptr_t)d.R) % 4 ||
      (d.R && d.ldr < d.N))
    return M3S_ERR_INVALID_ARG;
  // 31-bit offsets inside a tile of 256 rows, row and column numbers past a matrix's last tile
  if (d.M > 0x7fffffff - 256 || d.N > 0x7fffffff - 256 || d.lda >= (1 << 23) ||
      d.ldb >= (1 << 23) || d.ld_sb >= (1 << 23))
    return M3S_ERR_TOO_LARGE;
  GArgs a;
  a.A = (const uint8_t*)d.A, a.B = (const uint8_t*)d.B;
  a.sa = d.scale_a, a.sb = d.scale_b, a.bias = d.bias, a.R = d.R, a.C = d.C;
  a.lda = d.lda, a.ldb = d.ldb, a.ld_sa = d.ld_sa, a.ld_sb = d.ld_sb, a.ldc = d.ldc;
  a.ldr = d.ldr, a.M = d.M, a.N = d.N, a.K = d.K, a.groups = groups;
  a.out_type = d.out_type, a.gelu = d.gelu != 0;
  a.vec = (uintptr_t)d.C % 16 == 0 && d.ldc % (16 / size) == 0 && (uintptr_t)d.bias % 16 == 0 &&
          (!d.R || ((uintptr_t)d.R % 16 == 0 && d.ldr % 4 == 0));
  hipStream_t s = m3s_stream(stream);
  // Measured (graph replays on rotating inputs): M <= 16 5 x 7168 x 1792 6.2 us against 6.6 on
  // 32-row tiles, 1 x 1024 x 4096 5.6 against 8.8 (16 x 8192 x 4096 the other way: 11.1, 10.0).  W
  // waves share the K-tiles: 4 up to 16 of them (8: 7.2 us), 8 above (1 x 1024 x 4096 5.6, 4: 7.9)
  if (d.M <= 16) return groups > 16 ? launch_rows<8>(a, s) : launch_rows<4>(a, s);
  // 256^2 tiles once they fill most of the chip: 4096^3 66 us (64 x 128 tiles 100), 224 tiles of
  // 3500 x 4096 x 2048 36 (46); with 96 of them 3000 x 2000 x 2048 takes 32 us, 21 on 64 x 128.
  // The rule counts tiles, not what they hold: close to 160 (3300 x 3100 x 2048 52 us) and on 17 to
  // 100 rows of many columns (32 x 65,536 x 4096 82 us) 64 x 128 tiles are ahead (45 and 71), on
  // 192 rows they are not (102, 88)
  if ((int64_t)m3s_div_up(d.M, 256) * m3s_div_up(d.N, 256) >= 160) return launch_pp(a, s);
  // Few tiles leave a CU one block: two K groups in it, on the smallest tiles that one round of
  // the CUs holds (768 x 1024 x 4096, 192 tiles of 64^2: 11.5 us; one group 14.3, 64 x 128 15.8;
  // 196 x 768 x 4096 on 32-row tiles 9.5, 64^2 11.1; 1536 x 1024 x 4096, 192 tiles of 64 x 128:
  // 16.8, 64^2 21.1, one group 21.8).  Enough tiles: 64 x 128, one group (768 x 4096 x 1024 9.9 us,
  // two groups 13.6; 2000 x 2048 x 2048 15.1, 19.5)
  const int64_t m64 = m3s_div_up(d.M, 64);
  const int64_t b64 = m64 * m3s_div_up(d.N, 64), b128 = m64 * m3s_div_up(d.N, 128);
  if (b64 <= 96) return launch_tile<32, 64, 1, 4, 4, 2>(a, s);
  if (b64 <= 256) return launch_tile<64, 64, 2, 2, 4, 2>(a, s);
  if (b128 <= 256) return launch_tile<64, 128, 2, 2, 3, 2>(a, s);
  return launch_tile<64, 128, 2, 2, 2, 1>(a, s);
}
