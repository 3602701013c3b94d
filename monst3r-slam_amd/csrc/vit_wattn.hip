// Attention with a sliding window and first tokens that stay visible, over a key / value
// cache (gfx950): shared key / value heads, head dim 64 or 128, bf16 or f16.
//
// Query row i of sequence b stands at position p = kv_len[b] - q_len[b] + i, in frame
// f = floor(p / F) of F tokens.  It sees the keys j of [lo, hi) and of [0, min(sinks, hi)),
//   hi = clamp((f + 1) F, 0, kv_len),   lo = window ? clamp((f - window + 1) F, 0, hi) : 0
// (F = 1: the causal window of a token stream; F = tokens per image: a frame sees itself and
// the window - 1 frames before it).  o = softmax(scale q k^T) v over them, 0 for a row that
// sees nothing.
//
// Tiles: the heads_q / heads_kv query heads of a key head are packed with the query rows
// (packed row r = i G + g), so that a wave's 32 rows share every K / V tile that they read
// whatever G is, and single-token steps fill G of them.  A block is AW row waves x KS key
// splits; each key split has two slots for 32 NH keys of K and V in LDS, filled by LDS-DMA.
// S^T = K Q^T and O^T = V^T P^T with the 32x32x16 matrix instruction (keys, then head dims, on
// the accumulator rows; queries on the lanes), so the running maximum is a lane's own and P
// stays in registers.  lo, hi and the sinks are monotone in i, so a block
// walks [sink tiles | window tiles] only, and only the tiles where some row's border falls
// are masked (a second instantiation of the tile code).  Key rows past kv_len read as zeros
// (buffer bounds); a masked score is set to -inf whatever its key holds, and a value that is
// not finite reaches only the rows that see its key (fix_values).
//
// Measured (MI355X, head dim 128 on 4 key heads / 64 on 16): one token of 4 sequences over
// 65,536 keys 106 us, 5.1 TB/s of K and V (a large copy reaches 4.93); a 768-token frame over
// 6,912 keys 44 us, matrix pipe busy 28 % and vector issue 54 % of a busy CU's cycles; 2 x 8,192
// tokens (ragged), window 2,048: 263 us, 0.84 PF/s, 50 % and 52 %, CUs busy 80 % of the time at
// 1.9 GHz (zeros: 2.2 GHz, 212 us).
#include <math.h>
#include <algorithm>
#include <type_traits>
#include "vit_common.h"

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Mat;
template <>
struct Mat<bf16_t> {
  typedef bf16x8 v8;
  static constexpr unsigned short EXPO = 0x7f80;   // exponent bits: all set = inf or NaN
  // P is rounded to T for the matrix pipe.  bf16 has f32's exponents, so p = 2^(s - max)
  // loses nothing but the 8-bit rounding.
  static constexpr float P_SHIFT = 0.f;
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(float c, bf16_t x, bf16_t y) {   // c + x + y
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(v2{x, y}, v2{(bf16_t)1.f, (bf16_t)1.f}, c, false);
  }
};
template <>
struct Mat<_Float16> {
  typedef f16x8 v8;
  static constexpr unsigned short EXPO = 0x7c00;
  // f16: p is kept 2^7 times larger (at most 2^15 under the lazy rescale), so that keys down
  // to 2^-21 of the maximum keep all 11 bits and only those below 2^-32 vanish
  static constexpr float P_SHIFT = 7.f;
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float add2(float c, _Float16 x, _Float16 y) {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(v2{x, y}, v2{(_Float16)1.f, (_Float16)1.f}, c, false);
  }
};

constexpr float kRescale = 8.0f;   // log2 headroom of p before the running maximum moves

struct WArgs {
  const void *q, *k, *v;
  void* o;
  int64_t ld_q, stride_q, ld_k, stride_k, ld_v, stride_v, ld_o, stride_o;
  const int32_t *q_len, *kv_len;
  float* part;
  int window, sinks, frame;      // clamped to the cache by the host
  int rows, cache, heads_kv, group, batch;
  int splits, nqt;
  float c_log2;                  // scale * log2(e)
};

struct Range {
  int lo, hi, sk;   // keys [lo, hi) and [0, sk) are visible
};

__device__ __forceinline__ Range visible(const WArgs& a, int ql, int kv, int i) {
  const int p = kv - ql + i;   // |p| < 2^31; a 64-bit division would cost a short call 2 us
  int f = p;
  if (a.frame != 1) {
    f = p / a.frame;
    if (f * a.frame > p) f--;
  }
  Range r;
  r.hi = (int)std::min<int64_t>(std::max<int64_t>((f + 1ll) * a.frame, 0), kv);
  r.lo = a.window ? (int)std::min<int64_t>(
                        std::max<int64_t>(((int64_t)f - a.window + 1) * a.frame, 0), r.hi)
                  : 0;
  r.sk = min(a.sinks, r.hi);
  return r;
}

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

__device__ __forceinline__ uint32_t lds_addr(const char* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

// V^T fragments of two head-dim tiles (LDS addresses a0, a1) and 32 NH keys by the
// hardware-transposed read, with the wait for them in the same block.  (As a builtin the
// compiler cannot tell that the read does not alias the DMA ring, and drains the ring with
// vmcnt(0) before it: the tile in flight would be waited for inside every tile.)
template <int RB>   // bytes of a row
__device__ __forceinline__ void read_vt(uint32_t a0, uint32_t a1, s16x4 (&v)[2][4][2]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:%18\n\t"
      "ds_read_b64_tr_b16 %2, %16 offset:%19\n\tds_read_b64_tr_b16 %3, %16 offset:%20\n\t"
      "ds_read_b64_tr_b16 %4, %16 offset:%21\n\tds_read_b64_tr_b16 %5, %16 offset:%22\n\t"
      "ds_read_b64_tr_b16 %6, %16 offset:%23\n\tds_read_b64_tr_b16 %7, %16 offset:%24\n\t"
      "ds_read_b64_tr_b16 %8, %17\n\tds_read_b64_tr_b16 %9, %17 offset:%18\n\t"
      "ds_read_b64_tr_b16 %10, %17 offset:%19\n\tds_read_b64_tr_b16 %11, %17 offset:%20\n\t"
      "ds_read_b64_tr_b16 %12, %17 offset:%21\n\tds_read_b64_tr_b16 %13, %17 offset:%22\n\t"
      "ds_read_b64_tr_b16 %14, %17 offset:%23\n\tds_read_b64_tr_b16 %15, %17 offset:%24\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0][0][0]), "=&v"(v[0][0][1]), "=&v"(v[0][1][0]), "=&v"(v[0][1][1]),
        "=&v"(v[0][2][0]), "=&v"(v[0][2][1]), "=&v"(v[0][3][0]), "=&v"(v[0][3][1]),
        "=&v"(v[1][0][0]), "=&v"(v[1][0][1]), "=&v"(v[1][1][0]), "=&v"(v[1][1][1]),
        "=&v"(v[1][2][0]), "=&v"(v[1][2][1]), "=&v"(v[1][3][0]), "=&v"(v[1][3][1])
      : "v"(a0), "v"(a1), "i"(8 * RB), "i"(16 * RB), "i"(24 * RB), "i"(32 * RB), "i"(40 * RB),
        "i"(48 * RB), "i"(56 * RB)
      : "memory");
}
template <int RB>
__device__ __forceinline__ void read_vt(uint32_t a0, uint32_t a1, s16x4 (&v)[2][2][2]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:%10\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:%11\n\tds_read_b64_tr_b16 %3, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %9\n\tds_read_b64_tr_b16 %5, %9 offset:%10\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:%11\n\tds_read_b64_tr_b16 %7, %9 offset:%12\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0][0][0]), "=&v"(v[0][0][1]), "=&v"(v[0][1][0]), "=&v"(v[0][1][1]),
        "=&v"(v[1][0][0]), "=&v"(v[1][0][1]), "=&v"(v[1][1][0]), "=&v"(v[1][1][1])
      : "v"(a0), "v"(a1), "i"(8 * RB), "i"(16 * RB), "i"(24 * RB)
      : "memory");
}

// 16-B chunk swizzles of an LDS tile row (D * 2 bytes) against bank conflicts.  64 banks x 4 B
// are 256 B: two rows of D = 64, one of D = 128.  K is read by 16 lanes down 16 rows at one
// chunk, V by half waves as 4 rows x 64 B.
template <int D>
__device__ __forceinline__ int k_swz(int r) {
  return D == 64 ? (r >> 1) & 7 : r & 15;
}
template <int D>
__device__ __forceinline__ int v_swz(int r) {
  return D == 64 ? ((r >> 1) & 1) * 4 : (r & 3) * 4;
}

// WPS: waves per SIMD that the registers have to leave room for
template <typename T, int D, int AW, int KS, int NH, int WPS>
__global__ __launch_bounds__(AW* KS * 64, WPS) void wattn_kernel(WArgs a) {
  typedef typename Mat<T>::v8 v8;
  constexpr int KT = 32 * NH;              // keys per tile
  constexpr int DT = D / 32;               // head-dim tiles of 32
  constexpr int DS = D / 16;               // 16-deep steps over the head dim
  constexpr int CPR = D / 8;               // 16-B chunks per row
  constexpr int GT = AW * 64;              // threads of a key split
  constexpr int TILE = KT * D * 2;         // bytes of a K or V tile
  constexpr int RING = 4 * TILE;           // two slots of K, two of V, for each key split
  constexpr int ACH = TILE / 16 / GT;      // DMA instructions per wave, operand and tile
  constexpr bool OWN = AW == 1;            // a key split's rings are its one wave's own
  constexpr int RED = DT * 16 * 64 + 128;  // floats of a wave's partial: O^T, m, l
  static_assert(TILE % (16 * GT) == 0, "whole DMA instructions");
  static_assert((KS - 1) * AW * RED * 4 <= KS * RING, "partials fit in the rings");
  static_assert(KS * RING <= 160 * 1024, "LDS");
  __shared__ __attribute__((aligned(16))) char lds[KS * RING];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wall = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wid = wall % AW, ksp = wall / AW;
  const int gtid = tid - ksp * GT;
  char* const ring = lds + ksp * RING;
  const int r = lane & 31, hh = lane >> 5;
  // 1-D grid (row tile fastest, then key head, then batch x split), remapped so that an XCD's
  // blocks are neighbours: the row tiles of a key head find its K / V in one L2
  const int total = gridDim.x, orig = blockIdx.x;
  int lin = orig;
  if (total >= 16) {
    const int qq = total / 8, rr = total % 8, xcd = orig % 8;
    lin = (xcd < rr ? xcd * (qq + 1) : rr * (qq + 1) + (xcd - rr) * qq) + orig / 8;
  }
  const int qt = a.nqt - 1 - lin % a.nqt;   // the last rows see the most keys: first
  const int hz = lin / a.nqt;
  const int hk = hz % a.heads_kv;
  const int bz = hz / a.heads_kv;
  const int b = bz / a.splits, sp = bz - b * a.splits;

  const int kv = a.kv_len ? min(max(a.kv_len[b], 0), a.cache) : a.cache;
  const int ql = a.q_len ? min(max(a.q_len[b], 0), a.rows) : a.rows;
  const int G = a.group;
  const int R = ql * G;                     // packed rows of this sequence (host: < 2^31)
  const int rb0 = qt * (AW * 32);
  if (rb0 >= R) return;
  const int rb1 = min(rb0 + AW * 32, R) - 1;
  // the block's tiles: x < nsink sink tiles, then the window's
  const Range first = visible(a, ql, kv, rb0 / G), last = visible(a, ql, kv, rb1 / G);
  const int wlo = first.lo / KT, whi = (last.hi + KT - 1) / KT;
  const int nsink = min((last.sk + KT - 1) / KT, wlo);
  const int ntile = nsink + max(whi - wlo, 0);
  const int per = ntile / a.splits, rest = ntile - per * a.splits;
  const int x0 = sp * per + min(sp, rest), n = per + (sp < rest ? 1 : 0);
  // tiles [xa, xb) need no mask: behind every row's lo, before every row's hi
  const int xa = nsink + (last.lo + KT - 1) / KT - wlo;
  const int xb = nsink + first.hi / KT - wlo;
  const int nj = (n + KS - 1) / KS;                      // uniform trip count
  const int nme = n > ksp ? (n - ksp + KS - 1) / KS : 0;   // tiles of this key split
  const int ja = min(max(xa - x0 + KS - 1, 0) / KS, nj);
  const int jb = min(max(max(xb - x0, 0) / KS, ja), nj);

  // this wave's rows
  const int rw0 = rb0 + wid * 32;
  const int row = min(rw0 + r, R - 1), i = row / G, g = row - i * G;
  const Range mine = visible(a, ql, kv, i);
  const T* Q = (const T*)a.q + b * a.stride_q + (int64_t)i * a.ld_q + (hk * G + g) * D;
  v8 qf[DS];
#pragma unroll
  for (int ks = 0; ks < DS; ks++) qf[ks] = *reinterpret_cast<const v8*>(Q + ks * 16 + 8 * hh);
  if constexpr (!OWN) {   // wait before the DMA queue fills
#pragma unroll
    for (int ks = 0; ks < DS; ks++) asm volatile("" : "+v"(qf[ks]));
  }

  const char* const Kb = (const char*)((const T*)a.k + b * a.stride_k + hk * D);
  const char* const Vb = (const char*)((const T*)a.v + b * a.stride_v + hk * D);
  uint32_t k_off[ACH], v_off[ACH];
#pragma unroll
  for (int c = 0; c < ACH; c++) {
    const int q = c * GT + gtid, rr = q / CPR, slot = q % CPR;
    k_off[c] = (uint32_t)(rr * (int)a.ld_k + (slot ^ k_swz<D>(rr)) * 8) * 2u;
    v_off[c] = (uint32_t)(rr * (int)a.ld_v + (slot ^ v_swz<D>(rr)) * 8) * 2u;
  }
  auto tile_of = [&](int j) {
    const int x = x0 + ksp + KS * j;
    return x + (x < nsink ? 0 : wlo - nsink);
  };
  // K and V rows of tile j (if the group has one) into its slots; a descriptor's base is the
  // tile's first row, so offsets stay small in a cache of any length, and its size ends behind
  // row kv_len - 1
  const int64_t k_tile = a.ld_k * (KT * 2), v_tile = a.ld_v * (KT * 2);   // bytes
  auto k_slot = [&](int j) { return ring + (j & 1) * (2 * TILE); };
  auto v_slot = [&](int j) { return ring + (j & 1) * (2 * TILE) + TILE; };
  auto issue = [&](int j) __attribute__((always_inline)) {
    if (!OWN && j >= nme) return;
    const int t = tile_of(j);
    const int left = min(kv - t * KT, KT) - 1;   // >= 0: the tile holds a visible key
    // OWN: no branch, so that waits can count the instructions behind a tile; a tile that is
    // not there has no bytes
    const bool there = !OWN || j < nme;
    const __amdgpu_buffer_rsrc_t rK = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(Kb) + t * k_tile, (short)0,
        there ? left * (int)a.ld_k * 2 + D * 2 : 0, 0x00020000);
    const __amdgpu_buffer_rsrc_t rV = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(Vb) + t * v_tile, (short)0,
        there ? left * (int)a.ld_v * 2 + D * 2 : 0, 0x00020000);
    char* const sb = k_slot(j) + wid * 64 * 16;
#pragma unroll
    for (int c = 0; c < ACH; c++) {
      glds16(rK, sb + c * GT * 16, k_off[c]);
      glds16(rV, sb + TILE + c * GT * 16, v_off[c]);
    }
  };

  f32x16 oacc[DT];
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int e = 0; e < 16; e++) oacc[d][e] = 0.f;
  float m = -INFINITY, lsum[2] = {0.f, 0.f};   // Σ p over this lane's half of the keys
  // fragment offsets in a stage: K row r (+ 32 hs), chunk 2 ks + hh; V^T: head dims 32 d +
  // 16 gsel + 4 gp .. + 3 of key rows 16 c + 8 x + 4 hh + gq
  const int gi = lane & 15, gq = gi >> 2, gp = gi & 3, gsel = (lane >> 4) & 1;
  // (the swizzles are XORs of the chunk: steps along a row are XORs of the first's offset)
  const uint32_t kf_off = r * (D * 2) + ((hh ^ k_swz<D>(r)) * 16);
  const int vd = 16 * gsel + 4 * gp, vr = 4 * hh + gq;
  const uint32_t vt_off = vr * (D * 2) + (((vd >> 3) ^ v_swz<D>(vr)) * 16) + (vd & 7) * 2;

  // p = 2^(s - max) of masked scores, rounded to T as P^T's operand (16 keys each), and Σ p of
  // the rounded values (their errors cancel against P V's)
  auto exps = [&](f32x16 (&s)[NH], v8 (&pf)[2 * NH]) __attribute__((always_inline)) {
    const float mc = (m == -INFINITY ? 0.f : m * a.c_log2) - Mat<T>::P_SHIFT;
#pragma unroll
    for (int c = 0; c < 2 * NH; c++)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
#pragma unroll
        for (int z = e; z < e + 2; z++)
          pf[c][z] = (T)__builtin_amdgcn_exp2f(
              __builtin_fmaf(s[c >> 1][(c & 1) * 8 + z], a.c_log2, -mc));
        lsum[c & 1] = Mat<T>::add2(lsum[c & 1], pf[c][e], pf[c][e + 1]);
      }
  };
  // masks the scores of tile j
  auto mask = [&](int j, f32x16 (&s)[NH]) __attribute__((always_inline)) {
    const int k0 = tile_of(j) * KT + 4 * hh;
    const int lo = mine.lo - k0, sk = mine.sk - k0;
    const unsigned width = mine.hi - mine.lo;
#pragma unroll
    for (int hs = 0; hs < NH; hs++)
#pragma unroll
      for (int e = 0; e < 16; e++) {
        const int key = hs * 32 + (e & 3) + 8 * (e >> 2);
        const bool see = (unsigned)(key - lo) < width || key < sk;
        s[hs][e] = see ? s[hs][e] : -INFINITY;
      }
  };
  // the running maximum moves only when a tile exceeds it by more than 2^kRescale in p
  // (wave-uniform: after the first tiles the rescale is skipped)
  auto rescale = [&](float t) __attribute__((always_inline)) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t),
                                                       false, false);
    t = fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));   // the row's two lanes
    if (__builtin_amdgcn_ballot_w64((t - m) * a.c_log2 > kRescale)) {
      const float m_new = fmaxf(m, t);
      // a row that has seen nothing keeps -inf: 2^-inf = 0, never inf - inf
      const float alpha =
          __builtin_amdgcn_exp2f((m - (m_new == -INFINITY ? 0.f : m_new)) * a.c_log2);
      m = m_new;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) oacc[d][e] *= alpha;
      lsum[0] *= alpha;
      lsum[1] *= alpha;
    }
  };
  // 0 x inf in the matrix pipe would reach the rows that do not see the key: values that are not
  // finite are taken out of it and added to the rows that do
  auto fix_values = [&](int j, int d2, s16x4 (&vt)[2][2 * NH][2]) __attribute__((always_inline)) {
    u16x4 top = {0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < 2; d++)
#pragma unroll
      for (int c = 0; c < 2 * NH; c++)
#pragma unroll
        for (int x = 0; x < 2; x++)
          top = __builtin_elementwise_max(
              top, __builtin_bit_cast(u16x4, vt[d][c][x]) & (unsigned short)Mat<T>::EXPO);
    const bool bad = max(max(top[0], top[1]), max(top[2], top[3])) == Mat<T>::EXPO;
    if (__builtin_amdgcn_ballot_w64(bad) == 0) return;
    const int key0 = tile_of(j) * KT;
    const char* sV = v_slot(j);
#pragma unroll
    for (int d = 0; d < 2; d++)
#pragma unroll
      for (int c = 0; c < 2 * NH; c++)
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (((unsigned short)vt[d][c][x][e] & Mat<T>::EXPO) == Mat<T>::EXPO)
              vt[d][c][x][e] = 0;
#pragma unroll 1
    for (int kk = 0; kk < KT; kk++) {
      const int key = key0 + kk;
      const bool see = (key >= mine.lo && key < mine.hi) || key < mine.sk;
#pragma unroll
      for (int d = 0; d < 2; d++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
          const int dim = (d2 + d) * 32 + (e & 3) + 8 * (e >> 2) + 4 * hh;
          const T val = *reinterpret_cast<const T*>(
              sV + kk * (D * 2) + (((dim >> 3) ^ v_swz<D>(kk)) * 16) + (dim & 7) * 2);
          const unsigned short bits = __builtin_bit_cast(unsigned short, val);
          if (see && (bits & Mat<T>::EXPO) == Mat<T>::EXPO) oacc[d2 + d][e] += (float)val;
        }
    }
  };

  // A trip of AW > 1 row waves waits for its tile, lets every wave finish the one before, issues
  // the next one over that, and works alone (one row wave needs no barrier, and has two tiles on
  // their way from the start: what a short call waits for most): matrix and vector instructions
  // overlap across the waves of a SIMD (other blocks, at other places of their tiles).  Dealing
  // K Q^T of the next tile out between the exponentials of this one, or 64 rows a wave, changed
  // nothing (random inputs hold the clock at 1.9 GHz; the same call on zeros has 2.2 and takes 4/5
  // of the time).
  const Range wfirst = visible(a, ql, kv, min(rw0, R - 1) / G);
  const Range wlast = visible(a, ql, kv, min(rw0 + 31, R - 1) / G);
  auto work = [&](int j, auto mask_tag) __attribute__((always_inline)) {
    constexpr bool MASK = decltype(mask_tag)::value;
    if constexpr (MASK) {
      const int k0 = tile_of(j) * KT;   // the group has a tile j and some row of the wave sees it
      if (j >= nme || ((k0 >= wlast.hi || k0 + KT <= wfirst.lo) && k0 >= wlast.sk)) return;
    }
    f32x16 s[NH];
    const char* sK = k_slot(j);
#pragma unroll
    for (int ks = 0; ks < DS; ks++)
#pragma unroll
      for (int hs = 0; hs < NH; hs++) {
        if (ks == 0) {
#pragma unroll
          for (int e = 0; e < 16; e++) s[hs][e] = 0.f;
        }
        const v8 kf = *reinterpret_cast<const v8*>(sK + (kf_off ^ (ks * 32)) + hs * 32 * (D * 2));
        s[hs] = Mat<T>::mma(kf, qf[ks], s[hs]);
      }
    if constexpr (MASK) mask(j, s);
    float t = -INFINITY;
#pragma unroll
    for (int hs = 0; hs < NH; hs++)
#pragma unroll
      for (int e = 0; e < 16; e++) t = fmaxf(t, s[hs][e]);
    rescale(t);
    v8 pf[2 * NH];
    exps(s, pf);
    const uint32_t sbase = lds_addr(v_slot(j));
#pragma unroll
    for (int d2 = 0; d2 < DT; d2 += 2) {   // O^T += V^T P^T, two head-dim tiles at a time
      s16x4 vt[2][2 * NH][2];
      read_vt<D * 2>(sbase + (vt_off ^ (d2 * 64)), sbase + (vt_off ^ (d2 * 64 + 64)), vt);
      if constexpr (MASK) fix_values(j, d2, vt);
#pragma unroll
      for (int c = 0; c < 2 * NH; c++)
#pragma unroll
        for (int d = 0; d < 2; d++) {
          typedef short s16x8 __attribute__((ext_vector_type(8)));
          const s16x8 vf =
              __builtin_shufflevector(vt[d][c][0], vt[d][c][1], 0, 1, 2, 3, 4, 5, 6, 7);
          oacc[d2 + d] = Mat<T>::mma(__builtin_bit_cast(v8, vf), pf[c], oacc[d2 + d]);
        }
    }
  };
  auto trip = [&](int j, auto mask_tag) __attribute__((always_inline)) {
    if constexpr (OWN) {
      vm_wait<2 * ACH>();   // tile j has landed, j + 1 is on its way
      work(j, mask_tag);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      issue(j + 2);
    } else {
      vm_wait<0>();
      block_sync_lds();
      issue(j + 1);
      work(j, mask_tag);
    }
  };
  issue(0);
  if constexpr (OWN) {
    issue(1);
#pragma unroll
    for (int ks = 0; ks < DS; ks++) asm volatile("" : "+v"(qf[ks]));
  }
#pragma unroll 1
  for (int j = 0; j < ja; j++) trip(j, std::true_type{});
  const int je = max(ja, min(jb, n / KS));   // full tiles that every key group has
#pragma unroll 1
  for (int j = ja; j < je; j++) trip(j, std::false_type{});
#pragma unroll 1
  for (int j = je; j < nj; j++) trip(j, std::true_type{});

  float l = lsum[0] + lsum[1];
  l += __shfl_xor(l, 32, 64);
  if constexpr (KS > 1) {
    vm_wait<0>();
    block_sync_lds();   // ring reads done, no DMA in flight
    float* red = reinterpret_cast<float*>(lds);
    if (ksp > 0) {
      float* P = red + ((ksp - 1) * AW + wid) * RED;
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          reinterpret_cast<float4*>(P)[(d * 4 + e) * 64 + lane] =
              make_float4(oacc[d][4 * e], oacc[d][4 * e + 1], oacc[d][4 * e + 2],
                          oacc[d][4 * e + 3]);
      reinterpret_cast<float2*>(P + DT * 16 * 64)[lane] = make_float2(m, l);
    }
    block_sync_lds();
    if (ksp > 0) return;
#pragma unroll
    for (int s2 = 1; s2 < KS; s2++) {
      const float* P = red + ((s2 - 1) * AW + wid) * RED;
      const float2 ml = reinterpret_cast<const float2*>(P + DT * 16 * 64)[lane];
      const float M = fmaxf(m, ml.x);
      const float a0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - M) * a.c_log2);
      const float a1 = ml.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((ml.x - M) * a.c_log2);
      // a split without visible keys (m = -inf) has O = 0 unless its keys made NaN: kept
#pragma unroll
      for (int d = 0; d < DT; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float4 w = reinterpret_cast<const float4*>(P)[(d * 4 + e) * 64 + lane];
          oacc[d][4 * e] = oacc[d][4 * e] * a0 + w.x * a1;
          oacc[d][4 * e + 1] = oacc[d][4 * e + 1] * a0 + w.y * a1;
          oacc[d][4 * e + 2] = oacc[d][4 * e + 2] * a0 + w.z * a1;
          oacc[d][4 * e + 3] = oacc[d][4 * e + 3] * a0 + w.w * a1;
        }
      l = l * a0 + ml.y * a1;
      m = M;
    }
  }
  if (rw0 + r >= R) return;
  if (a.part) {   // grid splits: unnormalised O, m, l → [split][b][hk][packed row][D + 4] f32
    const int64_t rows = (int64_t)a.rows * G;
    float* P = a.part + ((((int64_t)sp * a.batch + b) * a.heads_kv + hk) * rows + row) * (D + 4);
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        *reinterpret_cast<float4*>(P + d * 32 + 8 * e + 4 * hh) =
            make_float4(oacc[d][4 * e], oacc[d][4 * e + 1], oacc[d][4 * e + 2], oacc[d][4 * e + 3]);
    if (hh == 0) *reinterpret_cast<float2*>(P + D) = make_float2(m, l);
    return;
  }
  const float inv_l = l == 0.f ? 0.f : 1.0f / l;
  T* O = (T*)a.o + b * a.stride_o + (int64_t)i * a.ld_o + (hk * G + g) * D;
#pragma unroll
  for (int d = 0; d < DT; d++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      T w[4];
#pragma unroll
      for (int x = 0; x < 4; x++) w[x] = (T)(oacc[d][4 * e + x] * inv_l);
      uint2 raw;
      __builtin_memcpy(&raw, w, 8);
      *reinterpret_cast<uint2*>(O + d * 32 + 8 * e + 4 * hh) = raw;
    }
}

// Join of the grid splits: M = max m_s, o = Σ O_s 2^((m_s - M) c) / Σ l_s 2^((m_s - M) c).
// A wave per (b, hk, packed row): 64 / (D / 8) lanes share the splits of 8 head dims, each with a
// running maximum of its own, and join by shuffles (fixed order).  One lane for all splits was
// latency bound: 25 us for 32 splits, a quarter of the 64k-key decode step that made them.
template <typename T, int D>
__global__ __launch_bounds__(256) void wattn_join_kernel(WArgs a) {
  constexpr int CH = D / 8, SL = 64 / CH, UN = 4;
  const uint32_t rows = a.rows * a.group, all = rows * a.heads_kv * a.batch;   // few: plan_of
  const uint32_t at = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= all) return;
  const int lane = threadIdx.x & 63, d8 = lane % CH * 8, sl = lane / CH;
  const int row = (int)(at % rows);
  const uint32_t bh = at / rows;
  const int hk = (int)(bh % a.heads_kv);
  const int64_t b = bh / a.heads_kv;
  const int i = row / a.group, g = row - i * a.group;
  if (a.q_len && i >= a.q_len[b]) return;
  const float* P0 = a.part + (int64_t)at * (D + 4);
  const int64_t step = (int64_t)all * (D + 4);
  float M = -INFINITY, L = 0.f, acc[8] = {};
  auto weight = [&](float m) { return m == -INFINITY ? 0.f : exp2f((m - M) * a.c_log2); };
  for (int s0 = sl; s0 < a.splits; s0 += SL * UN) {
    float m[UN], l[UN], v[UN][8];
#pragma unroll
    for (int u = 0; u < UN; u++) {
      const int s = s0 + u * SL;
      const float* P = P0 + min(s, a.splits - 1) * step;
      m[u] = s < a.splits ? P[D] : -INFINITY;
      l[u] = P[D + 1];
#pragma unroll
      for (int e = 0; e < 8; e++) v[u][e] = P[d8 + e];
    }
    float top = M;
#pragma unroll
    for (int u = 0; u < UN; u++) top = fmaxf(top, m[u]);
    const float old = M;
    M = top;
    const float w0 = weight(old);
    L *= w0;
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] *= w0;
#pragma unroll
    for (int u = 0; u < UN; u++) {
      if (s0 + u * SL >= a.splits) break;
      const float w = weight(m[u]);
      L += l[u] * w;
#pragma unroll
      for (int e = 0; e < 8; e++) acc[e] += v[u][e] * w;
    }
  }
#pragma unroll
  for (int o = CH; o < 64; o <<= 1) {
    const float m1 = __shfl_xor(M, o, 64), l1 = __shfl_xor(L, o, 64);
    const float m0 = M;
    M = fmaxf(m0, m1);
    const float w0 = weight(m0), w1 = weight(m1);
    L = L * w0 + l1 * w1;
#pragma unroll
    for (int e = 0; e < 8; e++) acc[e] = acc[e] * w0 + __shfl_xor(acc[e], o, 64) * w1;
  }
  if (sl) return;
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  T* O = (T*)a.o + b * a.stride_o + (int64_t)i * a.ld_o + (hk * a.group + g) * D + d8;
  T w[8];
#pragma unroll
  for (int e = 0; e < 8; e++) w[e] = (T)(acc[e] * inv);
#pragma unroll
  for (int x = 0; x < 2; x++) {
    uint2 raw;
    __builtin_memcpy(&raw, w + 4 * x, 8);
    reinterpret_cast<uint2*>(O)[x] = raw;
  }
}

// Launch shape from the sizes alone: row waves and key splits of a block, grid splits.
struct Plan {
  int aw, ks, splits, nqt;
  int64_t blocks, bytes;
};

Plan plan_of(const m3s_window_attention_desc& d) {
  const int64_t G = d.heads_q / d.heads_kv, R = (int64_t)d.rows * G;
  const int64_t hb = (int64_t)d.heads_kv * d.batch, b4 = (R + 127) / 128 * hb;
  const bool d64 = d.head_dim == 64;
  Plan p;
  // Up to 256 tiles of 32 rows, or one a key head (single tokens): a block each, 4 key splits
  // (16 sequences x 40 tokens over 4,000 keys, 8 heads of 128: 60-67 us, 4 x 2 waves 67; 512
  // tokens over 4,096 keys, 12 heads of 64 on 4: 21.5 us, 2 x 6 waves 24.3).  Up to 256 blocks of
  // 128 rows: many waves on few rows, 2 x 6 for D = 64 (a 768-token frame over 6,912 keys of 16
  // heads 43 us; 1 x 4 59, 4 x 1 94), 4 x 2 for D = 128 (12 heads 55 us; 1 x 4 92, 4 x 1 159).
  // Above, 4 row waves and several blocks a CU (8,192 tokens, 16 heads, window 2,048, D = 128:
  // 152 us, 4 x 2 167; D = 64: 91, 2 x 6 140; two such sequences of 128 267, 4 x 2 312).
  if ((R + 31) / 32 * hb <= 256 || R <= 32) p.aw = 1, p.ks = 4;
  else if (b4 <= 256) p.aw = d64 ? 2 : 4, p.ks = d64 ? 6 : 2;
  else p.aw = 4, p.ks = 1;
  const int kt = (d64 && p.aw != 2) || p.ks == 2 ? 64 : 32;
  p.nqt = (int)((R + p.aw * 32 - 1) / (p.aw * 32));
  // keys that a block may walk: the window (+ the span of its rows) and the sinks
  int64_t keys = d.cache_rows;
  if (d.window > 0 && d.window < d.cache_rows && d.frame < d.cache_rows) {
    const int64_t span = std::min<int64_t>(d.rows, p.aw * 32 / G + 2);
    keys = std::min<int64_t>(keys, (d.window + 1) * d.frame + span +
                                       std::min<int64_t>(d.sinks, d.cache_rows));
  }
  // blocks with key splits fill a CU: grid splits up to one block a CU, of four tiles a wave at
  // least (8 sequences x 1 token, window 4,096: 8 splits 16.3 us, 4 18.7, 16 17.3, 32 22.6; one to
  // two blocks a CU are not split: 40 sequences over 4,096 keys of 8 heads 156 us, with 2 splits
  // 143, but 20 of them 68, with 2 splits 81)
  const int64_t tiles = (keys + kt - 1) / kt, blocks = p.nqt * hb;
  int64_t splits = 1;
  if (p.ks > 1 && blocks <= 128)
    splits = std::min<int64_t>(256 / std::max<int64_t>(blocks, 1), tiles / (4 * p.ks));
  p.splits = (int)std::max<int64_t>(1, splits);
  p.blocks = blocks * p.splits;
  p.bytes = p.splits > 1 ? p.splits * hb * R * (d.head_dim + 4) * 4 : 0;
  return p;
}

bool shape_ok(const m3s_window_attention_desc& d) {
  if (d.batch < 0 || d.rows < 0 || d.cache_rows < 0 || d.heads_q <= 0 || d.heads_kv <= 0)
    return false;
  if (d.heads_q % d.heads_kv || (d.head_dim != 64 && d.head_dim != 128)) return false;
  if (d.dtype != M3S_BF16 && d.dtype != M3S_F16) return false;
  return d.window >= 0 && d.sinks >= 0 && d.frame >= 1;
}

// 32-bit packed rows, key positions (a tile past the last one too), head columns and
// tile-relative byte offsets (64 rows)
bool too_large(const m3s_window_attention_desc& d) {
  return (int64_t)d.rows * (d.heads_q / d.heads_kv) >= (1ll << 30) || d.heads_q > 65535 ||
         d.cache_rows > 0x7fffffff - 256 || (int64_t)d.heads_kv * d.batch >= (1ll << 31) ||
         d.ld_k >= (1 << 23) || d.ld_v >= (1 << 23);
}

template <typename T, int D, int AW, int KS, int NH, int WPS>
void launch(const WArgs& a, int64_t blocks, hipStream_t s) {
  hipLaunchKernelGGL((wattn_kernel<T, D, AW, KS, NH, WPS>), dim3((unsigned)blocks),
                     dim3(AW * KS * 64), 0, s, a);
}

template <typename T, int D>
void launch_all(const WArgs& a, const Plan& p, hipStream_t s) {
  constexpr bool d64 = D == 64;
  if (p.aw == 1) launch<T, D, 1, 4, d64 ? 2 : 1, 1>(a, p.blocks, s);
  else if (p.ks == 1) launch<T, D, 4, 1, d64 ? 2 : 1, 3>(a, p.blocks, s);
  else if constexpr (d64) launch<T, D, 2, 6, 1, 3>(a, p.blocks, s);
  else launch<T, D, 4, 2, 2, 2>(a, p.blocks, s);
  if (a.part) {
    const int64_t rows = (int64_t)a.rows * a.group * a.heads_kv * a.batch;
    hipLaunchKernelGGL((wattn_join_kernel<T, D>), dim3(m3s_div_up(rows, 4)), dim3(256), 0, s, a);
  }
}

}  // namespace

extern "C" size_t m3s_vit_window_attention_workspace_bytes(const m3s_window_attention_desc* desc) {
  if (!desc || !shape_ok(*desc) || too_large(*desc) || !desc->batch || !desc->rows) return 0;
  return (size_t)plan_of(*desc).bytes;
}

extern "C" int m3s_vit_window_attention(const m3s_window_attention_desc* desc, void* stream) {
  if (!desc) return M3S_ERR_INVALID_ARG;
  const m3s_window_attention_desc& d = *desc;
  if (!shape_ok(d)) return M3S_ERR_INVALID_ARG;
  if (!(d.scale >= 1.17549435e-38f) || !isfinite(d.scale * 1.4426950408889634f))
    return M3S_ERR_INVALID_ARG;
  if (d.batch == 0 || d.rows == 0) return M3S_OK;
  const int64_t wq = (int64_t)d.heads_q * d.head_dim, wk = (int64_t)d.heads_kv * d.head_dim;
  if (!d.q || !d.o || (uintptr_t)d.q % 16 || d.ld_q % 8 || d.stride_q % 8 || d.ld_q < wq ||
      (uintptr_t)d.o % 8 || d.ld_o % 4 || d.stride_o % 4 || d.ld_o < wq)
    return M3S_ERR_INVALID_ARG;
  if (d.cache_rows &&
      (!d.k || !d.v || ((uintptr_t)d.k | (uintptr_t)d.v) % 16 || d.ld_k % 8 || d.ld_v % 8 ||
       d.stride_k % 8 || d.stride_v % 8 || d.ld_k < wk || d.ld_v < wk))
    return M3S_ERR_INVALID_ARG;
  if (too_large(d)) return M3S_ERR_TOO_LARGE;
  Plan p = plan_of(d);
  if (p.splits > 1 && (!d.workspace || d.workspace_bytes < p.bytes || (uintptr_t)d.workspace % 16))
    p.blocks /= p.splits, p.splits = 1, p.bytes = 0;
  if (p.blocks >= (1ll << 32) / (p.aw * p.ks * 64)) return M3S_ERR_TOO_LARGE;   // threads
  WArgs a;
  a.q = d.q, a.k = d.k, a.v = d.v, a.o = d.o;
  a.ld_q = d.ld_q, a.stride_q = d.stride_q, a.ld_k = d.ld_k, a.stride_k = d.stride_k;
  a.ld_v = d.ld_v, a.stride_v = d.stride_v, a.ld_o = d.ld_o, a.stride_o = d.stride_o;
  a.q_len = d.q_len, a.kv_len = d.kv_len;
  // a window, sinks or frame longer than every position act as if there were no such limit
  const int64_t most = (int64_t)d.cache_rows + d.rows + 1;
  a.window = d.window > d.cache_rows ? 0 : (int)d.window;
  a.sinks = (int)std::min<int64_t>(d.sinks, d.cache_rows);
  a.frame = (int)std::min<int64_t>(std::min<int64_t>(d.frame, most), 0x7fffffff);
  a.rows = d.rows, a.cache = d.cache_rows, a.heads_kv = d.heads_kv;
  a.group = d.heads_q / d.heads_kv, a.batch = d.batch;
  a.splits = p.splits, a.nqt = p.nqt;
  a.c_log2 = d.scale * 1.4426950408889634f;
  a.part = p.splits > 1 ? (float*)d.workspace : nullptr;
  hipStream_t s = m3s_stream(stream);
  if (d.dtype == M3S_BF16) {
    if (d.head_dim == 64) launch_all<bf16_t, 64>(a, p, s);
    else launch_all<bf16_t, 128>(a, p, s);
  } else {
    if (d.head_dim == 64) launch_all<_Float16, 64>(a, p, s);
    else launch_all<_Float16, 128>(a, p, s);
  }
  M3S_LAUNCH_CHECK();
  return M3S_OK;
}
