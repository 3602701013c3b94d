// Norm of queries and keys per head and the position rotation in one pass (gfx950), with the
// new keys and values written where a cache wants them.
//
//   head x[0..D):  rms    y = x / sqrt(mean x^2 + eps) * gamma (+ beta)
//                  layer  y = (x - mean) / sqrt(mean (x - mean)^2 + eps) * gamma (+ beta)
//   then axis a of A (W = D / A values of the head, one position each) turns its pairs
//   (i, i + W/2) by t = pos[a] base^(-2i/W):  (u, w) -> (u cos t - w sin t, w cos t + u sin t).
//
// One read and one write of every element: HBM bound.  A lane owns 8 elements and their 8
// pair partners (two 16-B loads), so the rotation needs no exchange and the norm's sums take
// log2(D/16) shuffles; 4 (D = 64) or 8 (D = 128) lanes make a head.  A wave takes a token: its
// loads of up to 4 x 16 (D = 64) or 4 x 8 heads are under way before it works out the token's
// D/2 angles, one a lane, which all heads then share through LDS (computed per lane they would
// cost about 17 VALU operations an element, as many as the card issues in the time that the
// element's 4 bytes take).  Heads dealt out one after the other, each load behind the angles of
// its block, took 156 us where this takes 73 us (32,768 tokens of 20 heads of 128 and 4 value
// heads, f16: 5.5 TB/s, part of it in the last cache; a large copy reaches 4.93).  One token a
// wave: four that share a block's factors took 81 us.
// Angles: revolutions in f64 (pos times the host's table of base^(-2i/W) / 2 pi), reduced to
// [-1/2, 1/2] there and only then rounded to f32: an f32 angle of position 100,000 is off by
// up to 2^-8 radians.  The table holds an f64 and what it leaves of the extended-precision value:
// the f64 alone is off by 2^-24 of a half turn at positions of 2^30 and by 2^-15.5 at 2^40, the
// pair by 2^-24 up to 2^38 and 2^-23.7 at 2^40 (base 100 to 500,000, against 113 bits).
#include <math.h>
#include <type_traits>
#include "vit_common.h"

namespace {

struct RevTable {
  double rev[64];   // revolutions per position step of pair i of an axis
  float low[64];    // the value itself less rev
};

struct NormArgs {
  m3s_qk_norm_rope_desc d;
  uint32_t tokens;
};

template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

template <typename T, int D>
__global__ __launch_bounds__(256, 3) void qk_norm_rope_kernel(NormArgs a, RevTable rt) {
  constexpr int LPH = D / 16;       // lanes per head
  constexpr int HP = 64 / LPH;      // heads per pass of a wave
  constexpr int UN = 4;             // passes whose loads are in flight together
  __shared__ __attribute__((aligned(16))) float cs[4][2][D / 2];    // per wave: cos, sin
  __shared__ __attribute__((aligned(16))) float affine[2][2][D];    // gamma, beta of q, k
  const m3s_qk_norm_rope_desc& d = a.d;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int half = D / 2 / d.axes;
  const int grp = lane / LPH, l = lane % LPH;
  const int ax = l / (half / 8);
  const int lo = ax * 2 * half + (l - ax * (half / 8)) * 8;   // first element of the lane
  const int heads = d.heads_q + d.heads_kv * (d.v ? 2 : 1);
  float (&tab)[2][D / 2] = cs[wave];

  vec8<T> xu[UN], xw[UN];
  T* dst[UN];        // null: nothing to write
  // starts the loads of the heads h0 .. h0 + UN HP - 1 of row s
  auto load = [&](int64_t b, int64_t s, int64_t row, bool room, int h0) {
    const T* qs = (const T*)d.q + b * d.stride_q + s * d.ld_q;
    const T* ks = (const T*)d.k + b * d.stride_k + s * d.ld_k;
    const T* vs = (const T*)d.v + b * d.stride_v + s * d.ld_v;
    T* qd = (T*)d.q_out + b * d.stride_qo + s * d.ld_qo;
    T* kd = (T*)d.k_out + b * d.stride_ko + row * d.ld_ko;
    T* vd = (T*)d.v_out + b * d.stride_vo + row * d.ld_vo;
#pragma unroll
    for (int u = 0; u < UN; u++) {
      if (h0 + u * HP >= heads) break;
      const int h = h0 + u * HP + grp, hk = h - d.heads_q, hv = hk - d.heads_kv;
      const T* src = hk < 0 ? qs + h * D : hv < 0 ? ks + hk * D : vs + hv * D;
      dst[u] = hk < 0 ? qd + h * D : hv < 0 ? kd + hk * D : vd + hv * D;
      if (h >= heads || (hk >= 0 && !room)) {
        dst[u] = nullptr;
        continue;
      }
      xu[u] = *reinterpret_cast<const vec8<T>*>(src + lo);
      xw[u] = *reinterpret_cast<const vec8<T>*>(src + lo + half);
    }
  };
  auto finish = [&](int h0) {
#pragma unroll
    for (int u = 0; u < UN; u++) {
      if (h0 + u * HP >= heads) break;
      const int hk = h0 + u * HP + grp - d.heads_q;
      float x[2][8];
      // x, centred for a LayerNorm, times scale; its mean square
      auto stats = [&](float scale) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 8; i++)
          x[0][i] = (float)xu[u][i] * scale, x[1][i] = (float)xw[u][i] * scale;
        if (d.layer) {
          float m = 0.f;
#pragma unroll
          for (int i = 0; i < 8; i++) m += x[0][i] + x[1][i];
#pragma unroll
          for (int o = LPH / 2; o > 0; o >>= 1) m += __shfl_xor(m, o, 64);
          m *= 1.0f / D;
#pragma unroll
          for (int i = 0; i < 8; i++) x[0][i] -= m, x[1][i] -= m;
        }
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss += x[0][i] * x[0][i] + x[1][i] * x[1][i];
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o, 64);
        return ss * (1.0f / D);
      };
      float var = stats(1.f) + d.eps;
      if constexpr (std::is_same<T, bf16_t>::value) {
        // bf16 has f32's exponents: a head whose squares leave f32 (or whose sum does) is scaled
        const bool out = !(var >= 0x1p-96f && var <= 0x1p126f);
        if (__builtin_amdgcn_ballot_w64(out)) {   // wave-uniform: the shuffles need every lane
          const float scale = !out ? 1.f : var < 0x1p-96f ? 0x1p80f : 0x1p-80f;
          var = stats(scale) + d.eps * scale * scale;
        }
      }
      const float r = 1.0f / sqrtf(var);
      const float(&af)[2][D] = affine[hk < 0 ? 0 : 1];
#pragma unroll
      for (int p = 0; p < 2; p++)
#pragma unroll
        for (int i = 0; i < 8; i++)
          x[p][i] = x[p][i] * (r * af[0][lo + p * half + i]) + af[1][lo + p * half + i];
      vec8<T> yu, yw;
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float co = tab[0][l * 8 + i], si = tab[1][l * 8 + i];   // l * 8 = ax * half + ..
        yu[i] = (T)(x[0][i] * co - x[1][i] * si);
        yw[i] = (T)(x[1][i] * co + x[0][i] * si);
      }
      if (hk >= d.heads_kv) yu = xu[u], yw = xw[u];   // a value head: copied
      if (dst[u]) {
        *reinterpret_cast<vec8<T>*>(dst[u] + lo) = yu;
        *reinterpret_cast<vec8<T>*>(dst[u] + lo + half) = yw;
      }
    }
  };

  // A single token is a chain of loads: lengths, position and factors are asked for together
  // and before the heads, so that what waits for them does not wait for the heads as well.
  constexpr int AF = D / 64;   // factors per thread
  float af[AF];
#pragma unroll
  for (int c = 0; c < AF; c++) {
    const int i = c * 256 + tid, k = i / (2 * D), be = i / D & 1;
    const float* g = k ? (be ? d.beta_k : d.gamma_k) : (be ? d.beta_q : d.gamma_q);
    af[c] = g ? g[i & (D - 1)] : be ? 0.f : 1.f;
  }
  const int pa = lane % (D / 2) / half;
  const int pair = lane % (D / 2) - pa * half;
  const double rev = rt.rev[pair], low = rt.low[pair];
  const uint32_t n = blockIdx.x * 4u + wave, n1 = min(n, a.tokens - 1);
  const int64_t b = n1 / (uint32_t)d.rows, s = n1 - (uint32_t)b * (uint32_t)d.rows;
  const int64_t p = d.pos[b * d.stride_pos + s * d.axes + pa];
  const int64_t row = s + (d.kv_row ? d.kv_row[b] : 0);
  const int len = d.seq_len ? d.seq_len[b] : d.rows;
  const bool on = n < a.tokens && s < len, room = row >= 0 && row < d.cache_rows;
  if (on) load(b, s, row, room, 0);
#pragma unroll
  for (int c = 0; c < AF; c++) (&affine[0][0][0])[c * 256 + tid] = af[c];
  if (lane < D / 2) {
    const double x = (double)p;
    const double r = fma(x, low, fma(x, rev, -rint(x * rev)));
    float sn, c;
    sincospif((float)(2.0 * r), &sn, &c);
    tab[0][lane] = c;
    tab[1][lane] = sn;
  }
  __syncthreads();
  if (!on) return;
  finish(0);
  for (int h0 = UN * HP; h0 < heads; h0 += UN * HP) {
    load(b, s, row, room, h0);
    finish(h0);
  }
}

bool rows_ok(const void* p, int64_t ld, int64_t stride, int64_t width) {
  return p && (uintptr_t)p % 16 == 0 && ld % 8 == 0 && stride % 8 == 0 && ld >= width;
}

}  // namespace

extern "C" int m3s_vit_qk_norm_rope(const m3s_qk_norm_rope_desc* desc, void* stream) {
  if (!desc) return M3S_ERR_INVALID_ARG;
  const m3s_qk_norm_rope_desc& d = *desc;
  if (d.batch < 0 || d.rows < 0 || d.heads_q < 0 || d.heads_kv < 0) return M3S_ERR_INVALID_ARG;
  if ((d.head_dim != 64 && d.head_dim != 128) || (d.axes != 1 && d.axes != 2) ||
      (d.dtype != M3S_BF16 && d.dtype != M3S_F16))
    return M3S_ERR_INVALID_ARG;
  if (!(d.eps >= 0.f) || !(d.base > 0.f) || !isfinite(d.base) || !isfinite(d.eps))
    return M3S_ERR_INVALID_ARG;
  if (d.heads_q > 65535 || d.heads_kv > 65535) return M3S_ERR_TOO_LARGE;
  if (d.batch == 0 || d.rows == 0 || d.heads_q + d.heads_kv == 0) return M3S_OK;
  const int64_t wq = (int64_t)d.heads_q * d.head_dim, wk = (int64_t)d.heads_kv * d.head_dim;
  if (!d.pos || d.stride_pos < 0) return M3S_ERR_INVALID_ARG;
  if (d.heads_q && (!rows_ok(d.q, d.ld_q, d.stride_q, wq) ||
                    !rows_ok(d.q_out, d.ld_qo, d.stride_qo, wq)))
    return M3S_ERR_INVALID_ARG;
  if (d.heads_kv) {
    if (!rows_ok(d.k, d.ld_k, d.stride_k, wk) || !rows_ok(d.k_out, d.ld_ko, d.stride_ko, wk))
      return M3S_ERR_INVALID_ARG;
    if (d.v && (!rows_ok(d.v, d.ld_v, d.stride_v, wk) ||
                !rows_ok(d.v_out, d.ld_vo, d.stride_vo, wk)))
      return M3S_ERR_INVALID_ARG;
    if (d.cache_rows < 0 || (!d.kv_row && d.cache_rows < d.rows)) return M3S_ERR_INVALID_ARG;
  }
  NormArgs a;
  a.d = d;
  if (!d.heads_kv) a.d.v = nullptr;
  const int64_t tokens = (int64_t)d.batch * d.rows, blocks = (tokens + 3) / 4;
  if (blocks >= (1ll << 24)) return M3S_ERR_TOO_LARGE;   // 2^32 threads
  a.tokens = (uint32_t)tokens;
  // base^(-i/half) / 2 pi by one root and repeated products, in extended precision
  RevTable rt;
  const int half = d.head_dim / d.axes / 2;
  const long double step = powl((long double)d.base, -1.0L / half);
  long double f = 1.0L / (2.0L * 3.14159265358979323846264338327950288L);
  for (int i = 0; i < half; i++, f *= step)
    rt.rev[i] = (double)f, rt.low[i] = (float)(f - rt.rev[i]);
  hipStream_t s = m3s_stream(stream);
#define M3S_NORM(T, D)                                                                     \
  hipLaunchKernelGGL((qk_norm_rope_kernel<T, D>), dim3((unsigned)blocks), dim3(256), 0, s, a, rt)
  if (d.dtype == M3S_BF16) {
    if (d.head_dim == 64) M3S_NORM(bf16_t, 64);
    else M3S_NORM(bf16_t, 128);
  } else {
    if (d.head_dim == 64) M3S_NORM(_Float16, 64);
    else M3S_NORM(_Float16, 128);
  }
#undef M3S_NORM
  M3S_LAUNCH_CHECK();
  return M3S_OK;
}
