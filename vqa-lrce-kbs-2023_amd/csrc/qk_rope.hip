// Per-head RMS norm of queries and keys with the rotary position embedding in the same pass, forward and backward.
//
//   xn = x rsqrt(mean(x^2) + eps) w;   the pairs (a, b) of the first R of D dims: (a cos t - b sin t, b cos t + a sin t),
//   t = position * inv_freq[pair]; pairs are (i, R/2 + i), or (2i, 2i + 1) interleaved; the dims from R on stay.
// Backward: g = the inverse rotation of dy;  dw = sum g xhat,  dx = r (g w - xhat mean(g w xhat)),  xhat = x r.
//
// Memory-bound: every row is read and written once (the backward reads x and dy, the row's norm is recomputed).  A lane
// has VEC pairs of a row (two vectors of VEC values), a power of two of lanes a row, so a row's sums are a few shuffles;
// a wave has one token (or several, where its heads are few) and walks the token's heads, query heads first, so the angles are
// formed once a token.  They are formed as turns in 64 bits (position * frequency / 2 pi less its nearest integer): far
// positions lose nothing, and the sine and cosine of the remainder, f32 values, need no range reduction.  All arithmetic on the
// values is f32, rounded once.  The weight gradients are summed in registers over a workgroup's tokens, across its lanes in LDS, and
// over the workgroups by a second kernel in a fixed order.
// Measured: 4 x 8192 tokens of 32 + 8 heads, d 128, bf16: forward 117 us (671 MB, 5.7 TB/s), backward 206 + 5 us (1.0 GB, 4.9 TB/s);
// 10 x 333 tokens of 8 + 8 heads, d 96, f32: 10.8 us, 17.0 + 4.1 us.  The next tokens' rows fetched ahead cost registers and
// so waves: 133 and 232 us at the first size.
#include <algorithm>
#include <cmath>

#include "common.h"
#include "lrce_capi.h"

namespace {

struct RopeP {
  const void *q, *k, *gq, *gk;       // gq, gk: gradients of the outputs (backward)
  void *oq, *ok;                     // outputs; backward: dq, dk
  const float *qw, *kw, *freq;
  const void* pos;
  float* part;                       // backward: [workgroup][2][D]
  float *dqw, *dkw;
  long long sq[3], sk[3], sgq[3], sgk[3], soq[3], sok[3];
  long long pos_b;
  long long tokens;
  int L, H, Hk, D, R, inter, pos64, gpt, lgrp, nwg;
  float eps;
};

template <typename T> struct Io;
template <> struct Io<float> {
  static __device__ __forceinline__ float get(float x) { return x; }
  static __device__ __forceinline__ float put(float x) { return x; }
};
template <> struct Io<bf16> {
  static __device__ __forceinline__ float get(bf16 x) { return bf2f(x); }
  static __device__ __forceinline__ bf16 put(float x) { return f2bf(x); }
};
template <> struct Io<f16> {
  static __device__ __forceinline__ float get(f16 x) { return h2f(x); }
  static __device__ __forceinline__ f16 put(float x) { return f2h(x); }
};

template <typename T, int V> struct Vec { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct Vec<T, 1> { typedef T type; };

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float* x) {
  if constexpr (V == 1) x[0] = Io<T>::get(*p);
  else {
    const typename Vec<T, V>::type v = *reinterpret_cast<const typename Vec<T, V>::type*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = Io<T>::get(v[i]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float* x) {
  if constexpr (V == 1) *p = Io<T>::put(x[0]);
  else {
    typename Vec<T, V>::type v;
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = Io<T>::put(x[i]);
    *reinterpret_cast<typename Vec<T, V>::type*>(p) = v;
  }
}

// sum over the 2^n lanes of a row
__device__ __forceinline__ float row_sum(float x, int n) {
  for (int o = 1; o < (1 << n); o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}

// Where a lane's pairs [pi, pi + VEC) lie: two vectors at lo and hi; cs / sn: their angles (1, 0 from R on)
template <int VEC>
struct Pairs {
  int lo, hi, pi;
  bool on;
  float cs[VEC], sn[VEC];
  __device__ __forceinline__ void place(const RopeP& p, int first) {
    pi = first;
    on = pi < p.D / 2;
    const int half = p.R / 2;
    if (p.inter) { lo = 2 * pi; hi = 2 * pi + VEC; }
    else if (pi < half) { lo = pi; hi = half + pi; }
    else { lo = half + pi; hi = p.D / 2 + pi; }          // R + (pi - R/2), R + (D - R)/2 + (pi - R/2)
    if (!on) lo = hi = 0;
  }
  __device__ __forceinline__ void angles(const RopeP& p, double position) {
    constexpr double PER_TURN = 0.15915494309189533577;  // 1 / (2 pi)
#pragma unroll
    for (int i = 0; i < VEC; ++i) { cs[i] = 1.f; sn[i] = 0.f; }
    if (on && pi < p.R / 2) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const double turns = position * (double)p.freq[pi + i] * PER_TURN, x = 2.0 * (turns - __builtin_rint(turns));
        // x in f32 is up to 2^-25 half turns off, 1e-7 radians; the rest of it is added to first order (the second is below 2^-47)
        const float near = (float)x, rest = (float)(x - (double)near) * 3.14159265f;
        float s, c;
        sincospif(near, &s, &c);
        sn[i] = __builtin_fmaf(c, rest, s);
        cs[i] = __builtin_fmaf(-s, rest, c);
      }
    }
  }
  // x: lo vector then hi vector; rotated in place (dir = -1: back)
  __device__ __forceinline__ void turn(float* x, bool inter, float dir) const {
    if (inter) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float a = x[2 * i], b = x[2 * i + 1], s = dir * sn[i];
        x[2 * i] = a * cs[i] - b * s;
        x[2 * i + 1] = b * cs[i] + a * s;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float a = x[i], b = x[VEC + i], s = dir * sn[i];
        x[i] = a * cs[i] - b * s;
        x[VEC + i] = b * cs[i] + a * s;
      }
    }
  }
};

// NCH chunks of VEC pairs a lane (2 only where VEC = 1 and D > 128)
template <typename T, int VEC, int NCH, bool BWD>
__global__ void __launch_bounds__(256, BWD ? (VEC == 8 ? 3 : 4) : 5) qk_rope_kernel(RopeP p) {
  constexpr int W = 2 * VEC;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lanes = 1 << p.lgrp, ngrp = 64 >> p.lgrp, grp = lane >> p.lgrp, li = lane & (lanes - 1);
  const int tpw = ngrp / p.gpt;                           // tokens a wave
  const int hg = grp % p.gpt;                             // this group's first head
  Pairs<VEC> pr[NCH];
#pragma unroll
  for (int c = 0; c < NCH; ++c) pr[c].place(p, (li + c * lanes) * VEC);
  float dw[BWD ? 2 : 1][NCH][W];
  if constexpr (BWD) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < W; ++i) dw[a][c][i] = 0.f;
  }
  const float inv_d = 1.f / (float)p.D;
  for (long long t0 = ((long long)blockIdx.x * 4 + wave) * tpw; t0 < p.tokens; t0 += (long long)gridDim.x * 4 * tpw) {
    const long long tok = t0 + grp / p.gpt;
    const bool live = tok < p.tokens;
    const long long b = live ? tok / p.L : 0, l = live ? tok - b * p.L : 0;
    const long long pat = b * p.pos_b + l;
    const double position = p.pos64 ? (double)static_cast<const long long*>(p.pos)[pat] : (double)static_cast<const int*>(p.pos)[pat];
#pragma unroll
    for (int c = 0; c < NCH; ++c) pr[c].angles(p, position);
#pragma unroll
    for (int a = 0; a < 2; ++a) {                         // query heads, key heads
      const int nh = a ? p.Hk : p.H;
      const long long* sx = a ? p.sk : p.sq;
      const long long* so = a ? p.sok : p.soq;
      const long long* sg = a ? p.sgk : p.sgq;
      const T* xb = static_cast<const T*>(a ? p.k : p.q) + b * sx[0] + l * sx[1];
      const T* gb = BWD ? static_cast<const T*>(a ? p.gk : p.gq) + b * sg[0] + l * sg[1] : nullptr;
      T* ob = static_cast<T*>(a ? p.ok : p.oq) + b * so[0] + l * so[1];
      const float* wp = a ? p.kw : p.qw;
      float w[NCH][W];
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        load_vec<float, VEC>(wp + pr[c].lo, w[c]);
        load_vec<float, VEC>(wp + pr[c].hi, w[c] + VEC);
      }
      const int rounds = (nh + p.gpt - 1) / p.gpt;        // every lane of the wave runs the shuffles of every round
      for (int it = 0; it < rounds; ++it) {
        const int hd = hg + it * p.gpt;
        const bool act = live && hd < nh;
        float x[NCH][W], g[BWD ? NCH : 1][W];
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
#pragma unroll
          for (int i = 0; i < W; ++i) x[c][i] = 0.f;
          if (act && pr[c].on) {
            load_vec<T, VEC>(xb + hd * sx[2] + pr[c].lo, x[c]);
            load_vec<T, VEC>(xb + hd * sx[2] + pr[c].hi, x[c] + VEC);
          }
          if constexpr (BWD) {
#pragma unroll
            for (int i = 0; i < W; ++i) g[c][i] = 0.f;
            if (act && pr[c].on) {
              load_vec<T, VEC>(gb + hd * sg[2] + pr[c].lo, g[c]);
              load_vec<T, VEC>(gb + hd * sg[2] + pr[c].hi, g[c] + VEC);
            }
          }
#pragma unroll
          for (int i = 0; i < W; ++i) ss = __builtin_fmaf(x[c][i], x[c][i], ss);
        }
        if constexpr (!BWD) {
          const float r = 1.f / sqrtf(row_sum(ss, p.lgrp) * inv_d + p.eps);
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
#pragma unroll
            for (int i = 0; i < W; ++i) x[c][i] = x[c][i] * r * w[c][i];
            pr[c].turn(x[c], p.inter, 1.f);
            if (act && pr[c].on) {
              store_vec<T, VEC>(ob + hd * so[2] + pr[c].lo, x[c]);
              store_vec<T, VEC>(ob + hd * so[2] + pr[c].hi, x[c] + VEC);
            }
          }
        } else {
          float sg_ = 0.f;
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            pr[c].turn(g[c], p.inter, -1.f);
#pragma unroll
            for (int i = 0; i < W; ++i) sg_ = __builtin_fmaf(g[c][i] * w[c][i], x[c][i], sg_);
          }
          for (int o = 1; o < lanes; o <<= 1) {
            ss += __shfl_xor(ss, o, 64);
            sg_ += __shfl_xor(sg_, o, 64);
          }
          // (a group without a head or a token has ss = 0: with eps = 0 its 0 / 0 would reach the weights' gradients)
          const float r = act ? 1.f / sqrtf(ss * inv_d + p.eps) : 0.f, m = sg_ * r * inv_d;   // m = mean(g w xhat)
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            float o[W];
#pragma unroll
            for (int i = 0; i < W; ++i) {
              const float xh = x[c][i] * r;
              dw[a][c][i] = __builtin_fmaf(g[c][i], xh, dw[a][c][i]);
              o[i] = r * (g[c][i] * w[c][i] - xh * m);
            }
            if (act && pr[c].on) {
              store_vec<T, VEC>(ob + hd * so[2] + pr[c].lo, o);
              store_vec<T, VEC>(ob + hd * so[2] + pr[c].hi, o + VEC);
            }
          }
        }
      }
    }
  }
  if constexpr (BWD) {
    // lanes of the same pairs: over the wave's groups by shuffles, over the waves in LDS
    __shared__ float red[4][2][256];
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int c = 0; c < NCH; ++c)
#pragma unroll
        for (int i = 0; i < W; ++i) {
          float v = dw[a][c][i];
          for (int o = lanes; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
          if (grp == 0 && pr[c].on) red[wave][a][i < VEC ? pr[c].lo + i : pr[c].hi + i - VEC] = v;
        }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * p.D; e += 256) {
      const int a = e / p.D, d = e - a * p.D;
      p.part[(long long)blockIdx.x * 2 * p.D + e] = ((red[0][a][d] + red[1][a][d]) + red[2][a][d]) + red[3][a][d];
    }
  }
}

// dw[e] = the workgroups' sums, 16 columns a workgroup, 64 threads a column that each add every 64th in order
__global__ void __launch_bounds__(1024) qk_rope_dw_kernel(RopeP p) {
  __shared__ float red[64][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
  float s = 0.f;
  if (e < 2 * p.D) {
#pragma unroll 8
    for (int i = r; i < p.nwg; i += 64) s += p.part[(long long)i * 2 * p.D + e];
  }
  red[r][c] = s;
  __syncthreads();
  for (int o = 32; o > 0; o >>= 1) {
    if (r < o) red[r][c] += red[r + o][c];
    __syncthreads();
  }
  if (r == 0 && e < 2 * p.D) {
    if (e < p.D) p.dqw[e] = red[0][c];
    else p.dkw[e - p.D] = red[0][c];
  }
}

int rope_check(const LrceRopeDesc* d, bool bwd, const char* what) {
  if (!d) return lrce_fail(LRCE_E_ARG, "%s: null descriptor", what);
  if (d->B < 0 || d->L < 0 || d->H < 1 || d->Hk < 1) return lrce_fail(LRCE_E_ARG, "%s: bad sizes B=%d L=%d H=%d Hk=%d", what, d->B, d->L, d->H, d->Hk);
  if (d->D < 8 || d->D > 256 || d->D % 8) return lrce_fail(LRCE_E_ARG, "%s: head dim %d (a multiple of 8 up to 256)", what, d->D);
  if (d->R < 2 || d->R > d->D || d->R % 2) return lrce_fail(LRCE_E_ARG, "%s: %d rotated dims of %d (even, at least 2)", what, d->R, d->D);
  if (d->dtype < 0 || d->dtype > 2) return lrce_fail(LRCE_E_ARG, "%s: dtype %d", what, d->dtype);
  if (!(d->eps >= 0.f) || !std::isfinite(d->eps)) return lrce_fail(LRCE_E_ARG, "%s: eps must be finite and not negative", what);
  if (d->pos_bytes != 4 && d->pos_bytes != 8) return lrce_fail(LRCE_E_ARG, "%s: positions of %d bytes (4 or 8)", what, d->pos_bytes);
  if (!d->q_weight || !d->k_weight || !d->inv_freq) return lrce_fail(LRCE_E_ARG, "%s: null pointer", what);
  if (bwd && (!d->dq_weight || !d->dk_weight)) return lrce_fail(LRCE_E_ARG, "%s: null gradient pointer", what);
  if (d->B > 0 && d->L > 0) {
    if (!d->q || !d->k || !d->q_out || !d->k_out || !d->positions) return lrce_fail(LRCE_E_ARG, "%s: null pointer", what);
    if (bwd && (!d->gq || !d->gk)) return lrce_fail(LRCE_E_ARG, "%s: null gradient pointer", what);
  }
  return LRCE_OK;
}

// The backward leaves a row of partial sums a workgroup, four waves of at least a token each: up to 4 workgroups a CU
int64_t rope_wgs(int64_t tokens) { return std::max<int64_t>(1, std::min<int64_t>((tokens + 3) / 4, 1024)); }

struct RopePlan { int vec, lgrp, gpt, tpw; };

RopePlan rope_plan(const LrceRopeDesc* d, bool bwd) {
  const int es = d->dtype == 2 ? 4 : 2;
  auto fits = [&](int v) {
    if (d->D % (2 * v) || (d->R / 2) % v || ((d->D - d->R) / 2) % v) return false;
    const void* at[] = {d->q, d->k, d->q_out, d->k_out, bwd ? d->gq : nullptr, bwd ? d->gk : nullptr};
    const int64_t* st[] = {d->q_stride, d->k_stride, d->qo_stride, d->ko_stride, d->gq_stride, d->gk_stride};
    for (int i = 0; i < (bwd ? 6 : 4); ++i) {
      if (reinterpret_cast<uintptr_t>(at[i]) % (v * es)) return false;
      for (int k = 0; k < 3; ++k)
        if (st[i][k] % v) return false;
    }
    return !(reinterpret_cast<uintptr_t>(d->q_weight) % (v * 4 > 16 ? 16 : v * 4)) && !(reinterpret_cast<uintptr_t>(d->k_weight) % (v * 4 > 16 ? 16 : v * 4));
  };
  RopePlan f;
  f.vec = es == 4 ? 4 : 8;
  while (f.vec > 1 && !fits(f.vec)) f.vec /= 2;
  const int need = d->D / (2 * f.vec);
  f.lgrp = 0;
  while ((1 << f.lgrp) < need && f.lgrp < 6) ++f.lgrp;
  const int ngrp = 64 >> f.lgrp;
  int g = 1;
  while (g < ngrp && g < std::max(d->H, d->Hk)) g *= 2;
  f.gpt = g;
  f.tpw = ngrp / g;
  return f;
}

template <typename T, int VEC, int NCH, bool BWD>
void rope_go(const RopeP& p, int64_t grid, hipStream_t s) {
  qk_rope_kernel<T, VEC, NCH, BWD><<<(unsigned)grid, 256, 0, s>>>(p);
}
template <typename T, bool BWD>
void rope_vec(const RopeP& p, int vec, int64_t grid, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (vec == 8) return rope_go<T, 8, 1, BWD>(p, grid, s);
  if (vec == 4) return rope_go<T, 4, 1, BWD>(p, grid, s);
  if (vec == 2) return rope_go<T, 2, 1, BWD>(p, grid, s);
  if (p.D <= 128) return rope_go<T, 1, 1, BWD>(p, grid, s);
  rope_go<T, 1, 2, BWD>(p, grid, s);
}
template <bool BWD>
void rope_type(const RopeP& p, int dtype, int vec, int64_t grid, hipStream_t s) {
  if (dtype == 0) rope_vec<bf16, BWD>(p, vec, grid, s);
  else if (dtype == 1) rope_vec<f16, BWD>(p, vec, grid, s);
  else rope_vec<float, BWD>(p, vec, grid, s);
}

void rope_fill(const LrceRopeDesc* d, const RopePlan& f, RopeP& p) {
  p = RopeP{};
  p.q = d->q; p.k = d->k; p.gq = d->gq; p.gk = d->gk; p.oq = d->q_out; p.ok = d->k_out;
  p.qw = d->q_weight; p.kw = d->k_weight; p.freq = d->inv_freq; p.pos = d->positions;
  p.part = d->workspace; p.dqw = d->dq_weight; p.dkw = d->dk_weight;
  for (int i = 0; i < 3; ++i) {
    p.sq[i] = d->q_stride[i]; p.sk[i] = d->k_stride[i]; p.soq[i] = d->qo_stride[i]; p.sok[i] = d->ko_stride[i];
    p.sgq[i] = d->gq_stride[i]; p.sgk[i] = d->gk_stride[i];
  }
  p.pos_b = d->pos_stride; p.pos64 = d->pos_bytes == 8;
  p.tokens = (long long)d->B * d->L;
  p.L = d->L; p.H = d->H; p.Hk = d->Hk; p.D = d->D; p.R = d->R; p.inter = d->interleaved;
  p.gpt = f.gpt; p.lgrp = f.lgrp; p.eps = d->eps;
}

}  // namespace

extern "C" int lrce_qk_norm_rope_fwd(const LrceRopeDesc* d, void* stream) {
  if (const int rc = rope_check(d, false, "qk_norm_rope")) return rc;
  if (d->B == 0 || d->L == 0) return LRCE_OK;
  const RopePlan f = rope_plan(d, false);
  RopeP p;
  rope_fill(d, f, p);
  const int64_t grid = std::min<int64_t>((p.tokens + 4 * f.tpw - 1) / (4 * f.tpw), 1 << 20);
  rope_type<false>(p, d->dtype, f.vec, grid, static_cast<hipStream_t>(stream));
  return lrce_check_launch("qk_norm_rope");
}

extern "C" int64_t lrce_qk_norm_rope_bwd_workspace(int64_t tokens, int D) {
  if (tokens < 0 || D < 8 || D > 256 || D % 8) return -1;
  return rope_wgs(tokens) * 2 * D;
}

extern "C" int lrce_qk_norm_rope_bwd(const LrceRopeDesc* d, void* stream) {
  if (const int rc = rope_check(d, true, "qk_norm_rope_bwd")) return rc;
  const RopePlan f = rope_plan(d, true);
  RopeP p;
  rope_fill(d, f, p);
  p.nwg = (int)std::min<int64_t>(rope_wgs(p.tokens), f.vec == 8 ? 768 : 1024);   // what is resident: 3 or 4 waves a SIMD (1024 of 768: 268 us, not 207)
  if (!d->workspace || d->workspace_elems < (int64_t)p.nwg * 2 * d->D)
    return lrce_fail(LRCE_E_ARG, "qk_norm_rope_bwd: a workspace of %lld floats is needed", (long long)p.nwg * 2 * d->D);
  hipStream_t s = static_cast<hipStream_t>(stream);
  rope_type<true>(p, d->dtype, f.vec, p.nwg, s);
  qk_rope_dw_kernel<<<(2 * d->D + 15) / 16, 1024, 0, s>>>(p);
  return lrce_check_launch("qk_norm_rope_bwd");
}
