// Multi-head attention at general lengths on gfx950: head dims 32 / 64 / 96 / 128, bf16 or fp16, shared key / value
// heads, a key mask and / or causality, forward.
//
//   s_ij = scale q_i . k_j,  m_i = max_j s_ij,  l_i = sum_j exp(s_ij - m_i),  o_i = sum_j exp(s_ij - m_i) v_j / l_i,
//   lse_i = m_i + ln l_i
// over the keys that row i may see; a row that sees none gives o = 0, lse = -inf.  One pass over the keys with a
// running maximum and sum in f32.  S^T = K Q^T, so a lane owns one query: the row statistics are in-lane plus one
// exchange of the wave's halves, and P^T, rounded to 16 bits (half a unit in the last place of each weight, the size
// of the output's own rounding: the output's error is 1.2 - 1.4 times what f32 weights leave), is at once the B operand of
// O^T += V^T P^T.  The running maximum is raised only when a
// tile exceeds it by more than 2^8 (the weights then stay below 2^8, harmless in f32 and in both 16-bit types), which
// leaves the accumulators alone in nearly all tiles.
//
// Measured: 2 x 8 heads x 4096 x 4096, d 128, bf16 132 us (1040 TFLOP/s), causal with 2 x 16 heads on 4 147 us (935 TFLOP/s counted,
// 1008 formed; 165 in a loop of nothing else, where the clock falls); a plain 8192^3 product 1290 TFLOP/s.  The matrix pipe is busy 53 % of the cycles there, at a clock that the load
// holds near 1.7 GHz; LDS 26 %, without bank conflicts.  Bound by the waits for LDS reads (1 KB a matrix instruction) and
// by the exponentials: without these 133 of 141 us, without LDS reads 110, with nothing but products 103.  At d 32 (48 heads x
// 1568^2, 41 us) by the vector unit: an exponential and 4 to 5 more instructions a score against 64 multiply-adds.  One token over 32 caches of
// up to 8190 keys (32 heads on 8, d 128): 147 us, 5.0 TB/s of keys and values.
//
// attn_fwd_kernel: a wave has 32 query rows, a workgroup NW waves that share K / V tiles of 64 keys, double buffered.
// attn_split_kernel: few rows (single tokens).  All query heads of a key head are rows of one tile, so K / V are read
// once; each wave walks 32-key tiles of its own and the waves' shares of the keys are joined.
#include <algorithm>
#include <cmath>

#include "attention_util.h"

namespace {

// One query tile (32 rows): the state of a wave
template <int D, bool F16>
struct FwdState {
  bf16x8 q[D / 16];
  f32x16 acc[D / 32];
  float m, l;      // running maximum (raw scores), sum of this half's weights

  __device__ __forceinline__ void init(const bf16* row, int h) {
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) q[kk] = *reinterpret_cast<const bf16x8*>(row + 16 * kk + 8 * h);
    attn_landed(q);
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
    m = -INFINITY;
    l = 0.f;
  }
  // raw scores of the 32 keys from row r0 of the tile on
  __device__ __forceinline__ f32x16 scores(const TileRead<D>& rd, lds_cptr kt, int r0) const {
    f32x16 s = mfma32x32x16<F16>(rd.row(kt, r0, 0), q[0], f32x16{});
#pragma unroll
    for (int kk = 1; kk < D / 16; ++kk) s = mfma32x32x16<F16>(rd.row(kt, r0, kk), q[kk], s);
    return s;
  }
  // kw[blk]: bit = key of the block this lane's query may see, shifted by 4 h
  template <int NKB>
  __device__ __forceinline__ static void hide(f32x16 (&s)[NKB], const uint32_t* kw) {
#pragma unroll
    for (int blk = 0; blk < NKB; ++blk)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[blk][r] = (kw[blk] >> ((r & 3) + 8 * (r >> 2))) & 1 ? s[blk][r] : -INFINITY;
  }
  template <int NKB>
  __device__ __forceinline__ static float top(const f32x16 (&s)[NKB]) {
    float mx = s[0][0];
#pragma unroll
    for (int blk = 0; blk < NKB; ++blk)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[blk][r]);
    return fmaxf(mx, other_half(mx));
  }
  // the running maximum follows mx where it has to
  __device__ __forceinline__ void raise(float mx, float c) {
    if (__any(mx > m && !((mx - m) * c <= 8.f))) {
      const float mn = fmaxf(m, mx);
      const float a = mn > m ? __builtin_amdgcn_exp2f((m - mn) * c) : 1.f;
      l *= a;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] *= a;
      m = mn;
    }
  }
  __device__ __forceinline__ float offset(float c) const { return m == -INFINITY ? 0.f : m * c; }
  // scores -> weights (16 bits), their sum
  __device__ __forceinline__ void weigh(f32x16& s, bf16x8 (&pf)[2], float c, float mc) {
    float t[4] = {l, 0.f, 0.f, 0.f};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int r = 8 * half; r < 8 * half + 8; ++r) {
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -mc));
        t[r & 3] += s[r];
      }
      pf[half] = attn_pack<F16>(s, half);
    }
    l = (t[0] + t[1]) + (t[2] + t[3]);
  }
  // the 32 keys from row r0 of the tile on
  __device__ __forceinline__ void sum(const TileRead<D>& rd, lds_cptr vt, int r0, const bf16x8 (&pf)[2]) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = mfma32x32x16<F16>(rd.col(vt, r0 + 16 * k, i), pf[k], acc[i]);
  }
};

// Pipelined by one tile: the scores of the next tile (matrix pipe) are formed while the current one is exponentiated, its
// maximum while the current one is multiplied by V.  So K runs one tile ahead of V in LDS, two places each.
template <int D, bool F16, int NW, bool MASK>
__global__ void __launch_bounds__(NW * 64, 2) attn_fwd_kernel(AttnP p) {
  constexpr int KT = 64, TB = KT * D * 2;
  typedef TileStage<D, KT, NW> Stage;
  __shared__ __attribute__((aligned(1024))) char buf[4 * TB];            // K, K, V, V
  __shared__ uint64_t words[MASK ? ATTN_MASK_KEYS / KT : 1];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), h = lane >> 5;
  const Place at = attn_place(p, p.G);
  const int blk = p.nblk - 1 - at.blk, b = at.b, hq = at.hq, hk = hq / p.G, bh = b * p.H + hq;   // (causal: the last rows see most)
  const int i0 = blk * (32 * NW) + wave * 32;                            // this wave's first row
  const int row = min(i0 + (lane & 31), p.Lq - 1);
  const int last = min(blk * (32 * NW) + 32 * NW, p.Lq) - 1;             // the workgroup's last row
  const int nk = p.causal ? max(0, min(p.Lk, last + p.off + 1)) : p.Lk;
  const int nt = (nk + KT - 1) / KT;
  // tiles from tw on hold no key that this wave's rows see
  const int tw = p.causal ? min(nt, max(0, i0 + 31 + p.off + KT) / KT) : nt;

  FwdState<D, F16> st;
  st.init(p.q + b * p.sqb + row * p.sql + hq * p.sqh, h);
  TileRead<D> rd;
  rd.init(lane);
  Stage sk, sv;
  sk.init(lane, wave, p.skl);
  sv.init(lane, wave, p.svl);
  const char* kb = uni(p.k + b * p.skb + hk * p.skh);
  const char* vb = uni(p.v + b * p.svb + hk * p.svh);
  const long long kstep = p.skl * (2 * KT), vstep = p.svl * (2 * KT);
  lds_ptr lds = (lds_ptr)buf;
  LRCE_LDS uint64_t* lw = (LRCE_LDS uint64_t*)words;

  const int chunk = MASK ? ATTN_MASK_KEYS / KT : nt;
  for (int c0 = 0; c0 < nt; c0 += chunk) {
    const int c1 = min(nt, c0 + chunk);
    if constexpr (MASK) {
      __syncthreads();
      attn_pack_mask<NW>(p, b, c0, c1 - c0, lw, lane, wave);
      __syncthreads();
    }
    auto next = [&](int t, uint64_t& w) {      // the first tile from t on with a visible key
      if constexpr (MASK) {
        for (; t < c1; ++t)
          if ((w = uni64(lw[t - c0])) != 0) break;
      } else {
        w = low_bits(p.Lk - t * KT);
      }
      return t;
    };
    auto stage = [&](const Stage& s, const char* base, long long step, int t, uint64_t w, int at) {
      const uint32_t dst = attn_lds_u32(lds + at * TB);
      if (MASK && w != ~0ull) s.load(base + t * step, p.Lk - t * KT, w, dst, lane, wave);
      else s.load(base + t * step, p.Lk - t * KT, dst, wave);
    };
    f32x16 s[2];
    float mx;
    auto mask = [&](int t, uint64_t w, f32x16 (&x)[2]) {
      const int lim = i0 + p.off - t * KT;                               // the wave's first row sees keys up to t KT + lim
      const bool diag = p.causal && lim < KT - 1;
      if (diag || w != ~0ull) {
        const int mine = lim + (lane & 31);
        const uint32_t kw[2] = {((uint32_t)w & (diag ? upto(mine) : ~0u)) >> (4 * h),
                                ((uint32_t)(w >> 32) & (diag ? upto(mine - 32) : ~0u)) >> (4 * h)};
        st.template hide<2>(x, kw);
      }
    };
    uint64_t w = 0, w1 = 0, w2 = 0;
    int t = next(c0, w);
    if (t >= c1) continue;
    stage(sk, kb, kstep, t, w, 0);
    int t1 = next(t + 1, w1), cur = 0;
    attn_barrier();
    if (t1 < c1) stage(sk, kb, kstep, t1, w1, 1);
    stage(sv, vb, vstep, t, w, 2);
    if (t < tw) {
      s[0] = st.scores(rd, lds, 0);
      s[1] = st.scores(rd, lds, 32);
      mask(t, w, s);
      mx = st.template top<2>(s);
    }
    // a step: K of t1 and V of t are there, K of t and V before it are done with; the tiles after them are sent for
    auto step = [&] {
      attn_barrier();
      const int t2 = next(t1 + 1, w2);
      if (t2 < c1) stage(sk, kb, kstep, t2, w2, cur);
      if (t1 < c1) stage(sv, vb, vstep, t1, w1, 2 + (cur ^ 1));
      return t2;
    };
    int t2 = step();
    while (t1 < c1 && t1 < tw) {
      bf16x8 p0[2], p1[2];
      st.raise(mx, p.c);
      const float mc = st.offset(p.c);
      lds_cptr kt = lds + (cur ^ 1) * TB, vt = lds + (2 + cur) * TB;
      f32x16 sn[2];
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);                                     // the wave with matrix work first: 3 - 7 % at 2 waves a SIMD
      sn[0] = st.scores(rd, kt, 0);
      st.weigh(s[0], p0, p.c, mc);
      attn_interleave<D / 16, 128 / D * 7>();
      __builtin_amdgcn_sched_barrier(0);
      sn[1] = st.scores(rd, kt, 32);
      st.sum(rd, vt, 0, p0);
      st.weigh(s[1], p1, p.c, mc);
      attn_interleave<D / 8, 128 / D * 4>();
      __builtin_amdgcn_sched_barrier(0);
      st.sum(rd, vt, 32, p1);
      __builtin_amdgcn_s_setprio(0);
      mask(t1, w1, sn);
      mx = st.template top<2>(sn);
      s[0] = sn[0];
      s[1] = sn[1];
      t = t1; w = w1; t1 = t2; w1 = w2;
      cur ^= 1;
      t2 = step();
    }
    if (t < tw) {                                                        // this wave's last tile
      bf16x8 pf[2];
      st.raise(mx, p.c);
      const float mc = st.offset(p.c);
      lds_cptr vt = lds + (2 + cur) * TB;
#pragma unroll
      for (int blk = 0; blk < 2; ++blk) {
        st.weigh(s[blk], pf, p.c, mc);
        st.sum(rd, vt, 32 * blk, pf);
      }
    }
    while (t1 < c1) {                                                    // the other waves' steps
      t1 = t2; w1 = w2;
      cur ^= 1;
      t2 = step();
    }
  }
  const float l = st.l + other_half(st.l);
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const bool valid = i0 + (lane & 31) < p.Lq;
  bf16* o = p.out + b * p.sob + row * p.sol + hq * p.soh;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) attn_store<F16>(st.acc[i], inv, o + 32 * i, h, valid);
  if (valid && h == 0) p.lse[(long long)bh * p.Lq + row] = l == 0.f ? -INFINITY : st.m * p.scale + __logf(l);
}

// What a share (maximum m, sum l) counts at the common maximum mx; a share that saw nothing (its sums are zeros) counts nothing.
// A factor that underflows to 0 is multiplied all the same: a NaN among the share's values stays one, as within a share.
__device__ __forceinline__ float join_factor(float m, float l, float mx, float c) {
  return m == -INFINITY && l == 0.f ? 0.f : l != l ? l : __builtin_amdgcn_exp2f((m - mx) * c);
}

// The rows of a key head: r = i * G + g for query i and head g of the group, 32 a tile.  A workgroup takes the key tiles
// [split * split_tiles, ...) of 32 keys, wave w every NW-th of them; a wave has its own tiles in LDS and waits for nobody.
// NW = 2, 4: one workgroup a row tile, the waves' shares joined in LDS.  NW = 1: long key axes, cut into shares of one wave
// each (four to eight of them a CU: one's start and end is hidden by the others), joined by attn_join_kernel.
template <int D, bool F16, int NW>
__global__ void __launch_bounds__(64 * NW, D <= 64 ? 2 : 1) attn_split_kernel(AttnP p) {
  constexpr int KT = 32, TB = KT * D * 2, NST = 2;
  typedef TileStage<D, KT, 1> Stage;
  constexpr int OP = D + 4;                                              // padded row of a joined output tile (floats)
  constexpr int SZ = NW > 1 && NW * 32 * OP * 4 > NW * NST * 2 * TB ? NW * 32 * OP * 4 : NW * NST * 2 * TB;
  __shared__ __attribute__((aligned(1024))) char buf[SZ];
  __shared__ float sm[NW][32], sl[NW][32];
  const int lane = threadIdx.x & 63, wave = NW > 1 ? uni(threadIdx.x >> 6) : 0, h = lane >> 5, n = lane & 31;
  // shares go round the XCDs (batch rows differ in visible keys); the row tiles of one share meet on one where their number allows
  const int un = gridDim.x / p.nblk, id = blockIdx.x % un, rt = blockIdx.x / un;
  const int sp = id % p.nsplit, bk = id / p.nsplit, b = bk / p.Hk, hk = bk % p.Hk;
  const int R = p.Lq * p.G;
  const int r = min(rt * 32 + n, R - 1), qi = r / p.G, hq = hk * p.G + r % p.G;
  const int last = (min(rt * 32 + 31, R - 1)) / p.G;
  const int nk = p.causal ? max(0, min(p.Lk, last + p.off + 1)) : p.Lk;
  const int nt = (nk + KT - 1) / KT;
  const int b0 = sp * p.split_tiles, b1 = min(nt, b0 + p.split_tiles);   // split_tiles is a multiple of 2

  FwdState<D, F16> st;
  st.init(p.q + b * p.sqb + qi * p.sql + hq * p.sqh, h);
  TileRead<D> rd;
  rd.init(lane);
  Stage sk, sv;
  sk.init(lane, 0, p.skl);
  sv.init(lane, 0, p.svl);
  const char* kb = uni(p.k + b * p.skb + hk * p.skh);
  const char* vb = uni(p.v + b * p.svb + hk * p.svh);
  const long long kstep = p.skl * (2 * KT), vstep = p.svl * (2 * KT);
  lds_ptr lds = (lds_ptr)buf + wave * (NST * 2 * TB);

  // the mask bits of 128 tiles at a time: lane l has those of keys 64 l .. 64 l + 63
  const int chunk = p.mask ? 128 : max(b1 - b0, 1);
  for (int c0 = b0; c0 < b1; c0 += chunk) {
    const int c1 = min(b1, c0 + chunk);
    uint32_t mlo = 0, mhi = 0;
    if (p.mask)
      attn_mask_words<1>(p, b, c0 / 2, (c1 + 1) / 2, lane, [&](int w, uint64_t bits) {
        if (lane == w - c0 / 2) { mlo = (uint32_t)bits; mhi = (uint32_t)(bits >> 32); }
      });
    auto word = [&](int t) {
      if (!p.mask) return (uint32_t)low_bits(p.Lk - t * KT);
      const int w = (t - c0) >> 1;
      return (uint32_t)__builtin_amdgcn_readlane(((t - c0) & 1) ? mhi : mlo, w);
    };
    auto next = [&](int t, uint32_t& w) {
      for (; t < c1; t += NW)
        if ((w = word(t)) != 0) break;
      return t;
    };
    auto stage = [&](int t, uint32_t w, int cur) {
      const char *ka = kb + t * kstep, *va = vb + t * vstep;
      const uint32_t kd = attn_lds_u32(lds + 2 * cur * TB), vd = attn_lds_u32(lds + (2 * cur + 1) * TB);
      const int n = p.Lk - t * KT;
      if (p.mask && w != ~0u) {
        sk.load(ka, n, w, kd, lane, 0);
        sv.load(va, n, w, vd, lane, 0);
      } else {
        sk.load(ka, n, kd, 0);
        sv.load(va, n, vd, 0);
      }
    };
    uint32_t w0 = 0, w1 = 0, w2 = 0;
    int cur = 0;
    int t0 = next(c0 + wave, w0);
    if (t0 < c1) stage(t0, w0, 0);
    int t1 = next(t0 + NW, w1);
    if (t1 < c1) stage(t1, w1, 1);
    while (t0 < c1) {
      if (t1 < c1) attn_wait_vm<2 * Stage::NI>();
      else attn_wait_vm<0>();
      const int lim = p.causal ? qi + p.off - t0 * KT : 31;
      const bool masked = w0 != ~0u || (p.causal && __any(lim < 31));
      f32x16 s[1];
      bf16x8 pf[2];
      s[0] = st.scores(rd, lds + 2 * cur * TB, 0);
      if (masked) {
        const uint32_t kw[1] = {(w0 & upto(lim)) >> (4 * h)};
        st.template hide<1>(s, kw);
      }
      st.raise(st.template top<1>(s), p.c);
      st.weigh(s[0], pf, p.c, st.offset(p.c));
      st.sum(rd, lds + (2 * cur + 1) * TB, 0, pf);
      const int t2 = next(t1 + NW, w2);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // the tile's reads are done: its place may be filled
      if (t2 < c1) stage(t2, w2, cur);
      t0 = t1; w0 = w1;
      t1 = t2; w1 = w2;
      cur ^= 1;
    }
  }
  const float l = st.l + other_half(st.l);
  const long long rows = (long long)p.B * p.H * p.Lq;
  if constexpr (NW == 1) {
    // partials [split][row][D] and (maximum, sum), both before the division
    if (rt * 32 + n < R) {
      const long long at = (long long)sp * rows + ((long long)b * p.H + hq) * p.Lq + qi;
      float* dst = p.ws + at * D + 4 * h;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u)
          *reinterpret_cast<float4*>(dst + 32 * i + 8 * u) =
              make_float4(st.acc[i][4 * u], st.acc[i][4 * u + 1], st.acc[i][4 * u + 2], st.acc[i][4 * u + 3]);
      if (h == 0) *reinterpret_cast<float2*>(p.ws2 + 2 * at) = make_float2(st.m, l);
    }
  } else {
    // the waves' shares: o_w relative to m_w, joined at the common maximum
    if (h == 0) { sm[wave][n] = st.m; sl[wave][n] = l; }
    __syncthreads();
    float* so = reinterpret_cast<float*>(buf) + wave * 32 * OP;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = st.acc[i][4 * u + e];
        *reinterpret_cast<f32x4*>(so + n * OP + 32 * i + 8 * u + 4 * h) = x;
      }
    __syncthreads();
    constexpr int TPR = 64 * NW / 32, DP = D / TPR;                       // threads a row, values a thread
    const int rr = threadIdx.x / TPR, part = threadIdx.x % TPR, gr = rt * 32 + rr;
    if (gr >= R) return;
    float mx = sm[0][rr];
#pragma unroll
    for (int w = 1; w < NW; ++w) mx = fmaxf(mx, sm[w][rr]);
    float ls = 0.f, o[DP];
#pragma unroll
    for (int e = 0; e < DP; ++e) o[e] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float a = join_factor(sm[w][rr], sl[w][rr], mx, p.c);
      const float* src = reinterpret_cast<float*>(buf) + (w * 32 + rr) * OP + part * DP;
      ls += a * sl[w][rr];
#pragma unroll
      for (int e = 0; e < DP; ++e) o[e] += a * src[e];
    }
    const int gi = gr / p.G, gh = hk * p.G + gr % p.G;
    const float inv = ls > 0.f || ls != ls ? 1.f / ls : 0.f;
    bf16* dst = p.out + b * p.sob + gi * p.sol + gh * p.soh + part * DP;
#pragma unroll
    for (int e = 0; e < DP; e += 4) {
      bf16x4 x;
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = to16<F16>(o[e + k] * inv);
      *reinterpret_cast<bf16x4*>(dst + e) = x;
    }
    if (part == 0) p.lse[((long long)b * p.H + gh) * p.Lq + gi] = ls == 0.f ? -INFINITY : mx * p.scale + __logf(ls);
  }
}

// A row a workgroup: D / 4 threads a split, the splits in turn over the groups of threads, the groups joined in LDS
template <int D, bool F16>
__global__ void __launch_bounds__(256) attn_join_kernel(AttnP p) {
  constexpr int TPR = D / 4, GR = 256 / TPR;
  __shared__ float sa[256];
  __shared__ f32x4 so[GR][TPR];
  __shared__ float sl[GR];
  const long long rows = (long long)p.B * p.H * p.Lq, row = blockIdx.x;
  const int g = threadIdx.x / TPR, part = threadIdx.x % TPR;
  // the common maximum, then each split's factor, 256 splits at a time
  float mx = -INFINITY;
  for (int s = threadIdx.x; s < p.nsplit; s += 256) mx = fmaxf(mx, p.ws2[2 * (s * rows + row)]);
  mx = wave_max(mx);
  if ((threadIdx.x & 63) == 0) sa[threadIdx.x >> 6] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(sa[0], sa[1]), fmaxf(sa[2], sa[3]));
  float ls = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (int c0 = 0; c0 < p.nsplit; c0 += 256) {
    const int n = min(256, p.nsplit - c0);
    __syncthreads();
    if ((int)threadIdx.x < n) {
      const float2 ml = *reinterpret_cast<const float2*>(p.ws2 + 2 * ((c0 + threadIdx.x) * rows + row));
      const float a = join_factor(ml.x, ml.y, mx, p.c);
      sa[threadIdx.x] = a;
      ls += a * ml.y;
    }
    __syncthreads();
    if (g < GR) {
#pragma unroll 8
      for (int s = g; s < n; s += GR) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(p.ws + ((c0 + s) * rows + row) * D + 4 * part);
        o += sa[s] * x;
      }
    }
  }
  ls = wave_sum(ls);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sl[threadIdx.x >> 6] = ls;
  if (g < GR) so[g][part] = o;
  __syncthreads();
  if (threadIdx.x >= TPR) return;
  ls = (sl[0] + sl[1]) + (sl[2] + sl[3]);
  for (int k = 1; k < GR; ++k) o += so[k][part];
  const float inv = ls > 0.f || ls != ls ? 1.f / ls : 0.f;
  const int qi = row % p.Lq, hq = (row / p.Lq) % p.H;
  const long long b = row / p.Lq / p.H;
  bf16x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = to16<F16>(o[e] * inv);
  *reinterpret_cast<bf16x4*>(p.out + b * p.sob + qi * p.sol + hq * p.soh + 4 * part) = y;
  if (part == 0) p.lse[row] = ls == 0.f ? -INFINITY : mx * p.scale + __logf(ls);
}

}  // namespace

// ------------------------------------------------------------------------------------------- host side
int attn_check(const LrceAttnDesc* d, const char* what) {
  if (!d) return lrce_fail(LRCE_E_ARG, "%s: null descriptor", what);
  if (d->B < 0 || d->H < 1 || d->Hk < 1 || d->Lq < 0 || d->Lk < 0) return lrce_fail(LRCE_E_ARG, "%s: bad sizes B=%d H=%d Hk=%d Lq=%d Lk=%d", what, d->B, d->H, d->Hk, d->Lq, d->Lk);
  if (d->H % d->Hk) return lrce_fail(LRCE_E_ARG, "%s: %d query heads over %d key heads", what, d->H, d->Hk);
  if (d->D != 32 && d->D != 64 && d->D != 96 && d->D != 128) return lrce_fail(LRCE_E_ARG, "%s: head dim %d (32, 64, 96 or 128)", what, d->D);
  if (!(d->scale > 0.f) || !std::isfinite(d->scale)) return lrce_fail(LRCE_E_ARG, "%s: scale must be positive and finite", what);
  if (d->key_mask && d->mask_bytes != 1 && d->mask_bytes != 4 && d->mask_bytes != 8) return lrce_fail(LRCE_E_ARG, "%s: key mask entries of %d bytes (1, 4 or 8)", what, d->mask_bytes);
  if (d->B > 0 && d->Lq > 0 && (!d->q || !d->out || !d->lse)) return lrce_fail(LRCE_E_ARG, "%s: null pointer", what);
  if (d->B > 0 && d->Lk > 0 && (!d->k || !d->v)) return lrce_fail(LRCE_E_ARG, "%s: null pointer", what);
  const int64_t* st[] = {d->q_stride, d->k_stride, d->v_stride, d->o_stride};
  const void* at[] = {d->q, d->k, d->v, d->out};
  for (int i = 0; i < 4; ++i) {
    if (reinterpret_cast<uintptr_t>(at[i]) % 16) return lrce_fail(LRCE_E_ARG, "%s: tensors must start at multiples of 16 bytes", what);
    for (int k = 0; k < 3; ++k)
      if (st[i][k] % 8 || st[i][k] < 0) return lrce_fail(LRCE_E_ARG, "%s: strides must be multiples of 8 elements", what);
  }
  // rows are addressed by 32-bit byte offsets inside a tile of 64
  if (std::max(std::max(d->k_stride[1], d->v_stride[1]), d->q_stride[1]) >= (1ll << 23)) return lrce_fail(LRCE_E_ARG, "%s: a row stride of 2^23 elements or more", what);
  if ((int64_t)d->Lq + d->Lk >= (1ll << 30)) return lrce_fail(LRCE_E_ARG, "%s: too long", what);
  if ((int64_t)d->B * d->H * ((d->Lq + 31) / 32) >= (1ll << 31) || (int64_t)d->B * d->H * ((d->Lk + 31) / 32) >= (1ll << 31) ||
      (int64_t)d->Lq * d->H >= (1ll << 31))
    return lrce_fail(LRCE_E_ARG, "%s: too many rows", what);
  return LRCE_OK;
}

void attn_fill(const LrceAttnDesc* d, AttnP& p) {
  p = AttnP{};
  p.q = static_cast<const bf16*>(d->q); p.k = static_cast<const bf16*>(d->k); p.v = static_cast<const bf16*>(d->v);
  p.out = static_cast<bf16*>(d->out);
  p.lse = d->lse;
  p.mask = d->key_mask;
  p.smb = d->mask_stride; p.mask_bytes = d->mask_bytes;
  p.sqb = d->q_stride[0]; p.sql = d->q_stride[1]; p.sqh = d->q_stride[2];
  p.skb = d->k_stride[0]; p.skl = d->k_stride[1]; p.skh = d->k_stride[2];
  p.svb = d->v_stride[0]; p.svl = d->v_stride[1]; p.svh = d->v_stride[2];
  p.sob = d->o_stride[0]; p.sol = d->o_stride[1]; p.soh = d->o_stride[2];
  p.B = d->B; p.H = d->H; p.Hk = d->Hk; p.G = d->H / d->Hk; p.Lq = d->Lq; p.Lk = d->Lk;
  p.causal = d->causal; p.off = d->Lk - d->Lq;
  p.scale = d->scale; p.c = d->scale * ATTN_LOG2E;
  p.dout = static_cast<const bf16*>(d->dout);
  p.dq = static_cast<bf16*>(d->dq); p.dk = static_cast<bf16*>(d->dk); p.dv = static_cast<bf16*>(d->dv);
  p.sgb = d->g_stride[0]; p.sgl = d->g_stride[1]; p.sgh = d->g_stride[2];
  p.dqb = d->dq_stride[0]; p.dql = d->dq_stride[1]; p.dqh = d->dq_stride[2];
  p.dkb = d->dk_stride[0]; p.dkl = d->dk_stride[1]; p.dkh = d->dk_stride[2];
  p.dvb = d->dv_stride[0]; p.dvl = d->dv_stride[1]; p.dvh = d->dv_stride[2];
}

namespace {

struct FwdPlan {
  bool split;
  int waves;                 // of a workgroup
  int nblk, nsplit, split_tiles;
  int64_t grid, ws;
};

FwdPlan fwd_plan(const LrceAttnDesc* d) {
  FwdPlan f{};
  const int G = d->H / d->Hk;
  const int64_t rows = (int64_t)d->Lq * G;
  f.waves = d->Lq <= 64 ? 2 : 4;
  f.nblk = (d->Lq + 32 * f.waves - 1) / (32 * f.waves);
  f.grid = (int64_t)d->B * d->H * f.nblk;
  f.nsplit = 1;
  const int nt = (d->Lk + 31) / 32;
  const int64_t tiles = (int64_t)d->B * d->Hk * ((rows + 31) / 32);
  f.split = rows <= 32 || attn_few_rows(tiles, d->Lk, d->D, false);
  if (f.split) {
    f.nblk = (int)((rows + 31) / 32);
    const int64_t base = std::max<int64_t>(1, tiles);
    f.waves = attn_share_waves(d->D, base);
    f.split_tiles = std::max(2, (nt + 1) / 2 * 2);
    // one-wave shares of at least 16 tiles, about two and a half times as many as are resident (LDS: two stages of K and V), where
    // they cut the keys finer than the waves of one workgroup would and the join has few rows (7 heads x 1468 x 1468 d 32: 56 us in
    // two shares, 37 of them the join, 14 by four waves; 8 x 8 heads on 2, 16 rows, 4096 keys d 128: 26 and 38 us; 32 x 32 heads on 8,
    // one row, d 128: 147 and 174 us over up to 8190 keys).  It is set for caches of different fill; the mask is not looked at, and
    // where all caches are full, masked or not, the last takes 196 - 201 us, 180 by four waves.  B H Lq <= Lk is where the first of
    // these is told from the others: the join reads that many rows a share
    const int64_t resident = 256 * std::min<int64_t>(8, 160 * 1024 / (256 * d->D + 512));
    const int n = (int)std::max<int64_t>(1, std::min<int64_t>((5 * resident / 2 + base - 1) / base, nt / 16));
    if (nt > 32 && base < 512 && n > f.waves && (int64_t)d->B * d->H * d->Lq <= d->Lk) {
      f.waves = 1;
      f.split_tiles = ((nt + n - 1) / n + 1) / 2 * 2;
      f.nsplit = (nt + f.split_tiles - 1) / f.split_tiles;
      f.ws = (int64_t)f.nsplit * d->B * d->H * d->Lq * (d->D + 2);
    }
    f.grid = base * f.nsplit;
  }
  return f;
}

template <int D, bool F16>
void fwd_launch(const AttnP& p, const FwdPlan& f, hipStream_t s) {
  if (f.split) {
    if (f.waves == 4) {
      attn_split_kernel<D, F16, 4><<<(unsigned)f.grid, 256, 0, s>>>(p);
    } else if (f.waves == 2) {
      attn_split_kernel<D, F16, 2><<<(unsigned)f.grid, 128, 0, s>>>(p);
    } else {
      attn_split_kernel<D, F16, 1><<<(unsigned)f.grid, 64, 0, s>>>(p);
      attn_join_kernel<D, F16><<<(unsigned)((int64_t)p.B * p.H * p.Lq), 256, 0, s>>>(p);
    }
  } else if (f.waves == 2) {
    if (p.mask) attn_fwd_kernel<D, F16, 2, true><<<(unsigned)f.grid, 128, 0, s>>>(p);
    else attn_fwd_kernel<D, F16, 2, false><<<(unsigned)f.grid, 128, 0, s>>>(p);
  } else {
    if (p.mask) attn_fwd_kernel<D, F16, 4, true><<<(unsigned)f.grid, 256, 0, s>>>(p);
    else attn_fwd_kernel<D, F16, 4, false><<<(unsigned)f.grid, 256, 0, s>>>(p);
  }
}

}  // namespace

extern "C" int64_t lrce_attn_fwd_workspace(const LrceAttnDesc* d) {
  if (attn_check(d, "attn_fwd_workspace") != LRCE_OK) return -1;
  return d->B && d->Lq ? fwd_plan(d).ws : 0;
}

extern "C" int lrce_attn_fwd(const LrceAttnDesc* d, void* stream) {
  if (const int rc = attn_check(d, "attn_fwd")) return rc;
  if (d->B == 0 || d->Lq == 0) return LRCE_OK;
  const FwdPlan f = fwd_plan(d);
  if (f.grid >= (1ll << 31)) return lrce_fail(LRCE_E_ARG, "attn_fwd: too many rows");
  if (f.ws && (!d->workspace || d->workspace_elems < f.ws)) return lrce_fail(LRCE_E_ARG, "attn_fwd: a workspace of %lld floats is needed", (long long)f.ws);
  AttnP p;
  attn_fill(d, p);
  p.nblk = f.nblk; p.nsplit = f.nsplit; p.split_tiles = f.split_tiles;
  p.ws = d->workspace;
  if (f.ws) p.ws2 = p.ws + (int64_t)f.nsplit * d->B * d->H * d->Lq * d->D;
  hipStream_t s = static_cast<hipStream_t>(stream);
#define LRCE_ATTN_D(N) \
  case N: \
    if (d->f16) fwd_launch<N, true>(p, f, s); \
    else fwd_launch<N, false>(p, f, s); \
    break;
  switch (d->D) {
    LRCE_ATTN_D(32)
    LRCE_ATTN_D(64)
    LRCE_ATTN_D(96)
    LRCE_ATTN_D(128)
  }
#undef LRCE_ATTN_D
  return lrce_check_launch("attn_fwd");
}
