// Backward of the attention in attention.hip: the weights are recomputed from q, k and the saved log-sum-exp.
//
//   p_ij = exp(s_ij - lse_i),  delta_i = do_i . o_i,  ds_ij = p_ij (do_i . v_j - delta_i)
//   dv_j = sum_i p_ij do_i,  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i   (dk, dv: over the heads that share them)
//
// Two kernels (short axes: one, attn_bwd_short_kernel), each the only writer of what it sums, so there are no atomics and the
// result does not depend on timing:
// attn_dq_kernel has 32 queries a wave and walks the keys (three products; it also leaves lse in base 2 and delta for the
// other), attn_dkv_kernel has 32 keys a wave and walks the queries of all heads that share them (four products).  The
// scores are computed twice that way (7 products instead of 5), the price of having no read-modify-write of dq in memory.
// p and ds are rounded to 16 bits where they become operands (the matrix instructions that take f32 have a sixteenth of the
// rate); delta and ds are formed in f32.  With the forward's rounded weights this makes the gradients' error 1.4 times what f32
// weights leave.  In fp16 a ds above 65504 becomes infinite and one below 2^-25 is lost: the loss scale has to leave
// p |dout . v - delta| between.
// Measured: 2 x 16 heads on 4, 4096 x 4096 causal, d 128, bf16: 516 - 553 us as the clock under matrix load goes, of it dq 204 - 226 (3
// products, 910 - 1010 TFLOP/s), dk and dv 301 - 347 + 14 (4 products, 790 - 910; accumulators and operands of d 128 leave one wave a
// SIMD, so LDS reads and exponentials are not covered: the matrix pipe is busy 41 % of the cycles, 58 % in dq); 48 heads x 1568^2,
// d 32: 47 + 56 us, the vector unit.  Two waves for 32 keys, one with dv, one with dk, the weights handed over in LDS: the same at
// d 128 (514 against 518 us of backward, both in turn), slower below (d 64 533 against 493).
#include <algorithm>

#include "attention_util.h"

namespace {

// A wave's 32 query rows
template <int D, bool F16>
struct DqRow {
  bf16x8 q[D / 16], g[D / 16];
  float delta, lse2;
  __device__ __forceinline__ void init(const AttnP& p, int b, int hq, int bh, int i0, int row, bool valid, int lane, int h, bool tell) {
    const bf16* qr = p.q + b * p.sqb + row * p.sql + hq * p.sqh;
    const bf16* gr = p.dout + b * p.sgb + row * p.sgl + hq * p.sgh;
    const bf16* orow = p.out + b * p.sob + row * p.sol + hq * p.soh;
    bf16x8 o[D / 16];
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      q[kk] = *reinterpret_cast<const bf16x8*>(qr + 16 * kk + 8 * h);
      g[kk] = *reinterpret_cast<const bf16x8*>(gr + 16 * kk + 8 * h);
      o[kk] = *reinterpret_cast<const bf16x8*>(orow + 16 * kk + 8 * h);
    }
    const float lse = p.lse[(long long)bh * p.Lq + row];
    delta = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = __builtin_fmaf(from16<F16>(g[kk][j]), from16<F16>(o[kk][j]), delta);
    attn_landed(q);
    attn_landed(g);
    delta += other_half(delta);
    // a row that sees no key has lse = -inf and p = exp(s - inf) = 0; so have the rows behind the last
    lse2 = !valid || lse == -INFINITY ? INFINITY : lse * ATTN_LOG2E;
    const int nst = (p.Lq + 63) / 64 * 2;                                // 32-row blocks of statistics
    if (tell && i0 / 32 < nst) p.ws[((long long)bh * nst + i0 / 32) * 64 + lane] = h ? (valid ? delta : 0.f) : lse2;
    // the block that makes their number even
    if (tell && i0 / 32 == nst - 2 && i0 + 32 >= p.Lq) p.ws[((long long)bh * nst + nst - 1) * 64 + lane] = h ? 0.f : INFINITY;
  }
  // the 32 keys from row r0 of the tiles on: weights and dout . v (bit of ws = key there and not hidden, ls = the last key of the
  // block that the wave's first row sees; hidden pairs have weight 0)
  __device__ __forceinline__ void pairs(const AttnP& p, const TileRead<D>& rd, lds_cptr kt, lds_cptr vt, int r0, uint32_t ws, int ls, int n,
                                        int h, f32x16& s, f32x16& dp) const {
    s = mfma32x32x16<F16>(rd.row(kt, r0, 0), q[0], f32x16{});
    dp = mfma32x32x16<F16>(rd.row(vt, r0, 0), g[0], f32x16{});
#pragma unroll
    for (int kk = 1; kk < D / 16; ++kk) s = mfma32x32x16<F16>(rd.row(kt, r0, kk), q[kk], s);
#pragma unroll
    for (int kk = 1; kk < D / 16; ++kk) dp = mfma32x32x16<F16>(rd.row(vt, r0, kk), g[kk], dp);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.c, -lse2));
    const bool diag = p.causal && ls < 31;
    if (diag || ws != ~0u) {
      const uint32_t kw = (ws & (diag ? upto(ls + n) : ~0u)) >> (4 * h);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = (kw >> ((r & 3) + 8 * (r >> 2))) & 1 ? s[r] : 0.f;
    }
  }
  __device__ __forceinline__ void sum(const TileRead<D>& rd, lds_cptr kt, int r0, f32x16& s, const f32x16& dp, f32x16 (&acc)[D / 32]) const {
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] *= dp[r] - delta;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const bf16x8 f = attn_pack<F16>(s, half);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) acc[i] = mfma32x32x16<F16>(rd.col(kt, r0 + 16 * half, i), f, acc[i]);
    }
  }
  __device__ __forceinline__ void block(const AttnP& p, const TileRead<D>& rd, lds_cptr kt, lds_cptr vt, int r0, uint32_t ws, int ls, int n,
                                        int h, f32x16 (&acc)[D / 32]) const {
    f32x16 s, dp;
    pairs(p, rd, kt, vt, r0, ws, ls, n, h, s, dp);
    sum(rd, kt, r0, s, dp, acc);
  }
  // All that the rows see, in at most two blocks (at kt, vt and kt + step, vt + step): delta is the sum of weight times dout . v,
  // from a first walk over them.  The one from out would carry out's rounding to 16 bits, which counts where a few weights
  // are large (it falls off as 1 / keys).
  __device__ __forceinline__ void few(const AttnP& p, const TileRead<D>& rd, lds_cptr kt, lds_cptr vt, int step, uint32_t w0, int l0, uint32_t w1,
                                      int l1, int bh, int i0, bool valid, int lane, int h) {
    float d = 0.f;
#pragma unroll 1
    for (int x = 0; x < 2; ++x) {
      const uint32_t w = x ? w1 : w0;
      if (w == 0) continue;
      f32x16 s, dp;
      pairs(p, rd, kt + x * step, vt + x * step, 0, w, x ? l1 : l0, lane & 31, h, s, dp);
#pragma unroll
      for (int r = 0; r < 16; ++r) d = __builtin_fmaf(s[r], dp[r], d);
    }
    delta = d + other_half(d);
    if (h && valid) p.ws[((long long)bh * ((p.Lq + 63) / 64 * 2) + i0 / 32) * 64 + lane] = delta;
  }
};

template <int D, bool F16, int NW>
__global__ void __launch_bounds__(NW * 64, 2) attn_dq_kernel(AttnP p) {
  constexpr int KT = 64, TB = KT * D * 2;
  typedef TileStage<D, KT, NW> Stage;
  __shared__ __attribute__((aligned(1024))) char buf[4 * TB];
  __shared__ uint64_t words[ATTN_MASK_KEYS / KT];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const Place at = attn_place(p, p.G);
  const int blk = p.nblk - 1 - at.blk, b = at.b, hq = at.hq, hk = hq / p.G, bh = b * p.H + hq;
  const int i0 = blk * (32 * NW) + wave * 32;
  const bool valid = i0 + n < p.Lq;
  const int row = min(i0 + n, p.Lq - 1);
  const int last = min(blk * (32 * NW) + 32 * NW, p.Lq) - 1;
  const int nk = p.causal ? max(0, min(p.Lk, last + p.off + 1)) : p.Lk;
  const int nt = (nk + KT - 1) / KT;
  const int tw = p.causal ? min(nt, max(0, i0 + 31 + p.off + KT) / KT) : nt;   // tiles from tw on hold no key that this wave's rows see

  DqRow<D, F16> rw;
  rw.init(p, b, hq, bh, i0, row, valid, lane, h, true);

  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
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
  const int chunk = p.mask ? ATTN_MASK_KEYS / KT : nt;
  for (int c0 = 0; c0 < nt; c0 += chunk) {
    const int c1 = min(nt, c0 + chunk);
    if (p.mask) {
      __syncthreads();
      attn_pack_mask<NW>(p, b, c0, c1 - c0, lw, lane, wave);
      __syncthreads();
    }
    auto word = [&](int t) { return p.mask ? uni64(lw[t - c0]) : low_bits(p.Lk - t * KT); };
    auto next = [&](int t, uint64_t& w) {
      for (; t < c1; ++t)
        if ((w = word(t)) != 0) break;
      return t;
    };
    auto stage = [&](int t, uint64_t w, int cur) {
      const char *ka = kb + t * kstep, *va = vb + t * vstep;
      const uint32_t kd = attn_lds_u32(lds + 2 * cur * TB), vd = attn_lds_u32(lds + (2 * cur + 1) * TB);
      const int n = p.Lk - t * KT;
      if (p.mask && w != ~0ull) {
        sk.load(ka, n, w, kd, lane, wave);
        sv.load(va, n, w, vd, lane, wave);
      } else {
        sk.load(ka, n, kd, wave);
        sv.load(va, n, vd, wave);
      }
    };
    uint64_t w = 0, wn = 0;
    int t = next(c0, w), cur = 0;
    const int t_end = min(c1, tw);
    bool only = c0 == 0 && (c1 == nt || tw <= c1);                       // (until a second tile is found) the rows' keys lie in one tile
    if (t < c1) stage(t, w, 0);
    while (t < c1) {
      attn_barrier();
      const int tn = next(t + 1, wn);
      if (tn < c1) stage(tn, wn, cur ^ 1);
      const int lim = i0 + p.off - t * KT;
      lds_cptr kt = lds + 2 * cur * TB, vt = lds + (2 * cur + 1) * TB;
      only = only && tn >= t_end;
      if (only && t < t_end)
        rw.few(p, rd, kt, vt, TB / 2, (uint32_t)w, lim, p.causal && lim < 1 ? 0u : (uint32_t)(w >> 32), lim - 32, bh, i0, valid, lane, h);
#pragma unroll
      for (int sub = 0; sub < 2; ++sub) {
        const int ls = lim - 32 * sub;                                   // the wave's first row sees keys up to ls of the block
        const uint32_t ws = (uint32_t)(w >> (32 * sub));
        if (ws == 0 || (p.causal && ls + 31 < 0)) continue;
        rw.block(p, rd, kt, vt, 32 * sub, ws, ls, n, h, acc);
      }
      t = tn;
      w = wn;
      cur ^= 1;
    }
  }
  bf16* o = p.dq + b * p.dqb + row * p.dql + hq * p.dqh;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) attn_store<F16>(acc[i], p.scale, o + 32 * i, h, valid);
}

// The same for few rows: the waves of a workgroup have one tile of 32 rows between them, wave w every NW-th key tile of 32,
// and their sums are added in LDS
template <int D, bool F16, int NW>
__global__ void __launch_bounds__(64 * NW, D <= 64 ? 2 : 1) attn_dq_share_kernel(AttnP p) {
  constexpr int KT = 32, TB = KT * D * 2;
  typedef TileStage<D, KT, 1> Stage;
  constexpr int OP = D + 4;
  constexpr int SZ = NW * 32 * OP * 4 > NW * 4 * TB ? NW * 32 * OP * 4 : NW * 4 * TB;
  __shared__ __attribute__((aligned(1024))) char buf[SZ];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const Place at = attn_place(p, p.G);
  const int blk = p.nblk - 1 - at.blk, b = at.b, hq = at.hq, hk = hq / p.G, bh = b * p.H + hq;
  const int i0 = blk * 32;
  const bool valid = i0 + n < p.Lq;
  const int row = min(i0 + n, p.Lq - 1);
  const int nk = p.causal ? max(0, min(p.Lk, min(i0 + 31, p.Lq - 1) + p.off + 1)) : p.Lk;
  const int nt = (nk + KT - 1) / KT;
  DqRow<D, F16> rw;
  rw.init(p, b, hq, bh, i0, row, valid, lane, h, wave == 0);
  f32x16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  TileRead<D> rd;
  rd.init(lane);
  Stage sk, sv;
  sk.init(lane, 0, p.skl);
  sv.init(lane, 0, p.svl);
  const char* kb = uni(p.k + b * p.skb + hk * p.skh);
  const char* vb = uni(p.v + b * p.svb + hk * p.svh);
  const long long kstep = p.skl * (2 * KT), vstep = p.svl * (2 * KT);
  lds_ptr lds = (lds_ptr)buf + wave * (4 * TB);
  const int chunk = p.mask ? 128 : max(nt, 1);
  for (int c0 = 0; c0 < nt; c0 += chunk) {
    const int c1 = min(nt, c0 + chunk);
    uint32_t mlo = 0, mhi = 0;
    if (p.mask)
      attn_mask_words<1>(p, b, c0 / 2, (c1 + 1) / 2, lane, [&](int w, uint64_t bits) {
        if (lane == w - c0 / 2) { mlo = (uint32_t)bits; mhi = (uint32_t)(bits >> 32); }
      });
    // few visible tiles: the first wave has them all
    const int seen = p.mask ? __popcll(__ballot(mlo != 0)) + __popcll(__ballot(mhi != 0)) : nt;
    const bool few = nt <= chunk && seen <= 2;
    const int step = few ? 1 : NW;
    auto next = [&](int t, uint32_t& w) {
      for (; t < c1; t += step) {
        w = p.mask ? (uint32_t)__builtin_amdgcn_readlane(((t - c0) & 1) ? mhi : mlo, (t - c0) >> 1) : (uint32_t)low_bits(p.Lk - t * KT);
        if (w != 0) break;
      }
      return t;
    };
    auto stage = [&](int t, uint32_t w, int cur) {
      const char *ka = kb + t * kstep, *va = vb + t * vstep;
      const uint32_t kd = attn_lds_u32(lds + 2 * cur * TB), vd = attn_lds_u32(lds + (2 * cur + 1) * TB);
      const int m = p.Lk - t * KT;
      if (p.mask && w != ~0u) {
        sk.load(ka, m, w, kd, lane, 0);
        sv.load(va, m, w, vd, lane, 0);
      } else {
        sk.load(ka, m, kd, 0);
        sv.load(va, m, vd, 0);
      }
    };
    uint32_t w0 = 0, w1 = 0, w2 = 0;
    int cur = 0;
    int t0 = few && wave ? c1 : next(wave + c0, w0);
    if (t0 < c1) stage(t0, w0, 0);
    int t1 = next(t0 + step, w1);
    if (t1 < c1) stage(t1, w1, 1);
    if (few && t0 < c1) {
      attn_wait_vm<0>();
      rw.few(p, rd, lds, lds + TB, 2 * TB, w0, i0 + p.off - t0 * KT, t1 < c1 ? w1 : 0u, i0 + p.off - t1 * KT, bh, i0, valid, lane, h);
    }
    while (t0 < c1) {
      if (t1 < c1) attn_wait_vm<2 * Stage::NI>();
      else attn_wait_vm<0>();
      rw.block(p, rd, lds + 2 * cur * TB, lds + (2 * cur + 1) * TB, 0, w0, i0 + p.off - t0 * KT, n, h, acc);
      const int t2 = next(t1 + step, w2);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                 // the tile's reads are done: its place may be filled
      if (t2 < c1) stage(t2, w2, cur);
      t0 = t1; w0 = w1;
      t1 = t2; w1 = w2;
      cur ^= 1;
    }
  }
  __syncthreads();
  float* so = reinterpret_cast<float*>(buf) + wave * 32 * OP;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      f32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = acc[i][4 * u + e];
      *reinterpret_cast<f32x4*>(so + n * OP + 32 * i + 8 * u + 4 * h) = x;
    }
  __syncthreads();
  constexpr int TPR = 64 * NW / 32, DP = D / TPR;
  const int rr = threadIdx.x / TPR, part = threadIdx.x % TPR;
  if (i0 + rr >= p.Lq) return;
  bf16* dst = p.dq + b * p.dqb + (long long)(i0 + rr) * p.dql + hq * p.dqh + part * DP;
#pragma unroll
  for (int e = 0; e < DP; e += 4) {
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < NW; ++w) o += *reinterpret_cast<const f32x4*>(reinterpret_cast<float*>(buf) + (w * 32 + rr) * OP + part * DP + e);
    bf16x4 x;
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = to16<F16>(o[k] * p.scale);
    *reinterpret_cast<bf16x4*>(dst + e) = x;
  }
}

// Query tiles of 64 rows (two blocks of 32) of one head at a time; the heads of the group one after the other.  With
// p.nsplit > 1 a workgroup has its share of the (head, tile) list and leaves f32 sums that attn_dkv_sum_kernel adds in order.
template <int D, bool F16, int NW>
__global__ void __launch_bounds__(NW * 64, D <= 96 ? 2 : 1) attn_dkv_kernel(AttnP p) {
  constexpr int QT = 64, TB = QT * D * 2, SB = 1024;
  typedef TileStage<D, QT, NW> Stage;
  __shared__ __attribute__((aligned(1024))) char buf[4 * TB + 2 * SB];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const Place place = attn_place(p, p.nsplit);                           // (the splits take the place of the group's heads)
  const int blk = place.blk, b = place.b, hk = place.hq / p.nsplit, sp = place.hq % p.nsplit, bk = b * p.Hk + hk;
  const int j0 = blk * (32 * NW) + wave * 32, jw = blk * (32 * NW);
  const int j = j0 + n;
  bool keep = j < p.Lk;
  if (keep && p.mask) {
    const long long at = (long long)b * p.smb + j;
    keep = p.mask_bytes == 1 ? static_cast<const uint8_t*>(p.mask)[at] != 0
         : p.mask_bytes == 4 ? static_cast<const int*>(p.mask)[at] != 0 : static_cast<const long long*>(p.mask)[at] != 0;
  }
  const bool some = __any(keep), allk = __all(keep);
  const bool work = __syncthreads_or(some);

  f32x16 dk[D / 32], dv[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) { dk[i][r] = 0.f; dv[i][r] = 0.f; }

  TileRead<D> rd;
  rd.init(lane);
  Stage sq, sg;
  sq.init(lane, wave, p.sql);
  sg.init(lane, wave, p.sgl);
  lds_ptr lds = (lds_ptr)buf;
  const int nq = (p.Lq + QT - 1) / QT, nst = nq * 2;
  const int tf = p.causal ? min(nq, max(0, jw - p.off) / QT) : 0;          // the first tile with a row that sees key jw
  const int per = nq - tf;
  const long long total = work ? (long long)p.G * per : 0;
  const int e0 = (int)(total * sp / p.nsplit), e1 = (int)(total * (sp + 1) / p.nsplit);
  int hs = per ? e0 / per : 0, ts = tf + (per ? e0 % per : 0);          // the tile being staged
  auto stage = [&](int cur) {
    const int hq = hk * p.G + hs;
    const int rows = p.Lq - ts * QT;
    const char* qb = uni(p.q + b * p.sqb + hq * p.sqh + (long long)ts * QT * p.sql);
    const char* gb = uni(p.dout + b * p.sgb + hq * p.sgh + (long long)ts * QT * p.sgl);
    sq.load(qb, rows, attn_lds_u32(lds + 2 * cur * TB), wave);
    sg.load(gb, rows, attn_lds_u32(lds + (2 * cur + 1) * TB), wave);
    if (wave == 0) {
      const uint32_t o = lane * 16;
      attn_glds<1, 0>(attn_rsrc(uni(p.ws + (((long long)b * p.H + hq) * nst + 2 * ts) * 64), 512), &o, attn_lds_u32(lds + 4 * TB + cur * SB));
    }
    if (++ts == nq) { ts = tf; ++hs; }
  };
  int cur = 0, tc = ts;
  if (e0 < e1) stage(0);
  bf16x8 kf[D / 16], vf[D / 16];
  {
    const long long jr = min(j, p.Lk - 1);
    const bf16* kr = p.k + b * p.skb + jr * p.skl + hk * p.skh;
    const bf16* vr = p.v + b * p.svb + jr * p.svl + hk * p.svh;
    const bf16x8 zero = {};
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      kf[kk] = keep ? *reinterpret_cast<const bf16x8*>(kr + 16 * kk + 8 * h) : zero;
      vf[kk] = keep ? *reinterpret_cast<const bf16x8*>(vr + 16 * kk + 8 * h) : zero;
    }
    attn_landed(kf);
    attn_landed(vf);
  }
  for (int e = e0; e < e1; ++e) {
    attn_barrier();
    if (e + 1 < e1) stage(cur ^ 1);
    lds_cptr qt = lds + 2 * cur * TB, gt = lds + (2 * cur + 1) * TB, stt = lds + 4 * TB + cur * SB;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const int i0 = tc * QT + 32 * sub;
      const int lim = j0 - p.off - i0;                                   // row i0 + r sees the wave's first key from r = lim on
      if (!some || i0 >= p.Lq || (p.causal && lim > 31)) continue;
      f32x16 s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) s = mfma32x32x16<F16>(rd.row(qt, 32 * sub, kk), kf[kk], s);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) dp = mfma32x32x16<F16>(rd.row(gt, 32 * sub, kk), vf[kk], dp);
      const LRCE_LDS float* sl = (const LRCE_LDS float*)(stt + sub * 256) + 4 * h;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x4 l4 = *reinterpret_cast<const LRCE_LDS f32x4*>(sl + 8 * u);
#pragma unroll
        for (int x = 0; x < 4; ++x) s[4 * u + x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * u + x], p.c, -l4[x]));
      }
      if (!allk || (p.causal && lim + 31 > 0)) {
        const int first = p.causal ? lim + n : -64;                      // rows r >= first see this lane's key
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = keep && crow32(r, h) >= first ? s[r] : 0.f;
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const f32x4 d4 = *reinterpret_cast<const LRCE_LDS f32x4*>(sl + 32 + 8 * u);
#pragma unroll
        for (int x = 0; x < 4; ++x) dp[4 * u + x] = s[4 * u + x] * (dp[4 * u + x] - d4[x]);
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const bf16x8 pf = attn_pack<F16>(s, half), df = attn_pack<F16>(dp, half);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dv[i] = mfma32x32x16<F16>(rd.col(gt, 32 * sub + 16 * half, i), pf, dv[i]);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) dk[i] = mfma32x32x16<F16>(rd.col(qt, 32 * sub + 16 * half, i), df, dk[i]);
      }
    }
    if (++tc == nq) tc = tf;
    cur ^= 1;
  }
  const bool valid = j < p.Lk;
  if (p.nsplit == 1) {
    bf16* ok = p.dk + b * p.dkb + (long long)j * p.dkl + hk * p.dkh;
    bf16* ov = p.dv + b * p.dvb + (long long)j * p.dvl + hk * p.dvh;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      attn_store<F16>(dk[i], p.scale, ok + 32 * i, h, valid);
      attn_store<F16>(dv[i], 1.f, ov + 32 * i, h, valid);
    }
  } else if (valid) {
    // [split][dk, dv][B Hk Lk][D]
    const long long rows = (long long)p.B * p.Hk * p.Lk, at = (long long)bk * p.Lk + j;
    float* wk = p.ws2 + (2ll * sp * rows + at) * D;
    float* wv = wk + rows * D;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        f32x4 x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[e] = dk[i][4 * u + e] * p.scale; y[e] = dv[i][4 * u + e]; }
        *reinterpret_cast<f32x4*>(wk + 32 * i + 8 * u + 4 * h) = x;
        *reinterpret_cast<f32x4*>(wv + 32 * i + 8 * u + 4 * h) = y;
      }
  }
}

// dk / dv rows: the splits' f32 sums in order, one rounding.  A thread has 4 values.
template <int D, bool F16>
__global__ void __launch_bounds__(256) attn_dkv_sum_kernel(AttnP p) {
  const long long rows = (long long)p.B * p.Hk * p.Lk, n = 2 * rows * (D / 4);
  const long long e = (long long)blockIdx.x * 256 + threadIdx.x;
  if (e >= n) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < p.nsplit; ++s) {
    const float4 x = *reinterpret_cast<const float4*>(p.ws2 + 2ll * s * rows * D + 4 * e);
    a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
  }
  const int part = e % (D / 4);
  const long long at = e / (D / 4) % rows, j = at % p.Lk, bk = at / p.Lk, b = bk / p.Hk, hk = bk % p.Hk;
  bf16* dst = e >= rows * (D / 4) ? p.dv + b * p.dvb + j * p.dvl + hk * p.dvh : p.dk + b * p.dkb + j * p.dkl + hk * p.dkh;
  bf16x4 y;
  y[0] = to16<F16>(a.x); y[1] = to16<F16>(a.y); y[2] = to16<F16>(a.z); y[3] = to16<F16>(a.w);
  *reinterpret_cast<bf16x4*>(dst + 4 * part) = y;
}

// Up to 64 queries and 64 keys: one launch, a workgroup a (batch row, key head).  Both axes lie in LDS whole; waves 0 and 1 have
// 32 queries each and form dq, waves 2 and 3 have 32 keys each and form dk and dv, over the heads of the group in turn.  The two
// roles are mirror images: rows of one's own axis in registers, the other axis from LDS.  delta is the sum of the weights times
// dout . v (the query waves', handed over in LDS), so the forward's rounded out is not read.
template <int D, bool F16>
__global__ void __launch_bounds__(256, D <= 64 ? 2 : 1) attn_bwd_short_kernel(AttnP p) {
  constexpr int TB = 64 * D * 2;
  typedef TileStage<D, 64, 4> Stage;
  __shared__ __attribute__((aligned(1024))) char buf[4 * TB];            // K, V, Q, dout
  __shared__ float sl[64], sd[64];                                       // lse in base 2 and delta of the queries
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6), h = lane >> 5, n = lane & 31;
  const int b = blockIdx.x / p.Hk, hk = blockIdx.x % p.Hk;
  const bool keys = wave >= 2;
  const int x0 = 32 * (wave & 1);                                        // this wave's first query or key
  lds_ptr lds = (lds_ptr)buf;
  Stage sk, sv, sq, sg;
  sk.init(lane, wave, p.skl);
  sv.init(lane, wave, p.svl);
  sq.init(lane, wave, p.sql);
  sg.init(lane, wave, p.sgl);
  auto fetch = [&](int g) {
    const int hq = hk * p.G + g;
    sq.load(uni(p.q + b * p.sqb + hq * p.sqh), p.Lq, attn_lds_u32(lds + 2 * TB), wave);
    sg.load(uni(p.dout + b * p.sgb + hq * p.sgh), p.Lq, attn_lds_u32(lds + 3 * TB), wave);
    if (wave == 0) {
      const float x = p.lse[((long long)b * p.H + hq) * p.Lq + min(lane, p.Lq - 1)];
      sl[lane] = lane >= p.Lq || x == -INFINITY ? INFINITY : x * ATTN_LOG2E;
    }
  };
  uint64_t w = low_bits(p.Lk);
  if (p.mask) attn_mask_words<1>(p, b, 0, 1, lane, [&](int, uint64_t bits) { w = bits; });
  w = uni64(w);
  const char* kb = uni(p.k + b * p.skb + hk * p.skh);
  const char* vb = uni(p.v + b * p.svb + hk * p.svh);
  sk.load(kb, p.Lk, w, attn_lds_u32(lds), lane, wave);
  sv.load(vb, p.Lk, w, attn_lds_u32(lds + TB), lane, wave);
  fetch(0);
  TileRead<D> rd;
  rd.init(lane);
  lds_cptr mine = lds + (keys ? 0 : 2 * TB), other = lds + (keys ? 2 * TB : 0);      // own axis, the axis that is summed over
  f32x16 da[D / 32], dv[D / 32];                                         // dq or dk, dv
  auto clear = [&](f32x16 (&x)[D / 32]) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) x[i][r] = 0.f;
  };
  clear(da);
  clear(dv);
  for (int g = 0; g < p.G; ++g) {
    if (g) {
      attn_barrier();                                                    // the head before it is done with
      fetch(g);
    }
    attn_barrier();
    bf16x8 ra[D / 16], rb[D / 16];
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      ra[kk] = rd.row(mine, x0, kk);
      rb[kk] = rd.row(mine + TB, x0, kk);
    }
    f32x16 s[2], dp[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      s[x] = mfma32x32x16<F16>(rd.row(other, 32 * x, 0), ra[0], f32x16{});
      dp[x] = mfma32x32x16<F16>(rd.row(other + TB, 32 * x, 0), rb[0], f32x16{});
#pragma unroll
      for (int kk = 1; kk < D / 16; ++kk) {
        s[x] = mfma32x32x16<F16>(rd.row(other, 32 * x, kk), ra[kk], s[x]);
        dp[x] = mfma32x32x16<F16>(rd.row(other + TB, 32 * x, kk), rb[kk], dp[x]);
      }
    }
    if (keys) {
      const bool keep = (w >> (x0 + n)) & 1;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int first = keep ? (p.causal ? x0 + n - p.off - 32 * x : -64) : 64;    // rows r >= first see this lane's key
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 l4 = *reinterpret_cast<const f32x4*>(sl + 32 * x + 8 * u + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * u + e;
            const float t = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][r], p.c, -l4[e]));
            s[x][r] = crow32(r, h) >= first ? t : 0.f;
          }
        }
      }
    } else {
      const float lse2 = sl[x0 + n];
      float d = 0.f;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const uint32_t kw = ((uint32_t)(w >> (32 * x)) & (p.causal ? upto(x0 + n + p.off - 32 * x) : ~0u)) >> (4 * h);
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float t = __builtin_amdgcn_exp2f(__builtin_fmaf(s[x][r], p.c, -lse2));
          s[x][r] = (kw >> ((r & 3) + 8 * (r >> 2))) & 1 ? t : 0.f;
          d = __builtin_fmaf(s[x][r], dp[x][r], d);
        }
      }
      d += other_half(d);
      if (h == 0) sd[x0 + n] = d;
    }
    __syncthreads();
    if (keys) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const bf16x8 pf = attn_pack<F16>(s[x], half);
#pragma unroll
          for (int i = 0; i < D / 32; ++i) dv[i] = mfma32x32x16<F16>(rd.col(other + TB, 32 * x + 16 * half, i), pf, dv[i]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const f32x4 d4 = *reinterpret_cast<const f32x4*>(sd + 32 * x + 8 * u + 4 * h);
#pragma unroll
          for (int e = 0; e < 4; ++e) s[x][4 * u + e] *= dp[x][4 * u + e] - d4[e];
        }
      }
    } else {
      const float delta = sd[x0 + n];
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[x][r] *= dp[x][r] - delta;
    }
#pragma unroll
    for (int x = 0; x < 2; ++x)
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const bf16x8 f = attn_pack<F16>(s[x], half);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) da[i] = mfma32x32x16<F16>(rd.col(other, 32 * x + 16 * half, i), f, da[i]);
      }
    if (!keys) {
      const bool valid = x0 + n < p.Lq;
      bf16* o = p.dq + b * p.dqb + (long long)(x0 + n) * p.dql + (hk * p.G + g) * p.dqh;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) attn_store<F16>(da[i], p.scale, o + 32 * i, h, valid);
      clear(da);
    }
  }
  if (keys) {
    const bool valid = x0 + n < p.Lk;
    bf16* ok = p.dk + b * p.dkb + (long long)(x0 + n) * p.dkl + hk * p.dkh;
    bf16* ov = p.dv + b * p.dvb + (long long)(x0 + n) * p.dvl + hk * p.dvh;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      attn_store<F16>(da[i], p.scale, ok + 32 * i, h, valid);
      attn_store<F16>(dv[i], 1.f, ov + 32 * i, h, valid);
    }
  }
}

struct BwdPlan {
  bool share, brief;
  int wq, wk, nbq, nbk, nsplit;
  int64_t gq, gk, stat, part;
};

BwdPlan bwd_plan(const LrceAttnDesc* d) {
  BwdPlan f{};
  // one launch for short axes; many heads on few key heads would be left to few workgroups.  Measured (64 x 64, one launch / two
  // kernels): 600 heads d 64, 40 x 40 11.3 / 15.3 us, 2400 heads d 128 91 / 120, 4 x 32 heads d 128 in groups of 8 18.7 / 20.9, in
  // groups of 32 (d 64) 67 / 23, 64 x 128 heads in groups of 16 (d 64) 63 / 112
  f.brief = d->Lq > 0 && d->Lq <= 64 && d->Lk > 0 && d->Lk <= 64 && (d->H / d->Hk <= 8 || (int64_t)d->B * d->Hk >= 512);
  if (f.brief) {
    f.gq = (int64_t)d->B * d->Hk;
    return f;
  }
  f.wq = d->Lq <= 64 ? 2 : 4;
  f.wk = d->Lk <= 64 ? 2 : 4;
  const int64_t row_tiles = (int64_t)d->B * d->H * ((d->Lq + 31) / 32);
  f.share = attn_few_rows(row_tiles, d->Lk, d->D, true);
  if (f.share) f.wq = attn_share_waves(d->D, row_tiles);
  f.nbq = f.share ? (d->Lq + 31) / 32 : (d->Lq + 32 * f.wq - 1) / (32 * f.wq);
  f.nbk = (d->Lk + 32 * f.wk - 1) / (32 * f.wk);
  f.gq = (int64_t)d->B * d->H * f.nbq;
  f.stat = (int64_t)d->B * d->H * ((d->Lq + 63) / 64) * 128;
  const int64_t base = std::max<int64_t>(1, (int64_t)d->B * d->Hk * f.nbk), tiles = (int64_t)(d->H / d->Hk) * ((d->Lq + 63) / 64);
  // dk / dv: the query axis is cut where the key blocks alone make fewer than 512 workgroups, at least 8 tiles a share (measured, 2 x
  // 4096 x 4096 d 128: 256 key blocks of 4 heads each, causal: 1 / 2 / 3 shares 702 / 516 / 543 us; 512 key blocks 466 us uncut, 518 in 2)
  f.nsplit = (int)std::max<int64_t>(1, std::min<int64_t>(512 / base, tiles / 8));
  f.gk = (int64_t)d->B * d->Hk * f.nbk * f.nsplit;
  if (f.nsplit > 1) f.part = 2ll * f.nsplit * d->B * d->Hk * d->Lk * d->D;
  return f;
}

template <int D, bool F16>
void bwd_launch(AttnP p, const BwdPlan& f, hipStream_t s) {
  if (f.brief) {
    attn_bwd_short_kernel<D, F16><<<(unsigned)f.gq, 256, 0, s>>>(p);
    return;
  }
  if (f.gq) {
    p.nblk = f.nbq;
    if (f.share && f.wq == 2) attn_dq_share_kernel<D, F16, 2><<<(unsigned)f.gq, 128, 0, s>>>(p);
    else if (f.share) attn_dq_share_kernel<D, F16, 4><<<(unsigned)f.gq, 256, 0, s>>>(p);
    else if (f.wq == 2) attn_dq_kernel<D, F16, 2><<<(unsigned)f.gq, 128, 0, s>>>(p);
    else attn_dq_kernel<D, F16, 4><<<(unsigned)f.gq, 256, 0, s>>>(p);
  }
  if (f.gk) {
    p.nblk = f.nbk;
    p.nsplit = f.nsplit;
    if (f.wk == 2) attn_dkv_kernel<D, F16, 2><<<(unsigned)f.gk, 128, 0, s>>>(p);
    else attn_dkv_kernel<D, F16, 4><<<(unsigned)f.gk, 256, 0, s>>>(p);
    if (f.nsplit > 1) {
      const int64_t n = 2ll * p.B * p.Hk * p.Lk * (D / 4);
      attn_dkv_sum_kernel<D, F16><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(p);
    }
  }
}

int bwd_check(const LrceAttnDesc* d, const char* what) {
  if (const int rc = attn_check(d, what)) return rc;
  const int64_t* st[] = {d->g_stride, d->dq_stride, d->dk_stride, d->dv_stride};
  const void* at[] = {d->dout, d->dq, d->dk, d->dv};
  for (int i = 0; i < 4; ++i) {
    if (d->B > 0 && (i < 2 ? d->Lq : d->Lk) > 0 && !at[i]) return lrce_fail(LRCE_E_ARG, "%s: null gradient pointer", what);
    if (reinterpret_cast<uintptr_t>(at[i]) % 16) return lrce_fail(LRCE_E_ARG, "%s: tensors must start at multiples of 16 bytes", what);
    for (int k = 0; k < 3; ++k)
      if (st[i][k] % 8 || st[i][k] < 0) return lrce_fail(LRCE_E_ARG, "%s: strides must be multiples of 8 elements", what);
  }
  if (d->g_stride[1] >= (1ll << 23)) return lrce_fail(LRCE_E_ARG, "%s: a row stride of 2^23 elements or more", what);
  return LRCE_OK;
}

}  // namespace

extern "C" int64_t lrce_attn_bwd_workspace(const LrceAttnDesc* d) {
  if (attn_check(d, "attn_bwd_workspace") != LRCE_OK) return -1;
  const BwdPlan f = bwd_plan(d);
  return f.stat + f.part;
}

extern "C" int lrce_attn_bwd(const LrceAttnDesc* d, void* stream) {
  if (const int rc = bwd_check(d, "attn_bwd")) return rc;
  if (d->B == 0) return LRCE_OK;
  const BwdPlan f = bwd_plan(d);
  if (f.gq >= (1ll << 31) || f.gk >= (1ll << 31) || (int64_t)d->B * d->Hk * d->Lk * (d->D / 2) >= (1ll << 38))
    return lrce_fail(LRCE_E_ARG, "attn_bwd: too many rows");
  if (f.stat + f.part && (!d->workspace || d->workspace_elems < f.stat + f.part))
    return lrce_fail(LRCE_E_ARG, "attn_bwd: a workspace of %lld floats is needed", (long long)(f.stat + f.part));
  AttnP p;
  attn_fill(d, p);
  p.ws = d->workspace;
  p.ws2 = p.ws + f.stat;
  hipStream_t s = static_cast<hipStream_t>(stream);
#define LRCE_ATTN_D(N) \
  case N: \
    if (d->f16) bwd_launch<N, true>(p, f, s); \
    else bwd_launch<N, false>(p, f, s); \
    break;
  switch (d->D) {
    LRCE_ATTN_D(32)
    LRCE_ATTN_D(64)
    LRCE_ATTN_D(96)
    LRCE_ATTN_D(128)
  }
#undef LRCE_ATTN_D
  return lrce_check_launch("attn_bwd");
}
