// Device helpers shared by the attention kernels (attention.hip: forward; attention_bwd.hip: backward).
// Internal linkage: included by each .hip.
//
// Layout facts that all of them use (wave64, v_mfma_f32_32x32x16):
//  * an accumulator tile [m][n] holds n = lane & 31 and m = (reg & 3) + 8 (reg >> 2) + 4 (lane >> 5);
//  * its registers 8s .. 8s+7, rounded to 16 bits, are a B operand [k][n] whose k runs over the 16 rows of
//    slice s in the order 4h + {0..3}, 8 + 4h + {0..3} (h = lane >> 5).  The contraction does not care about
//    the order as long as the A operand follows it, so a score tile feeds the next product from registers;
//  * that A operand is the transpose of a row-major tile: ds_read_b64_tr_b16 delivers it from LDS.
// Tiles lie in LDS row-major, 2 D bytes a row, their 16-byte chunks XOR-swizzled by a function of the row
// under which both the row reads (8 rows, one chunk) and the transposing reads (4 rows, a chunk pair) fall on
// all banks.  They are filled by buffer loads straight to LDS: rows past the end or masked out are given an
// offset outside the buffer and arrive as zeros, so what memory holds there (NaN included) enters no product.
#pragma once
#include "common.h"
#include "lrce_capi.h"

// kernel arguments
struct AttnP {
  const bf16 *q, *k, *v, *dout;
  bf16 *out, *dq, *dk, *dv;
  float* lse;          // [B][H][Lq]
  const void* mask;    // [B][Lk], mask_bytes an entry, 0 = key hidden
  long long sqb, sql, sqh, skb, skl, skh, svb, svl, svh, sob, sol, soh, sgb, sgl, sgh;   // strides of q, k, v, out, dout
  long long dqb, dql, dqh, dkb, dkl, dkh, dvb, dvl, dvh;                                   // of dq, dk, dv
  long long smb;
  int B, H, Hk, G, Lq, Lk, causal, mask_bytes, off;   // G = H / Hk, off = Lk - Lq
  float scale, c;      // c = scale * log2(e)
  int nblk, nsplit, split_tiles;
  float* ws;           // forward: partials of the splits; backward: row statistics, then partials
  float* ws2;
};

// host side, shared by the two files' entry points: argument checks (an LRCE_E_* code) and the kernel arguments
int attn_check(const LrceAttnDesc* d, const char* what);
void attn_fill(const LrceAttnDesc* d, AttnP& p);

// Whether the waves of a workgroup share 32 rows and divide the keys, rather than have 32 rows each: where row tiles alone
// leave the chip's 1024 SIMDs without a second wave to fill the first one's waits, and the key axis is long enough to divide.
// Measured (us divided / not; forward, then dq with dk and dv): 64 heads x 8 tiles x 1024 keys d 64 10.9 / 21.6; 32 heads x 22 tiles
// x 700 keys d 64 16 / 16, 40 / 40, 32 x 19 x 800 d 32 11 / 14, 25 / 28.  A divided workgroup of the wide heads holds two stages a
// wave in 49 or 64 KB of LDS: at 64 x 9 x 1213 d 96 30 / 27, 67 / 68, 64 x 8 x 1024 d 96 25 / 22, 47 / 52, and where
// they are more than the two a CU that fit, 64 x 9 x 1213 d 128 50 / 31, 101 / 87, 32 x 19 x 800 35 / 22, 63 / 55 (32 x 16 x 512 15 / 16,
// 38 / 42).
inline bool attn_few_rows(int64_t row_tiles, int Lk, int D, bool bwd) {
  return Lk >= 192 && row_tiles <= (D <= 64 ? 768 : !bwd ? 500 : D == 96 ? 768 : 512);
}
// ... and how many waves: a wave has two stages of K and V of 32 keys in LDS (8 to 32 KB); four waves of the wide ones would
// leave one workgroup a CU
inline int attn_share_waves(int D, int64_t row_tiles) { return D <= 64 || row_tiles <= 256 ? 4 : 2; }

namespace {

typedef __attribute__((ext_vector_type(4))) int i32x4;
typedef LRCE_LDS char* lds_ptr;
typedef const LRCE_LDS char* lds_cptr;

constexpr float ATTN_LOG2E = 1.4426950408889634f;
constexpr int ATTN_MASK_KEYS = 16384;   // keys whose mask bits lie in LDS at a time

__device__ __forceinline__ int crow32(int reg, int h) { return (reg & 3) + 8 * (reg >> 2) + 4 * h; }

// XOR of the 16-byte chunk index.  LDS serves 256 bytes a cycle: 16 lanes of a row read (16 rows, one chunk) and 32 lanes
// of a transposing read (4 rows, an aligned group of 4 chunks) have to fall on the 16 chunk places of 256 bytes.  A row
// is 16, 8, 12 or 4 chunks, so rows themselves take turns of 1, 2, 4 or 4 places; the XOR does the rest with 4, 3, 2 or 2 bits.
template <int D>
__device__ __forceinline__ int attn_swz(int row) {
  if constexpr (D == 128) return ((row & 3) << 2) | ((row >> 2) & 3);
  else if constexpr (D == 64) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else return (row >> 2) & 3;
}

// Per-lane byte offsets of the operand reads of a tile [rows][D]
template <int D>
struct TileRead {
  static constexpr int NV = D == 128 ? 8 : D == 64 ? 4 : 2, NT = D == 128 ? 4 : D == 64 ? 2 : 1, PITCH = 2 * D;
  int ka[NV], va[NT];
  __device__ __forceinline__ void init(int lane) {
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int j = 0; j < NV; ++j) ka[j] = r * PITCH + (((2 * j + h) ^ attn_swz<D>(r)) << 4);
    const int g = lane >> 4, i = lane & 15, q = i >> 2, p = i & 3, row = 4 * (g >> 1) + q;
#pragma unroll
    for (int j = 0; j < NT; ++j)
      va[j] = row * PITCH + (((4 * j + 2 * (g & 1) + (p >> 1)) ^ attn_swz<D>(row)) << 4) + (p & 1) * 8;
  }
  // A[m = row r0 + lane & 31][k = 16 kk + 8 h ..]   (r0 a multiple of 32)
  __device__ __forceinline__ bf16x8 row(lds_cptr t, int r0, int kk) const {
    return *reinterpret_cast<const LRCE_LDS bf16x8*>(t + ka[kk % NV] + (kk / NV) * (NV * 32) + r0 * PITCH);
  }
  // A[m = column 32 blk + lane & 31][k = rows r0 .. r0 + 15 in the accumulator's order]   (r0 a multiple of 16).  The swizzle
  // of row + 8 is that of row with bit 1 flipped.
  __device__ __forceinline__ bf16x8 col(lds_cptr t, int r0, int blk) const {
    bf16x8 o;
#pragma unroll
    for (int h2 = 0; h2 < 2; ++h2) {
      const int at = (va[blk % NT] + (blk / NT) * (NT * 64)) ^ (h2 * 32);
      s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LRCE_LDS s16x4*)(t + at + (r0 + 8 * h2) * PITCH));
      const bf16x4 b = __builtin_bit_cast(bf16x4, v);
      o[4 * h2 + 0] = b[0]; o[4 * h2 + 1] = b[1]; o[4 * h2 + 2] = b[2]; o[4 * h2 + 3] = b[3];
    }
    return o;
  }
};

__device__ __forceinline__ uint32_t attn_lds_u32(lds_cptr p) { return (uint32_t)(uintptr_t)p; }
// Workgroup -> (head, block).  Without causality a head's blocks are neighbours on one XCD, whose L2 keeps its K and V.  With
// it the blocks differ in work: the longest of all heads come first, and a head's workgroups stay on one XCD where the
// number of (batch, key head) pairs allows (ids go round the 8 XCDs), query heads of a group together.
struct Place { int b, hq, blk; };
__device__ __forceinline__ Place attn_place(const AttnP& p, int heads_per_key) {
  Place x;
  if (p.causal) {
    const int nk = p.B * p.Hk, n = nk * heads_per_key, j = blockIdx.x % n, bk = j % nk;
    x.blk = blockIdx.x / n;
    x.b = bk / p.Hk;
    x.hq = (bk % p.Hk) * heads_per_key + j / nk;
  } else {
    const int id = xcd_remap(blockIdx.x, gridDim.x), bh = id / p.nblk, h = p.Hk * heads_per_key;
    x.blk = id % p.nblk;
    x.b = bh / h;
    x.hq = bh % h;
  }
  return x;
}

// Scheduling: GROUPS times one matrix instruction, then VALU vector instructions (the compiler's own order clusters each kind)
template <int GROUPS, int VALU>
__device__ __forceinline__ void attn_interleave() {
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x2, VALU, 0);
  }
}
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ const char* uni(const void* p) {
  const uint64_t a = reinterpret_cast<uintptr_t>(p);
  return reinterpret_cast<const char*>((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a) |
                                       ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32)) << 32));
}

// A buffer of `bytes` bytes at a wave-uniform address; what lies at or past its end reads as zeros
__device__ __forceinline__ i32x4 attn_rsrc(const char* base, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uintptr_t>(base);
  i32x4 rs;
  rs[0] = (int)(uint32_t)a;
  rs[1] = (int)(uint32_t)((a >> 32) & 0xffffu);
  rs[2] = (int)bytes;
  rs[3] = 0x00020000;
  return rs;
}
// N loads of 64 lanes x 16 bytes from rs + voff[i] to LDS at dst + i * STEP (wave-uniform, 1 KB each).  In asm, so that the
// compiler does not drain the loads in flight before every LDS read; the loops' own waits order them.
template <int N, int STEP>
__device__ __forceinline__ void attn_glds(i32x4 rs, const uint32_t* voff, uint32_t dst) {
  unsigned keep;
  if constexpr (N >= 4) {
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %6\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %5, 0 offen lds\n\ts_add_u32 m0, m0, %7\n\t"
                 "s_nop 0\n\tbuffer_load_dwordx4 %2, %5, 0 offen lds\n\ts_add_u32 m0, m0, %7\n\ts_nop 0\n\t"
                 "buffer_load_dwordx4 %3, %5, 0 offen lds\n\ts_add_u32 m0, m0, %7\n\ts_nop 0\n\tbuffer_load_dwordx4 %4, %5, 0 offen lds\n\t"
                 "s_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff[0]), "v"(voff[1]), "v"(voff[2]), "v"(voff[3]), "s"(rs), "s"(dst), "n"(STEP) : "memory", "scc");
    attn_glds<N - 4, STEP>(rs, voff + 4, dst + 4 * STEP);
  } else if constexpr (N >= 1) {
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds\n\ts_mov_b32 m0, %0"
                 : "=&s"(keep) : "v"(voff[0]), "s"(rs), "s"(dst) : "memory");
    attn_glds<N - 1, STEP>(rs, voff + 1, dst + STEP);
  }
}
// Operands that a loop with loads to LDS in flight reads from registers have to have landed before it: the compiler, which
// does not see those loads, would else wait for every load at the operands' first use in each iteration.
template <int N>
__device__ __forceinline__ void attn_landed(bf16x8 (&x)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(x[i]));
}
template <int N>
__device__ __forceinline__ void attn_wait_vm() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// this wave's loads have landed and every wave is past its reads
__device__ __forceinline__ void attn_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// Staging of tiles [ROWS][D] by NW waves: NI loads of 1 KB each a wave
template <int D, int ROWS, int NW>
struct TileStage {
  static constexpr int CH = D / 8, NI = ROWS * CH / (64 * NW), BYTES = ROWS * D * 2;
  static_assert(NI * 64 * NW == ROWS * CH, "whole loads");
  uint32_t voff[NI];
  uint32_t pitch;
  __device__ __forceinline__ static int row_of(int i, int lane, int wave) { return ((i * NW + wave) * 64 + lane) / CH; }
  __device__ __forceinline__ void init(int lane, int wave, long long ld) {
    pitch = (uint32_t)(ld * 2);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int id = (i * NW + wave) * 64 + lane, row = id / CH, cp = id % CH;
      voff[i] = (uint32_t)row * pitch + (uint32_t)((cp ^ attn_swz<D>(row)) << 4);
    }
  }
  // bytes of the tile's first n rows (0 < n)
  __device__ __forceinline__ uint32_t bytes(int n) const { return (uint32_t)(min(n, ROWS) - 1) * pitch + 2 * D; }
  // the tile at base, of which the first n rows exist
  __device__ __forceinline__ void load(const char* base, int n, uint32_t dst, int wave) const {
    attn_glds<NI, NW * 1024>(attn_rsrc(base, bytes(n)), voff, dst + (uint32_t)wave * 1024);
  }
  // the same; row r is left zero where bit r of keep is 0
  __device__ __forceinline__ void load(const char* base, int n, uint64_t keep, uint32_t dst, int lane, int wave) const {
    uint32_t o[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) o[i] = ((keep >> row_of(i, lane, wave)) & 1) ? voff[i] : 0x80000000u;
    attn_glds<NI, NW * 1024>(attn_rsrc(base, bytes(n)), o, dst + (uint32_t)wave * 1024);
  }
};

// Mask bits of the 64-key words w0, w0 + STEP, ... below w1 of batch row b: put(word, bits), bit l = key 64 word + l is there and
// not hidden.  Up to eight words are loaded before the first is looked at.
template <int STEP, typename T, typename F>
__device__ __forceinline__ void attn_mask_words_of(const T* m, int Lk, int w0, int w1, int lane, F&& put) {
  for (int c = w0; c < w1; c += 8 * STEP) {
    T x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i * STEP < w1) x[i] = m[min((c + i * STEP) * 64 + lane, Lk - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int w = c + i * STEP;
      if (w < w1) put(w, __ballot(x[i] != 0 && w * 64 + lane < Lk));
    }
  }
}
template <int STEP, typename F>
__device__ __forceinline__ void attn_mask_words(const AttnP& p, int b, int w0, int w1, int lane, F&& put) {
  const long long at = (long long)b * p.smb;
  if (p.mask_bytes == 1) attn_mask_words_of<STEP>(static_cast<const uint8_t*>(p.mask) + at, p.Lk, w0, w1, lane, put);
  else if (p.mask_bytes == 4) attn_mask_words_of<STEP>(static_cast<const int*>(p.mask) + at, p.Lk, w0, w1, lane, put);
  else attn_mask_words_of<STEP>(static_cast<const long long*>(p.mask) + at, p.Lk, w0, w1, lane, put);
}
// ... of the tiles [t0, t0 + n) to LDS
template <int NW>
__device__ __forceinline__ void attn_pack_mask(const AttnP& p, int b, int t0, int n, LRCE_LDS uint64_t* words, int lane, int wave) {
  attn_mask_words<NW>(p, b, t0 + wave, t0 + n, lane, [&](int w, uint64_t bits) {
    if (lane == 0) words[w - t0] = bits;
  });
}
__device__ __forceinline__ uint64_t uni64(uint64_t x) {
  return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x) |
         ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32);
}
__device__ __forceinline__ uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }
// the low n + 1 bits of a word (n < 0: none)
__device__ __forceinline__ uint32_t upto(int n) { return n >= 31 ? ~0u : n < 0 ? 0u : (2u << n) - 1; }

__device__ __forceinline__ float other_half(float x) {
  const unsigned u = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float((threadIdx.x & 32) ? s[0] : s[1]);
}

// registers 8s .. 8s+7 of an accumulator tile as 16-bit values (round to nearest)
template <bool F16>
__device__ __forceinline__ bf16x8 attn_pack(const f32x16& a, int s) {
  bf16x8 o;
#pragma unroll
  for (int j = 0; j < 8; ++j) o[j] = to16<F16>(a[8 * s + j]);
  return o;
}

// A transposed accumulator tile [d = 32 rows][row = lane & 31], times mul, into the row at dst (16 bits): the halves
// exchange 4-value groups so that each lane stores 16 bytes at a time
template <bool F16>
__device__ __forceinline__ void attn_store(const f32x16& a, float mul, bf16* dst, int h, bool valid) {
#pragma unroll
  for (int u = 0; u < 4; u += 2) {
    unsigned x[2], y[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      bf16x2 t;
      t[0] = to16<F16>(a[4 * u + 2 * e] * mul); t[1] = to16<F16>(a[4 * u + 2 * e + 1] * mul);
      x[e] = __builtin_bit_cast(unsigned, t);
      t[0] = to16<F16>(a[4 * u + 4 + 2 * e] * mul); t[1] = to16<F16>(a[4 * u + 5 + 2 * e] * mul);
      y[e] = __builtin_bit_cast(unsigned, t);
    }
    uint4 o;
    const auto s0 = __builtin_amdgcn_permlane32_swap(x[0], y[0], false, false);
    const auto s1 = __builtin_amdgcn_permlane32_swap(x[1], y[1], false, false);
    o.x = s0[0]; o.y = s1[0]; o.z = s0[1]; o.w = s1[1];
    if (valid) *reinterpret_cast<uint4*>(dst + 8 * (u + h)) = o;
  }
}

}  // namespace
