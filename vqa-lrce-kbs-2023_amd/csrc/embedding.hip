// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   y[n] = scale W[ids[n]],   dW[v] = scale sum over n with ids[n] = v of dy[n], added in token order.
//
// Forward: a wave a row, memory-bound.
// Backward: a scatter by atomics would add in an order that changes from run to run, and tokens of one frequent word
// would queue on one row.  Instead the tokens are sorted by id (stable: equal ids keep their order), the sorted list is cut
// into pieces, and a workgroup adds the rows of one piece in f32, run by run.  A run inside the piece is a
// finished row of dW; a run that crosses the piece's ends leaves a partial row, and embed_join_kernel adds a run's
// partials in order.  Every row of dW has one writer and a fixed order of additions: the result is the same bits each time.
// The sort is a radix sort of up to 9 bits a pass: up to SORT_N tokens in one workgroup's LDS; above, a histogram and a
// scatter launch a pass (workgroups of 2048 tokens, of 8192 above 2^18 tokens: each reads every workgroup's counts).  Rows
// without tokens have to be zero: the workgroups that the sort leaves idle clear dW meanwhile.
// Few tokens (up to SMALL_N) need neither sort nor pieces: embed_small_kernel clears and adds in one launch, workgroup b
// having the rows v = b mod the grid and picking its tokens out of the list itself.
// Ids outside the table give a row of NaN forward and no gradient; so has padding_idx no gradient.
// Measured: 65521 tokens, table 128000 x 1024, bf16: forward 43 us (268 MB, 6.2 TB/s), backward 92 us of sort and clearing (524 MB of
// zeros alone: 77 us at the rate of a fill), 73 us of sums, 13 us of joins; 8190 tokens, 30522 x 768 f32 from bf16: 7 us, 23 us of
// sort (the clearing, 15 us, beside it), 8 + 5 us; 320 tokens of that table: 3 us, 15 us (94 MB cleared).
#include <algorithm>

#include "common.h"
#include "lrce_capi.h"

namespace {

constexpr int SORT_N = 8192;       // tokens of a sorting workgroup
constexpr int SORT_T = 1024, SORT_W = SORT_T / 64, SORT_R = SORT_N / SORT_T;   // threads, waves, rounds of 64 places a wave
constexpr int SMALL_N = 512;
constexpr int BINS = 512;
constexpr int CHUNK = 16;          // rows of dy in flight a thread

template <typename T> __device__ __forceinline__ float to_f(T x) { return (float)x; }
// scale * x as an f32 value, then rounded to T: the same bits for every pair of types (the compiler would fuse the product with
// the rounding to fp16)
template <typename T>
__device__ __forceinline__ T scaled(float x, float scale) {
  float v = x * scale;
  asm("" : "+v"(v));
  return (T)v;
}

__device__ __forceinline__ uint32_t token_key(const void* ids, int ids64, long long n, uint32_t V, long long pad) {
  const long long id = ids64 ? static_cast<const long long*>(ids)[n] : (long long)static_cast<const int*>(ids)[n];
  return id < 0 || id >= (long long)V || id == pad ? V : (uint32_t)id;
}

template <typename TW, typename TY, int VEC>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const void* __restrict__ ids, int ids64, long long N, long long V, int C,
                                                        const TW* __restrict__ w, long long ldw, TY* __restrict__ y, float scale) {
  typedef TW wv __attribute__((ext_vector_type(VEC)));
  typedef TY yv __attribute__((ext_vector_type(VEC)));
  const int lane = threadIdx.x & 63;
  for (long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); n < N; n += (long long)gridDim.x * 4) {
    const long long id = ids64 ? static_cast<const long long*>(ids)[n] : (long long)static_cast<const int*>(ids)[n];
    const bool ok = id >= 0 && id < V;
    const TW* src = w + (ok ? id : 0) * ldw;
    for (int c = lane * VEC; c < C; c += 64 * VEC) {
      yv o;
      if constexpr (VEC == 1) o[0] = scaled<TY>(ok ? to_f(src[c]) : __builtin_nanf(""), scale);
      else {
        const wv x = *reinterpret_cast<const wv*>(src + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = scaled<TY>(ok ? to_f(x[i]) : __builtin_nanf(""), scale);
      }
      if constexpr (VEC == 1) y[n * C + c] = o[0];
      else *reinterpret_cast<yv*>(y + n * C + c) = o;
    }
  }
}

struct SortP {
  const void* ids;
  long long N, pad;
  int ids64;
  uint32_t V;
  const uint32_t *kin, *iin;   // null: the ids themselves
  uint32_t *kout, *iout;
  uint32_t* hist;              // [workgroup][BINS]
  int shift, bits, passes, nwg, rounds;
  float* fill;                 // this launch's part of dW to clear
  long long fill_n;            // in floats, from a 16-byte boundary
};

// workgroups [first, gridDim.x) clear p.fill
__device__ __forceinline__ void clear_part(const SortP& p, int first) {
  const long long nt = (long long)(gridDim.x - first) * blockDim.x;
  const long long t = (long long)(blockIdx.x - first) * blockDim.x + threadIdx.x;
  const long long n4 = p.fill_n >> 2;
  float4* d = reinterpret_cast<float4*>(p.fill);
  for (long long i = t; i < n4; i += nt) d[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (t < (p.fill_n & 3)) p.fill[4 * n4 + t] = 0.f;
}

// lanes with the same digit (of those that count)
__device__ __forceinline__ uint64_t same_digit(uint32_t d, int bits, bool on) {
  uint64_t m = __ballot(on);
  for (int b = 0; b < bits; ++b) {
    const uint64_t v = __ballot((d >> b) & 1);
    m &= (d >> b) & 1 ? v : ~v;
  }
  return on ? m : 0;
}

struct SortLds {
  uint32_t cnt[SORT_W][BINS];
  uint32_t base[BINS];
  uint32_t wsum[SORT_W];
};

// Ranks of a workgroup's keys (place = wave * per + round * 64 + lane): rank[r] counts the wave's earlier keys of the same
// digit; afterwards s.cnt[wave][d] = keys of digit d in earlier waves, s.base[d] = the workgroup's keys of smaller digits
__device__ __forceinline__ void rank_keys(SortLds& s, const uint32_t* key, const bool* on, int rounds, int shift, int bits, uint32_t* rank) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t dm = (1u << bits) - 1;
  for (int i = threadIdx.x; i < SORT_W * BINS; i += SORT_T) (&s.cnt[0][0])[i] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < SORT_R; ++r) {
    if (r < rounds) {
      const uint32_t d = (key[r] >> shift) & dm;
      const uint64_t m = same_digit(d, bits, on[r]);
      const uint32_t before = __popcll(m & ((1ull << lane) - 1));
      rank[r] = before + (on[r] ? s.cnt[wave][d] : 0);
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if (on[r] && before == 0) s.cnt[wave][d] += (uint32_t)__popcll(m);   // the first lane of each digit
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  __syncthreads();
  uint32_t total = 0;
  if (threadIdx.x < BINS) {
#pragma unroll
    for (int w = 0; w < SORT_W; ++w) {
      const uint32_t c = s.cnt[w][threadIdx.x];
      s.cnt[w][threadIdx.x] = total;
      total += c;
    }
  }
  // exclusive sums over the digits (the first BINS threads hold one each)
  uint32_t x = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63) s.wsum[wave] = x;
  __syncthreads();
  if (threadIdx.x < BINS) {
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += s.wsum[w];
    s.base[threadIdx.x] = before + x - total;
  }
  __syncthreads();
}

// All passes of up to SORT_N tokens in one workgroup; the others clear dW
__global__ void __launch_bounds__(SORT_T) embed_sort_kernel(SortP p) {
  if (blockIdx.x > 0) return clear_part(p, 1);
  __shared__ SortLds s;
  __shared__ uint32_t sk[SORT_N];
  __shared__ uint16_t si[SORT_N];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int rounds = (int)((p.N + SORT_T - 1) / SORT_T);
  uint32_t key[SORT_R], rank[SORT_R];
  uint16_t idx[SORT_R];
  bool on[SORT_R];
#pragma unroll
  for (int r = 0; r < SORT_R; ++r) {
    const int at = (wave * rounds + r) * 64 + lane;
    on[r] = r < rounds && at < p.N;
    key[r] = on[r] ? token_key(p.ids, p.ids64, at, p.V, p.pad) : 0;
    idx[r] = (uint16_t)at;
  }
  for (int ps = 0; ps < p.passes; ++ps) {
    const int shift = ps * p.bits;
    rank_keys(s, key, on, rounds, shift, p.bits, rank);
    const uint32_t dm = (1u << p.bits) - 1;
#pragma unroll
    for (int r = 0; r < SORT_R; ++r)
      if (on[r]) {
        const uint32_t d = (key[r] >> shift) & dm, at = s.base[d] + s.cnt[wave][d] + rank[r];
        sk[at] = key[r];
        si[at] = idx[r];
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < SORT_R; ++r) {
      const int at = (wave * rounds + r) * 64 + lane;
      if (on[r]) { key[r] = sk[at]; idx[r] = si[at]; }
    }
  }
#pragma unroll
  for (int r = 0; r < SORT_R; ++r) {
    const int at = (wave * rounds + r) * 64 + lane;
    if (on[r]) { p.kout[at] = key[r]; p.iout[at] = idx[r]; }
  }
}

__device__ __forceinline__ uint32_t sort_key(const SortP& p, long long at) {
  return p.kin ? p.kin[at] : token_key(p.ids, p.ids64, at, p.V, p.pad);
}

// one pass over many workgroups: digit counts ...
__global__ void __launch_bounds__(SORT_T) embed_hist_kernel(SortP p) {
  if ((int)blockIdx.x >= p.nwg) return clear_part(p, p.nwg);
  __shared__ uint32_t cnt[BINS];
  for (int i = threadIdx.x; i < BINS; i += SORT_T) cnt[i] = 0;
  __syncthreads();
  const uint32_t dm = (1u << p.bits) - 1;
  for (int r = 0; r < p.rounds; ++r) {
    const long long at = ((long long)blockIdx.x * p.rounds + r) * SORT_T + threadIdx.x;
    if (at < p.N) atomicAdd(&cnt[(sort_key(p, at) >> p.shift) & dm], 1u);    // counts only: any order gives the same
  }
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += SORT_T) p.hist[(long long)blockIdx.x * BINS + i] = cnt[i];
}
// ... and the stable scatter: a key's place = keys of smaller digits + of its digit in earlier workgroups + its rank here
__global__ void __launch_bounds__(SORT_T) embed_scatter_kernel(SortP p) {
  if ((int)blockIdx.x >= p.nwg) return clear_part(p, p.nwg);
  __shared__ SortLds s;
  __shared__ uint32_t all[BINS], mine[BINS], wsum[BINS / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t key[SORT_R], idx[SORT_R], rank[SORT_R];
  bool on[SORT_R];
#pragma unroll
  for (int r = 0; r < SORT_R; ++r) {
    const long long at = (long long)blockIdx.x * p.rounds * SORT_T + (wave * p.rounds + r) * 64 + lane;
    on[r] = r < p.rounds && at < p.N;
    key[r] = on[r] ? sort_key(p, at) : 0;
    idx[r] = on[r] ? (p.iin ? p.iin[at] : (uint32_t)at) : 0;
  }
  uint32_t total = 0, x = 0;
  if (threadIdx.x < BINS) {
    uint32_t before = 0;
#pragma unroll 8
    for (int w = 0; w < p.nwg; ++w) {
      const uint32_t c = p.hist[(long long)w * BINS + threadIdx.x];
      if (w < (int)blockIdx.x) before += c;
      total += c;
    }
    mine[threadIdx.x] = before;
  }
  x = total;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  if (lane == 63 && wave < BINS / 64) wsum[wave] = x;
  __syncthreads();
  if (threadIdx.x < BINS) {
    uint32_t before = 0;
    for (int w = 0; w < wave; ++w) before += wsum[w];
    all[threadIdx.x] = before + x - total + mine[threadIdx.x];
  }
  rank_keys(s, key, on, p.rounds, p.shift, p.bits, rank);                     // (its barriers order `all` too)
  const uint32_t dm = (1u << p.bits) - 1;
#pragma unroll
  for (int r = 0; r < SORT_R; ++r)
    if (on[r]) {
      const uint32_t d = (key[r] >> p.shift) & dm, at = all[d] + s.cnt[wave][d] + rank[r];
      p.kout[at] = key[r];
      p.iout[at] = idx[r];
    }
}

struct SumP {
  float *dw, *part;            // part [piece][2][C]: the run that came in from the left, the run that goes on to the right
  long long N;
  uint32_t V;
  int C, accumulate, piece;    // places of a piece (a multiple of CHUNK)
  float scale;
};

template <int VEC>
__device__ __forceinline__ void put_row(float* dst, const float* a, bool add) {
  if constexpr (VEC == 1) dst[0] = add ? dst[0] + a[0] : a[0];
  else {
#pragma unroll
    for (int v = 0; v < VEC; v += 4) {
      float4 x = make_float4(a[v], a[v + 1], a[v + 2], a[v + 3]);
      if (add) {
        const float4 y = *reinterpret_cast<const float4*>(dst + v);
        x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
      }
      *reinterpret_cast<float4*>(dst + v) = x;
    }
  }
}

// A piece's runs; thread t has the columns [VEC t, VEC t + VEC) of a stripe of blockDim.x VEC columns (blockIdx.y).  The
// rows come CHUNK at a time, all in flight together (those behind the last key that counts are read but not added).
template <typename T, int VEC>
__global__ void __launch_bounds__(256) embed_sum_kernel(SumP p, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ idx,
                                                        const T* __restrict__ dy) {
  typedef T tv __attribute__((ext_vector_type(VEC)));
  const long long p0 = (long long)blockIdx.x * p.piece;
  const int n = (int)min((long long)p.piece, p.N - p0), c = (blockIdx.y * blockDim.x + threadIdx.x) * VEC;
  if (c >= p.C) return;
  const uint32_t beyond = p0 + n < p.N ? keys[p0 + n] : p.V;    // the key right of the piece
  bool left = p0 > 0 && keys[p0 - 1] == keys[p0];                // the current run came in from the left
  float a[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) a[e] = 0.f;
  for (int i0 = 0; i0 < n; i0 += CHUNK) {
    uint32_t key[CHUNK];
    tv x[CHUNK];
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) {
      const long long at = p0 + min(i0 + i, n - 1);
      key[i] = keys[at];
      x[i] = *reinterpret_cast<const tv*>(dy + (long long)idx[at] * p.C + c);
    }
    if (key[0] == p.V) return;                                   // what has no gradient is sorted last
    const uint32_t after = i0 + CHUNK < n ? keys[p0 + i0 + CHUNK] : beyond;
#pragma unroll
    for (int i = 0; i < CHUNK; ++i) {
      if (i0 + i >= n || key[i] == p.V) break;
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[e] += to_f(x[i][e]);
      const bool end = i0 + i + 1 == n;
      const uint32_t nx = end ? beyond : i + 1 < CHUNK ? key[i + 1 < CHUNK ? i + 1 : 0] : after;
      if (nx != key[i] || end) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[e] *= p.scale;
        float* dst = left ? p.part + (2 * (long long)blockIdx.x) * p.C
                   : nx == key[i] ? p.part + (2 * (long long)blockIdx.x + 1) * p.C : p.dw + (long long)key[i] * p.C;
        put_row<VEC>(dst + c, a, p.accumulate && !left && nx != key[i]);
        left = false;
#pragma unroll
        for (int e = 0; e < VEC; ++e) a[e] = 0.f;
      }
    }
  }
}

// A run that begins in piece x and goes on: its partial rows.  The pieces it covers are counted 256 at a time (a thread a
// piece); then each of the four waves adds a quarter of the rows in order, and the quarters are added in order.
template <int VEC>
__global__ void __launch_bounds__(256) embed_join_kernel(SumP p, const uint32_t* __restrict__ keys) {
  typedef float fv __attribute__((ext_vector_type(VEC)));
  const long long x = blockIdx.x, end = (x + 1) * p.piece;
  if (end >= p.N) return;
  const uint32_t id = keys[end - 1];
  if (id == p.V || keys[end] != id) return;
  if (x > 0 && keys[x * p.piece - 1] == id) return;      // it began in an earlier piece
  __shared__ fv red[3][64];
  const long long pieces = (p.N + p.piece - 1) / p.piece;
  long long m = 0;                                       // pieces from x + 1 on that begin with the run
  for (int got = 256; got == 256; m += got) {
    const long long y = x + 1 + m + threadIdx.x;
    got = __syncthreads_count(y < pieces && keys[min(y, pieces - 1) * p.piece] == id);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = (blockIdx.y * 64 + lane) * VEC;
  fv a = {};
  if (c < p.C) {
    if (wave == 0) a = *reinterpret_cast<const fv*>(p.part + (2 * x + 1) * p.C + c);
    const long long y0 = x + 1 + m * wave / 4, y1 = x + 1 + m * (wave + 1) / 4;
#pragma unroll 16
    for (long long y = y0; y < y1; ++y) a += *reinterpret_cast<const fv*>(p.part + 2 * y * p.C + c);
    if (wave) red[wave - 1][lane] = a;
  }
  __syncthreads();
  if (wave == 0 && c < p.C) {
    a = ((a + red[0][lane]) + red[1][lane]) + red[2][lane];
    put_row<VEC>(p.dw + (long long)id * p.C + c, reinterpret_cast<const float*>(&a), p.accumulate);
  }
}

// The whole gradient for N <= SMALL_N tokens: a workgroup lists its tokens in order, clears its rows without tokens, and adds
// the others, each row by the waves that its columns take, 8 rows of dy in flight
template <typename T, int VEC>
__global__ void __launch_bounds__(1024) embed_small_kernel(SumP p, const void* __restrict__ ids, int ids64, long long pad,
                                                           const T* __restrict__ dy) {
  typedef T tv __attribute__((ext_vector_type(VEC)));
  __shared__ uint32_t row[SMALL_N], wsum[SMALL_N / 64];
  __shared__ uint16_t tok[SMALL_N];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t k = (int)threadIdx.x < p.N ? token_key(ids, ids64, threadIdx.x, p.V, pad) : p.V;
  const bool mine = k != p.V && k % gridDim.x == blockIdx.x;
  const uint64_t m = __ballot(mine);
  if (lane == 0 && wave < SMALL_N / 64) wsum[wave] = __popcll(m);
  __syncthreads();
  int n = 0;
  for (int w = 0; w < SMALL_N / 64; ++w) {
    if (w == wave && mine) {
      const int at = n + __popcll(m & ((1ull << lane) - 1));
      row[at] = k;
      tok[at] = (uint16_t)threadIdx.x;
    }
    n += wsum[w];
  }
  __syncthreads();
  if (!p.accumulate)
    for (long long v = blockIdx.x + (long long)wave * gridDim.x; v < p.V; v += 16ll * gridDim.x) {
      bool has = false;
      for (int i = lane; i < n; i += 64) has |= row[i] == v;
      if (__any(has)) continue;
      float* d = p.dw + v * p.C;
      if constexpr (VEC > 1)
        for (int c = 4 * lane; c < p.C; c += 256) *reinterpret_cast<float4*>(d + c) = make_float4(0.f, 0.f, 0.f, 0.f);
      else
        for (int c = lane; c < p.C; c += 64) d[c] = 0.f;
    }
  const int wpr = min(16, (p.C + 64 * VEC - 1) / (64 * VEC)), groups = 16 / wpr, g = wave / wpr, c0 = ((wave % wpr) * 64 + lane) * VEC;
  if (g >= groups) return;
  int seen = 0;                                           // rows met so far; group g adds those with seen = g mod groups
  for (int i = 0; i < n; ++i) {
    const uint32_t v = row[i];
    bool before = false;
    for (int j = lane; j < i; j += 64) before |= row[j] == v;
    if (__any(before) || seen++ % groups != g) continue;
    for (int c = c0; c < p.C; c += wpr * 64 * VEC) {
      float a[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[e] = 0.f;
      for (int base = i & ~63; base < n; base += 64) {
        uint64_t hit = 0;
        for (int j = 0; j < 64 && base + j < n; ++j) hit |= (uint64_t)(row[base + j] == v) << j;
        while (hit) {
          tv x[8];
          int num = 0;
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const int j = hit ? __builtin_ctzll(hit) : 0;
            if (hit) ++num;
            x[q] = *reinterpret_cast<const tv*>(dy + (long long)tok[hit ? base + j : i] * p.C + c);
            hit &= hit - 1;
          }
#pragma unroll
          for (int q = 0; q < 8; ++q)
            if (q < num) {
#pragma unroll
              for (int e = 0; e < VEC; ++e) a[e] += to_f(x[q][e]);
            }
        }
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) a[e] *= p.scale;
      put_row<VEC>(p.dw + (long long)v * p.C + c, a, p.accumulate);
    }
  }
}

template <typename TW, typename TY>
void fwd_vec(int vec, const void* ids, int ids64, int64_t N, int64_t V, int C, const void* w, int64_t ldw, void* y, float scale, hipStream_t s) {
  const unsigned grid = (unsigned)std::min<int64_t>((N + 3) / 4, 1 << 20);
  const TW* wp = static_cast<const TW*>(w);
  TY* yp = static_cast<TY*>(y);
  if (vec == 8) embed_fwd_kernel<TW, TY, 8><<<grid, 256, 0, s>>>(ids, ids64, N, V, C, wp, ldw, yp, scale);
  else if (vec == 4) embed_fwd_kernel<TW, TY, 4><<<grid, 256, 0, s>>>(ids, ids64, N, V, C, wp, ldw, yp, scale);
  else embed_fwd_kernel<TW, TY, 1><<<grid, 256, 0, s>>>(ids, ids64, N, V, C, wp, ldw, yp, scale);
}

struct EmbPlan {
  int nwg, passes, bits, rounds, piece;
  int64_t pieces, words, part;   // 32-bit words of the sort, floats of the partial rows
};
EmbPlan emb_plan(int64_t N, int64_t V, int C) {
  EmbPlan f{};
  if (N <= SMALL_N) return f;
  int bits = 1;
  while (bits < 31 && (V >> bits)) ++bits;               // keys 0 .. V
  f.passes = (bits + 8) / 9;
  f.bits = (bits + f.passes - 1) / f.passes;
  f.rounds = N <= (1 << 18) ? 2 : SORT_R;
  f.nwg = N <= SORT_N ? 0 : (int)((N + f.rounds * SORT_T - 1) / (f.rounds * SORT_T));
  // pieces: short while that fills the chip (a frequent word's run is added in parallel), longer when there are enough
  f.piece = N <= 16384 ? CHUNK : 2 * CHUNK;
  f.pieces = (N + f.piece - 1) / f.piece;
  f.words = (N <= SORT_N ? 2 : 4) * N + (int64_t)f.nwg * BINS;
  f.words = (f.words + 3) / 4 * 4;
  f.part = 2 * f.pieces * C;
  return f;
}

}  // namespace

extern "C" int lrce_embedding_fwd(const void* ids, int ids_bytes, int64_t n, const void* w, int64_t ld_w, int64_t rows, int cols, int w_type,
                                  void* y, int y_type, float scale, void* stream) {
  if (n < 0 || rows < 1 || cols < 1 || rows >= (1ll << 31)) return lrce_fail(LRCE_E_ARG, "embedding: bad sizes n=%lld rows=%lld cols=%d", (long long)n, (long long)rows, cols);
  if (ids_bytes != 4 && ids_bytes != 8) return lrce_fail(LRCE_E_ARG, "embedding: ids of %d bytes (4 or 8)", ids_bytes);
  if (w_type < 0 || w_type > 2 || y_type < 0 || y_type > 2 || (w_type != 2 && y_type != w_type)) return lrce_fail(LRCE_E_ARG, "embedding: types %d -> %d", w_type, y_type);
  if (ld_w < cols) return lrce_fail(LRCE_E_ARG, "embedding: row pitch %lld < %d", (long long)ld_w, cols);
  if (n == 0) return LRCE_OK;
  if (!ids || !w || !y) return lrce_fail(LRCE_E_ARG, "embedding: null pointer");
  const int ws = w_type == 2 ? 4 : 2, ys = y_type == 2 ? 4 : 2;
  int vec = w_type == 2 ? 4 : 8;
  if (cols % vec || ld_w % vec || reinterpret_cast<uintptr_t>(w) % (vec * ws) || reinterpret_cast<uintptr_t>(y) % (vec * ys)) vec = 1;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int i64 = ids_bytes == 8;
  if (w_type == 0) fwd_vec<bf16, bf16>(vec, ids, i64, n, rows, cols, w, ld_w, y, scale, s);
  else if (w_type == 1) fwd_vec<f16, f16>(vec, ids, i64, n, rows, cols, w, ld_w, y, scale, s);
  else if (y_type == 0) fwd_vec<float, bf16>(vec, ids, i64, n, rows, cols, w, ld_w, y, scale, s);
  else if (y_type == 1) fwd_vec<float, f16>(vec, ids, i64, n, rows, cols, w, ld_w, y, scale, s);
  else fwd_vec<float, float>(vec, ids, i64, n, rows, cols, w, ld_w, y, scale, s);
  return lrce_check_launch("embedding");
}

extern "C" int64_t lrce_embedding_bwd_workspace(int64_t n, int64_t rows, int cols) {
  if (n < 0 || n >= (1ll << 31) || rows < 1 || rows >= (1ll << 31) || cols < 1) return -1;
  const EmbPlan f = emb_plan(n, rows, cols);
  return f.words + f.part;
}

extern "C" int lrce_embedding_bwd(const void* ids, int ids_bytes, int64_t n, const void* dy, int dy_type, float* dw, int64_t rows, int cols,
                                  float scale, int64_t padding_idx, int accumulate, float* workspace, int64_t workspace_elems, void* stream) {
  if (n < 0 || n >= (1ll << 31) || rows < 1 || cols < 1 || rows >= (1ll << 31)) return lrce_fail(LRCE_E_ARG, "embedding_bwd: bad sizes n=%lld rows=%lld cols=%d", (long long)n, (long long)rows, cols);
  if (ids_bytes != 4 && ids_bytes != 8) return lrce_fail(LRCE_E_ARG, "embedding_bwd: ids of %d bytes (4 or 8)", ids_bytes);
  if (dy_type < 0 || dy_type > 2) return lrce_fail(LRCE_E_ARG, "embedding_bwd: type %d", dy_type);
  if (padding_idx < -1 || padding_idx >= rows) return lrce_fail(LRCE_E_ARG, "embedding_bwd: padding_idx %lld of %lld rows (-1: none)", (long long)padding_idx, (long long)rows);
  if (!dw || reinterpret_cast<uintptr_t>(dw) % 16) return lrce_fail(LRCE_E_ARG, "embedding_bwd: dw must start at a multiple of 16 bytes");
  if (n > 0 && (!ids || !dy)) return lrce_fail(LRCE_E_ARG, "embedding_bwd: null pointer");
  if (n == 0 && accumulate) return LRCE_OK;
  const EmbPlan f = emb_plan(n, rows, cols);
  if (n > SMALL_N && (!workspace || workspace_elems < f.words + f.part || reinterpret_cast<uintptr_t>(workspace) % 16))
    return lrce_fail(LRCE_E_ARG, "embedding_bwd: a workspace of %lld floats at a multiple of 16 bytes is needed", (long long)(f.words + f.part));
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int es = dy_type == 2 ? 4 : 2;
  const bool al16 = reinterpret_cast<uintptr_t>(dy) % 16 == 0;
  const int vec = es == 2 && cols % 8 == 0 && al16 ? 8 : es == 4 && cols % 4 == 0 && al16 ? 4 : 1;
  SumP q{};
  q.dw = dw; q.N = n; q.V = (uint32_t)rows; q.C = cols; q.accumulate = accumulate; q.scale = scale;
  if (n <= SMALL_N) {
    const unsigned grid = (unsigned)std::min<int64_t>(rows, 512);
#define LRCE_EMB_SMALL(T, W) \
    if (vec == W) embed_small_kernel<T, W><<<grid, 1024, 0, s>>>(q, ids, ids_bytes == 8, padding_idx, static_cast<const T*>(dy)); \
    else embed_small_kernel<T, 1><<<grid, 1024, 0, s>>>(q, ids, ids_bytes == 8, padding_idx, static_cast<const T*>(dy));
    if (dy_type == 0) { LRCE_EMB_SMALL(bf16, 8) }
    else if (dy_type == 1) { LRCE_EMB_SMALL(f16, 8) }
    else { LRCE_EMB_SMALL(float, 4) }
#undef LRCE_EMB_SMALL
    return lrce_check_launch("embedding_bwd");
  }
  SortP p{};
  p.ids = ids; p.N = n; p.ids64 = ids_bytes == 8; p.V = (uint32_t)rows; p.pad = padding_idx;
  p.bits = f.bits; p.passes = f.passes; p.nwg = f.nwg; p.rounds = f.rounds;
  const int64_t total = accumulate ? 0 : rows * cols;
  // clearing workgroups: as many as fill the chip twice over, fewer for small tables
  auto clearers = [](int64_t floats) { return (unsigned)std::min<int64_t>((floats + 16 * SORT_T - 1) / (16 * SORT_T), 512); };
  uint32_t* wk = reinterpret_cast<uint32_t*>(workspace);
  uint32_t *key = wk, *idx = wk + n;
  if (n <= SORT_N) {
    p.kout = key; p.iout = idx;
    p.fill = dw; p.fill_n = total;
    embed_sort_kernel<<<1 + clearers(total), SORT_T, 0, s>>>(p);
  } else {
    uint32_t *k2 = wk + 2 * n, *i2 = wk + 3 * n;
    p.hist = wk + 4 * n;
    const int64_t step = (total / (3 * f.passes) + 3) / 4 * 4;            // each launch clears its share, a scatter twice a histogram's
    int64_t done = 0;
    auto share = [&](int parts, bool last) {
      p.fill = dw + done;
      p.fill_n = last ? total - done : std::min(parts * step, total - done);
      done += p.fill_n;
      return (unsigned)f.nwg + clearers(p.fill_n);
    };
    for (int ps = 0; ps < f.passes; ++ps) {
      const bool even = (f.passes - 1 - ps) % 2 == 0;                     // the last pass writes key / idx
      p.shift = ps * f.bits;
      p.kout = even ? key : k2; p.iout = even ? idx : i2;
      if (ps > 0) { p.kin = even ? k2 : key; p.iin = even ? i2 : idx; }
      embed_hist_kernel<<<share(1, false), SORT_T, 0, s>>>(p);
      embed_scatter_kernel<<<share(2, ps + 1 == f.passes), SORT_T, 0, s>>>(p);
    }
  }
  {
    q.part = workspace + f.words;
    q.piece = f.piece;
    const unsigned th = (unsigned)std::min(256, ((cols + vec - 1) / vec + 63) / 64 * 64);
    const dim3 grid((unsigned)f.pieces, (unsigned)((cols + th * vec - 1) / (th * vec)));
#define LRCE_EMB_SUM(T, W) \
    if (vec == W) embed_sum_kernel<T, W><<<grid, th, 0, s>>>(q, key, idx, static_cast<const T*>(dy)); \
    else embed_sum_kernel<T, 1><<<grid, th, 0, s>>>(q, key, idx, static_cast<const T*>(dy));
    if (dy_type == 0) { LRCE_EMB_SUM(bf16, 8) }
    else if (dy_type == 1) { LRCE_EMB_SUM(f16, 8) }
    else { LRCE_EMB_SUM(float, 4) }
#undef LRCE_EMB_SUM
    if (f.pieces > 1) {
      if (cols % 4 == 0) embed_join_kernel<4><<<dim3((unsigned)f.pieces, (unsigned)((cols + 255) / 256)), 256, 0, s>>>(q, key);
      else embed_join_kernel<1><<<dim3((unsigned)f.pieces, (unsigned)((cols + 63) / 64)), 256, 0, s>>>(q, key);
    }
  }
  return lrce_check_launch("embedding_bwd");
}
