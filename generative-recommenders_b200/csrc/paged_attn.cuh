// What the kernels of paged attention share: the call, the units of work and how they are cut, and the numbers that
// codes stand for.
#pragma once

#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace b200hstu {

constexpr int PA_BLOCK = 16;       // positions that lie on one page, whatever its size

struct PagedAttn {
  PagedCache cache;
  const void *q;
  void *out;
  IndexTensor lengths, q_offsets, targets;
  int64_t q_rs, q_hs, rows;
  int Hq, group, W, c;
  bool q_vec;                // 16-byte loads of q
  bool whole_units;          // a CTA takes whole units instead of an equal run of tiles: nothing to join
  float alpha, scale;
  // workspace
  int *status;
  int4 *joins;               // [CTA][2]
  float *part_o, *part_ml;   // [CTA][2][rows of a block][D], [CTA][2][rows of a block][2]
};

// ---------------------------------------------------------------------------------------
// units of work
// ---------------------------------------------------------------------------------------
// What block `rb` of the new rows (times query heads of a cache head) of sequence b has to read: positions
// [begin, end), that is [lo, hi) in multiples of 16; positions in [all_lo, all_hi) are seen by every row.  Positions past
// the table are left out, however long a sequence says it is: rows that see any are NaN (RowSees::past).
struct UnitRange {
  int lo, hi, all_lo, all_hi, begin, end;
  template <int TILE> __device__ __forceinline__ int first_tile() const { return lo / TILE; }
  template <int TILE> __device__ __forceinline__ int tiles() const { return (hi + TILE - 1) / TILE - lo / TILE; }
};
struct SeqShape {
  int len, new_rows, q_start, targets, rows;   // rows: new rows times heads of a group
};
__device__ __forceinline__ SeqShape seq_shape(const PagedAttn &a, int b) {
  SeqShape s;
  s.q_start = a.q_offsets[b];
  s.new_rows = min(a.q_offsets[b + 1], (int)a.rows) - s.q_start;
  s.len = min(max(a.lengths[b], 0), 0x7fffffff - 1024);   // (so that no position or tile's end passes 32 bits)
  s.targets = a.targets ? a.targets[b] : 0;
  s.rows = s.new_rows > 0 && s.q_start >= 0 ? s.new_rows * a.group : 0;
  return s;
}
template <int RB>
__device__ __forceinline__ UnitRange unit_range(const PagedAttn &a, const SeqShape &s, int rb) {
  const int i0 = rb * RB / a.group, i1 = (min((rb + 1) * RB, s.rows) - 1) / a.group;
  const int p0 = s.len - s.new_rows + i0, p1 = s.len - s.new_rows + i1;
  UnitRange r{0, PA_BLOCK, 0, 0, 0, 0};
  if (p1 < 0) return r;   // nothing visible: one block, all of it masked
  const RowSees lo = row_sees(max(p0, 0), s.len, s.targets, a.c, a.W), hi = row_sees(p1, s.len, s.targets, a.c, a.W);
  const int end = min(max(max(lo.hi, hi.hi), p1 + 1), a.cache.positions());
  if (lo.lo >= end) return r;
  r.begin = lo.lo;
  r.end = end;
  r.lo = lo.lo / PA_BLOCK * PA_BLOCK;
  r.hi = (end + PA_BLOCK - 1) / PA_BLOCK * PA_BLOCK;
  r.all_lo = hi.lo;
  // (a row that is no candidate sees itself right behind the rest)
  r.all_hi = min(lo.hi + (lo.hi == lo.self), hi.hi + (hi.hi == hi.self));
  if (p0 < a.c) r.all_hi = p0 < 0 ? 0 : min(r.all_hi, a.c + 1);
  r.all_hi = min(r.all_hi, end);
  return r;
}
template <int RB>
__device__ __forceinline__ int blocks_of_rows(const SeqShape &s) { return (s.rows + RB - 1) / RB; }
// The work of a sequence: its units' tiles, or its units where CTAs take whole ones.
template <int RB, int TILE>
__device__ __forceinline__ int64_t seq_work(const PagedAttn &a, int b) {
  const SeqShape s = seq_shape(a, b);
  if (a.whole_units) return (int64_t)blocks_of_rows<RB>(s) * a.cache.H;
  int64_t n = 0;
  for (int rb = 0; rb < blocks_of_rows<RB>(s); ++rb) n += unit_range<RB>(a, s, rb).template tiles<TILE>();
  return n * a.cache.H;
}

// CTA c of G takes tiles (or units) [W c / G, W (c + 1) / G); the CTA that tile t belongs to:
__device__ __forceinline__ int64_t first_tile(int64_t W, int c, int G) { return W * c / G; }
__device__ __forceinline__ int cta_of_tile(int64_t W, int64_t t, int G) { return (int)(((t + 1) * G - 1) / W); }


// The unit that a CTA is at, of those it has tiles of: sequence b, block of rows rb, head h; `tile` is the next of
// the unit's `tiles`, `here` the number that are this CTA's.
template <int RB, int TILE>
struct Walk {
  SeqShape seq;
  UnitRange range;
  int b, rb, h, tile, tiles, here;
  int64_t unit_begin, left;   // the unit's first tile of all; work of this CTA from here on

  __device__ __forceinline__ void take(const PagedAttn &a) {
    here = a.whole_units ? tiles : (int)min(left, (int64_t)(tiles - tile));
  }
  // the next unit; false where the CTA has no more
  __device__ __forceinline__ bool next(const PagedAttn &a) {
    left -= a.whole_units ? 1 : here;
    if (left <= 0) return false;
    unit_begin += tiles;
    tile = 0;
    if (++h == a.cache.H) {
      h = 0;
      if (++rb >= blocks_of_rows<RB>(seq)) {
        rb = 0;
        do seq = seq_shape(a, ++b);
        while (seq.rows == 0);
      }
      range = unit_range<RB>(a, seq, rb);
      tiles = range.template tiles<TILE>();
    }
    take(a);
    return true;
  }
  __device__ __forceinline__ bool whole() const { return tile == 0 && here == tiles; }
  __device__ __forceinline__ int slot() const { return tile > 0 ? 0 : 1; }
};

template <int WARPS>
struct RunSmem {
  int64_t sum[WARPS];
  int64_t start[2];
};
// The whole CTA: the work there is, the CTAs that have some (returned; 0 for one that has none), and where this one
// begins.
template <int RB, int TILE, int WARPS>
__device__ __forceinline__ int find_run(const PagedAttn &a, RunSmem<WARPS> &s, int64_t &total, Walk<RB, TILE> &walk) {
  constexpr int THREADS = 32 * WARPS;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t first = tid < a.cache.B ? seq_work<RB, TILE>(a, tid) : 0;   // (kept: mostly there are no others)
  int64_t mine = first;
  for (int b = tid + THREADS; b < a.cache.B; b += THREADS) mine += seq_work<RB, TILE>(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) s.sum[warp] = mine;
  if (tid == 0) a.joins[2 * blockIdx.x] = make_int4(-1, 0, 0, 0);
  __syncthreads();
  total = 0;
  for (int w = 0; w < WARPS; ++w) total += s.sum[w];
  const int G = (int)min((int64_t)gridDim.x, total);   // (every CTA below this has work)
  if ((int)blockIdx.x >= G) return 0;
  const int64_t begin = first_tile(total, blockIdx.x, G);
  walk.left = first_tile(total, blockIdx.x + 1, G) - begin;
  int64_t before = 0;
  for (int base = 0; base < a.cache.B; base += THREADS) {
    const int b = base + tid;
    const int64_t n = base == 0 ? first : b < a.cache.B ? seq_work<RB, TILE>(a, b) : 0;
    int64_t upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();
    if (lane == 31) s.sum[warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += s.sum[w];
    upto += before;
    if (n > 0 && begin < upto && begin >= upto - n) {
      s.start[0] = b;
      s.start[1] = begin - (upto - n);
    }
    for (int w = 0; w < WARPS; ++w) before += s.sum[w];
    if (before > begin) break;
  }
  __syncthreads();
  walk.b = (int)s.start[0], walk.rb = 0;
  int64_t into = s.start[1];
  walk.seq = seq_shape(a, walk.b);
  if (a.whole_units) {
    walk.rb = (int)(into / a.cache.H);
    walk.range = unit_range<RB>(a, walk.seq, walk.rb);
    walk.tiles = walk.range.template tiles<TILE>();
    walk.h = (int)(into - (int64_t)walk.rb * a.cache.H), walk.tile = 0;
    walk.unit_begin = 0;   // (nobody asks)
  } else {
    walk.range = unit_range<RB>(a, walk.seq, 0);
    walk.tiles = walk.range.template tiles<TILE>();
    while (into >= (int64_t)walk.tiles * a.cache.H) {
      into -= (int64_t)walk.tiles * a.cache.H;
      walk.range = unit_range<RB>(a, walk.seq, ++walk.rb);
      walk.tiles = walk.range.template tiles<TILE>();
    }
    walk.h = (int)(into / walk.tiles), walk.tile = (int)(into - (int64_t)walk.h * walk.tiles);
    walk.unit_begin = begin - walk.tile;
  }
  walk.take(a);
  return G;
}
// One thread: where the CTA is the first to go on with a unit that another one began, it says so to the join.
template <int RB, int TILE>
__device__ __forceinline__ void leave_join(const PagedAttn &a, const Walk<RB, TILE> &w, int64_t total, int G) {
  if (w.whole() || w.slot() != 0) return;
  const int c0 = cta_of_tile(total, w.unit_begin, G), c1 = cta_of_tile(total, w.unit_begin + w.tiles - 1, G);
  if (c0 + 1 != (int)blockIdx.x) return;
  a.joins[2 * blockIdx.x] = make_int4(c1, min(RB, w.seq.rows - w.rb * RB), w.h, w.rb * RB);
  a.joins[2 * blockIdx.x + 1] = make_int4(w.seq.q_start, 0, 0, 0);
}
// rows of q that no sequence has, before the first offset and past the last: zeros
template <typename T, int D, int THREADS>
__device__ __forceinline__ void clear_rows_of_nobody(const PagedAttn &a) {
  const int64_t row = (int64_t)a.Hq * D;
  const int64_t before = a.cache.B > 0 ? min((int64_t)max(0, a.q_offsets[0]), a.rows) * row : 0;
  const int64_t from = a.cache.B > 0 ? max(0, a.q_offsets[a.cache.B]) * row : 0;
  for (int64_t x = (int64_t)blockIdx.x * THREADS + threadIdx.x; x < before + a.rows * row - from;
       x += (int64_t)gridDim.x * THREADS)
    static_cast<T *>(a.out)[x < before ? x : x - before + from] = from_f32<T>(0.f);
}

// ---------------------------------------------------------------------------------------
// numbers
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Codes to numbers; the kernel's instructions are mostly these.
// (x & MASK) | BITS in one operation: left to itself the compiler takes two
template <uint32_t MASK, uint32_t BITS>
__device__ __forceinline__ uint32_t masked_or(uint32_t x) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "n"(MASK), "r"(BITS));
  return r;
}
// float16: a code in the low bits of 1024's mantissa is 1024 + code (the usual way to a float without a conversion),
// four bits further up 1024 + 16 code - pairs 0 and 1 of `x` without a shift, 2 and 3 of x >> 8.  Pair i holds codes i and i + 4.
__device__ __forceinline__ uint32_t k_pair(uint32_t x, bool up) {
  return up ? masked_or<0x00f000f0u, 0x64006400u>(x) : masked_or<0x000f000fu, 0x64006400u>(x);
}
__device__ __forceinline__ uint32_t k_exact(uint32_t pair, bool up) {   // code - 8, or 16 (code - 8)
  const __half2 off = up ? __half2half2(__ushort_as_half(0x6480)) : __half2half2(__ushort_as_half(0x6408));   // 1152, 1032
  __half2 h = __hsub2(*reinterpret_cast<__half2 *>(&pair), off);
  return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

int paged_attn_tc(const PagedAttn &a, bool bf16, bool softmax, int grid, cudaStream_t st);

}  // namespace b200hstu
