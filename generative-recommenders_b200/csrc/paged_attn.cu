// Attention of new rows over the paged 4-bit K / V cache.
//
//   out[i] = sum_j mask(i, j) f(alpha <q_i, k_j>) v_j,   f = SiLU * scale or softmax over the visible j
//
// Codes are small whole numbers, so the products run on the tensor cores without rounding them:
// k_j = s_j (c_j - 8) for every group of 64 values, hence <q, k_j> = sum over groups of s_j <q, c_j - 8>, the
// scales entering in fp32 after the product; sum_j p_j v_j = sum_j (p_j s_j) (c_j - 8), the scales entering the
// weights before they are rounded.
//
// One row per user is bound by the cache's bytes.  The work is cut into equal runs of 64 positions over all
// (sequence, block of rows, head) units, however long each is, one run per CTA; a unit that several CTAs share
// leaves partial results, which paged_attn_join_kernel adds up in order.
#include "paged_attn.cuh"

#include <atomic>

namespace b200hstu {

namespace {

constexpr int PA_THREADS = 128, PA_WARPS = 4;
constexpr int PA_STAGES = 2;       // tiles of a warp in shared memory
constexpr int PA_TILE = 64;        // positions that work is cut at
constexpr int JOIN_PARTS = 16;     // of a unit's pieces, added up side by side
constexpr int JOIN_FEW = 4;        // up to so many pieces, rows are side by side

// ---------------------------------------------------------------------------------------
// fragments
// ---------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// For the second, bfloat16 (weights may have any size): 128 + code, less 136 (exact).
__device__ __forceinline__ uint32_t v_pair(uint32_t x) { return masked_or<0x000f000fu, 0x43004300u>(x); }
__device__ __forceinline__ uint32_t v_exact(uint32_t raw) {
  const __nv_bfloat162 off = __halves2bfloat162(__ushort_as_bfloat16(0x4308), __ushort_as_bfloat16(0x4308));
  __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162 *>(&raw), off);
  return *reinterpret_cast<uint32_t *>(&v);
}
// contiguous bytes (a multiple of 16) into shared memory, counted by an mbarrier
__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// Row r of a product's 16 (the keys of a block) is position key_of(r) of it: of the pairs of rows that a warp reads
// for the second product no more than two meet in a bank.
__device__ __forceinline__ int key_of(int r) {
  const int x = (r >> 1) & 3;
  return (r & 8) + ((r & 1) ? 4 + ((x + 2) & 3) : x);
}

// the scales of one key
template <int G64>
__device__ __forceinline__ void load_scales(const uint8_t *p, float (&s)[G64]) {
  if constexpr (G64 == 1) {
    s[0] = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t *>(p) << 16);
  } else {
#pragma unroll
    for (int w = 0; w < G64; w += 2) {
      const uint32_t two = *reinterpret_cast<const uint32_t *>(p + 2 * w);
      s[w] = __uint_as_float(two << 16);
      s[w + 1] = __uint_as_float(two & 0xffff0000u);
    }
  }
}

// float16 numbers that add up to a value of q (of a row scaled by a power of two to at most 1), and bfloat16
// ones that add up to a weight.  bfloat16 for weights because they may have any size; two of them for 16-bit results,
// too, because the rounding of a single one would be as large as the result's own (512 users' step: 5 % of the time).
template <typename T> struct Terms;
template <> struct Terms<__nv_bfloat16> { static constexpr int Q = 1, P = 2; static constexpr bool BF16 = true; };
template <> struct Terms<__half> { static constexpr int Q = 1, P = 2; static constexpr bool BF16 = false; };
template <> struct Terms<float> { static constexpr int Q = 3, P = 3; };

// ---------------------------------------------------------------------------------------
// few rows of a unit at a time: NT * 8, or one (NT = 0)
// ---------------------------------------------------------------------------------------
// The first product is K Q^T (16 keys x 8 rows), so that a row of q costs an eighth of an instruction and not a
// sixteenth of a twice as large one; its result, transposed in 8 x 8 blocks, is the second operand of
// V^T P^T (16 values x 8 rows).  Each warp takes tiles of its own and has its own two stages, filled by bulk copies
// that it asks for itself: no warp waits for another until the unit's end.
//
// One row (a step of a model without shared heads): the eight columns are copies of it, so every lane has the scores
// of its keys whatever column it stands for, and the four lanes that share keys take a block of the tile each: a
// score's scales, mask, exponential and weight are worked out once, not eight times.
//
// What bounds it where there is work enough is not the bytes (47 % of DRAM's time) but short dependent chains at 2.7
// warps a scheduler, with the pipe of the logic operations, most of them codes to numbers, busy 52 % of the time and
// issue slots 51 %; elsewhere the way to the first tile and the joining.
// Measured with the call and the join, heads of 128, bf16: one row of each of 512 users, 0.50 GB of cache, 155 - 160 us
// (3.2 TB/s); of 32 users of 16384 each 77 us (3.7 TB/s), with 8 rows each 96 us, with 16 134 us; a history of 200001
// with four rows for each of 2 key heads 34 us (1.6 TB/s).
template <typename T, int D, int NT, bool SOFTMAX>
__global__ void __launch_bounds__(PA_THREADS) paged_attn_kernel(PagedAttn a) {
  constexpr bool ONE = NT == 0;
  constexpr int N = ONE ? 1 : NT, RB = ONE ? 1 : 8 * NT, G64 = D / 64, QT = Terms<T>::Q, PT = Terms<T>::P;
  constexpr bool EXACT = QT > 2;                      // codes less 8 in all of the first product
  constexpr int TK = D == 256 ? 32 : 64, BLOCKS = TK / PA_BLOCK;            // positions and blocks of a stage
  constexpr int STEP = ONE ? BLOCKS : 2;                                   // blocks whose weights are made together
  constexpr int ROW = D / 2, SROW = 2 * G64;                               // bytes of a position's codes and scales
  constexpr int V_AT = TK * ROW, KS_AT = 2 * V_AT, VS_AT = KS_AT + TK * SROW, STAGE = VS_AT + TK * SROW;
  constexpr int RING = PA_STAGES * STAGE, PITCH = D + 4;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t s_full[PA_WARPS][PA_STAGES];
  __shared__ RunSmem<PA_WARPS> s_run;
  __shared__ float s_ml[PA_WARPS][RB][2];
  __shared__ int s_sees[RB][3];
  __shared__ int s_abort;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;

  ptx::allow_dependents();
  clear_rows_of_nobody<T, D, PA_THREADS>(a);
  if (lane == 0) {
    for (int x = 0; x < PA_STAGES; ++x) ptx::mbar_init(ptx::smem_u32(&s_full[warp][x]), 1);
    ptx::fence_mbar_init();
  }
  if (tid == 0) {
    s_abort = 0;
    if (blockIdx.x == 0) *a.status = 0;   // (a wait gives up seconds after this)
  }
  int64_t total;
  Walk<RB, PA_TILE> walk;
  const int G = find_run(a, s_run, total, walk);
  if (G == 0) return;

  uint8_t *ring = smem + warp * RING;
  const uint32_t ring32 = ptx::smem_u32(ring), full32 = ptx::smem_u32(&s_full[warp][0]);
  const ptx::WaitCtx wait{&s_abort, a.status};
  uint32_t asked = 0, taken = 0;       // stages that this warp has asked for and waited for
  // where this lane finds its operands in a block
  const int key0 = key_of(g), k_at = key0 * ROW + 8 * t, s_at = key0 * SROW;
  const int v_at[2] = {key_of(2 * t) * ROW + 4 * g, key_of(2 * t + 1) * ROW + 4 * g};

  // ------------------------------------------------------------------ units
  while (true) {
    const SeqShape &seq = walk.seq;
    const UnitRange &range = walk.range;
    const int r0 = walk.rb * RB, nrows = min(RB, seq.rows - r0), h = walk.h;

    // ---------------------------------------------------------------- this warp's stages of the piece
    const int from = max(range.lo, (range.first_tile<PA_TILE>() + walk.tile) * PA_TILE) / TK;              // stages of the piece: TK
    const int to = (min(range.hi, (range.first_tile<PA_TILE>() + walk.tile + walk.here) * PA_TILE) + TK - 1) / TK;   // positions from TK x on
    const int first = from + (to - from) * warp / PA_WARPS, last = from + (to - from) * (warp + 1) / PA_WARPS;
    int64_t entry = -1;          // page first_page + lane
    int first_page = -64;
    auto request = [&](int x) {
      if (x >= last) return;
      const uint32_t stage = asked++ % PA_STAGES, bar = full32 + 8 * stage;
      // a lane for each run of positions on one page, and of these for K's and V's codes and scales
      const int shift = a.cache.page_shift, run = lane >> 2, part = lane & 3;
      const int lo = max(max(range.lo, x * TK), ((x * TK >> shift) + run) << shift);
      const int hi = min(min(range.hi, x * TK + TK), ((x * TK >> shift) + run + 1) << shift);
      const bool on = lane < 16 && lo < hi;
      const int last_page = (min(range.hi, x * TK + TK) - 1) >> shift;
      if (last_page - first_page >= 32) {
        first_page = x * TK >> shift;
        entry = a.cache.page_of(walk.b, (int64_t)(first_page + lane) << shift);
      }
      const int64_t page = __shfl_sync(0xffffffffu, entry, on ? (lo >> shift) - first_page : 0);
      const int bytes = on && page >= 0 ? (hi - lo) * (part < 2 ? ROW : SROW) : 0;
      const uint32_t at = part == 0 ? 0 : part == 1 ? V_AT : part == 2 ? KS_AT : VS_AT;
      const uint32_t dst = ring32 + stage * STAGE + at + (lo - x * TK) * (part < 2 ? ROW : SROW);
      if (on && page < 0 && part == 2) {   // no such page: whoever sees these positions gets NaN
        for (int y = 0; y < (hi - lo) * SROW / 4; ++y)
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(dst + 4 * y), "r"(0x7fff7fffu) : "memory");
        ptx::fence_proxy_async();
      }
      const uint32_t sum = __reduce_add_sync(0xffffffffu, (uint32_t)bytes);
      if (lane == 0) ptx::mbar_arrive_expect_tx(bar, sum);
      __syncwarp();
      if (bytes > 0) {
        const int place = lo & ((1 << shift) - 1);
        const uint8_t *src = a.cache.page(page, h) + (part < 2 ? a.cache.codes_at(part) + place * ROW
                                                               : a.cache.scales_at(part - 2) + place * SROW);
        bulk_load(dst, src, bytes, bar);
      }
    };
#pragma unroll
    for (int x = 0; x < PA_STAGES; ++x) request(first + x);

    // q as the second operand of the first product: row g of every eight, values 64 w + 16 t + 8 j + ..; scaled by
    // a power of two to at most 1, odd pairs by another sixteenth (k_pair)
    uint32_t qf[N][G64][4][2][QT];
    float qoff[N][G64][2], mul[N][2];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int r = ONE ? r0 : r0 + n * 8 + g;
      const bool on = ONE || n * 8 + g < nrows;
      const int i = on ? r / a.group : 0;
      const T *qr = static_cast<const T *>(a.q) + (int64_t)(seq.q_start + i) * a.q_rs +
                    (int64_t)(h * a.group + (on ? r - i * a.group : 0)) * a.q_hs;
      float f[G64][2][8], most = 0.f;
#pragma unroll
      for (int w = 0; w < G64; ++w)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const T *p = qr + 64 * w + 16 * t + 8 * j;
          if (a.q_vec) {
            uint4 raw[sizeof(T) / 2];
#pragma unroll
            for (int x = 0; x < (int)sizeof(T) / 2; ++x) raw[x] = __ldg(reinterpret_cast<const uint4 *>(p) + x);
#pragma unroll
            for (int x = 0; x < 8; ++x) f[w][j][x] = to_f32(reinterpret_cast<const T *>(raw)[x]);
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x) f[w][j][x] = to_f32(p[x]);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            if (!on) f[w][j][x] = 0.f;
            most = fmaxf(most, fabsf(f[w][j][x]));
          }
        }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      // 2^e with most <= 2^e, both it and its inverse normal numbers (infinities and NaN go their way)
      const int e = min(max((__float_as_int(most) >> 23) - 126, -125), 125);
      const float down = __int_as_float((127 - e) << 23);
#pragma unroll
      for (int y = 0; y < 2; ++y)
        mul[n][y] = __int_as_float((127 + __shfl_sync(0xffffffffu, e, 8 * t + 4 * y)) << 23) * a.alpha *
                    (SOFTMAX ? 1.4426950408889634f : 1.f);
#pragma unroll
      for (int w = 0; w < G64; ++w) {
        float off = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            f[w][j][x] *= down;
            if (x & 1) off -= f[w][j][x] * 72.f, f[w][j][x] *= 0.0625f;   // of 64 + code
          }
#pragma unroll
          for (int term = 0; term < QT; ++term) {
#pragma unroll
            for (int p2 = 0; p2 < 2; ++p2) {
              qf[n][w][2 * j + p2][0][term] = pack_f16(f[w][j][2 * p2], f[w][j][2 * p2 + 4]);
              qf[n][w][2 * j + p2][1][term] = pack_f16(f[w][j][2 * p2 + 1], f[w][j][2 * p2 + 5]);
            }
#pragma unroll
            for (int x = 0; x < 8; ++x) f[w][j][x] -= __half2float(__float2half_rn(f[w][j][x]));
          }
        }
        off += __shfl_xor_sync(0xffffffffu, off, 1);
        off += __shfl_xor_sync(0xffffffffu, off, 2);
        qoff[n][w][0] = __shfl_sync(0xffffffffu, off, 8 * t);
        qoff[n][w][1] = __shfl_sync(0xffffffffu, off, 8 * t + 4);
      }
    }
    RowSees one{0, 0, -1};
    if (ONE) {
      one = row_sees(seq.len - seq.new_rows + r0 / a.group, seq.len, seq.targets, a.c, a.W);
    } else {
      if (tid < RB) {
        const RowSees s = tid < nrows ? row_sees(seq.len - seq.new_rows + (r0 + tid) / a.group, seq.len, seq.targets, a.c, a.W)
                                      : RowSees{0, 0, -1};
        s_sees[tid][0] = s.lo;
        s_sees[tid][1] = s.hi;
        s_sees[tid][2] = s.self;
      }
      __syncthreads();
    }

    float o[N][G64][4][4], top[N][2], sum[N][2];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      top[n][0] = top[n][1] = -3.0e38f;
      sum[n][0] = sum[n][1] = 0.f;
#pragma unroll
      for (int w = 0; w < G64; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[n][w][i][x] = 0.f;
    }
    // a higher reference for column y's weights (as a power of two)
    auto raise = [&](int n, int y, float m) {
      m = fmaxf(top[n][y], m);
      const float old = ex2(top[n][y] - m);
      top[n][y] = m;
      sum[n][y] *= old;
#pragma unroll
      for (int w = 0; w < G64; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][w][i][y] *= old, o[n][w][i][y + 2] *= old;
    };

    for (int x = first; x < last; ++x) {
      const uint32_t stage = taken % PA_STAGES;
      ptx::mbar_wait(wait, full32 + 8 * stage, (taken / PA_STAGES) & 1, 951);
      ++taken;
      const uint8_t *tile_st = ring + stage * STAGE;
      const int tile_pos = x * TK;
      const bool masked = tile_pos < range.all_lo || tile_pos + TK > range.all_hi;
#pragma unroll
      for (int step = 0; step < BLOCKS / STEP; ++step) {
        const uint8_t *st = tile_st + step * STEP * PA_BLOCK * ROW, *sc = tile_st + KS_AT + step * STEP * PA_BLOCK * SROW;
        const int pos0 = tile_pos + step * STEP * PA_BLOCK;
        if (pos0 >= range.hi || pos0 + STEP * PA_BLOCK <= range.lo) continue;
        // ---------------------------------------------------------- scores
        float acc[STEP][N][G64][4];
#pragma unroll
        for (int bl = 0; bl < STEP; ++bl) {
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int w = 0; w < G64; ++w)
#pragma unroll
              for (int y = 0; y < 4; ++y) acc[bl][n][w][y] = EXACT ? 0.f : qoff[n][w][y & 1];
#pragma unroll
          for (int w = 0; w < G64; ++w) {
            const uint2 c0 = *reinterpret_cast<const uint2 *>(st + bl * PA_BLOCK * ROW + k_at + 32 * w);
            const uint2 c1 = *reinterpret_cast<const uint2 *>(st + bl * PA_BLOCK * ROW + k_at + 32 * w + 8 * ROW);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
#pragma unroll
              for (int p2 = 0; p2 < 2; ++p2) {
                const uint32_t x0 = (j ? c0.y : c0.x) >> (8 * p2), x1 = (j ? c1.y : c1.x) >> (8 * p2);
                uint32_t f[4] = {k_pair(x0, false), k_pair(x1, false), k_pair(x0, true), k_pair(x1, true)};
                // (1024 + code less 1032 before the product: the sum would lose 2^-18 of its terms' size to the 1024; the
                // 64 of the others, which is left to it, costs 2^-21.  1 - 3 % of the time, 3 - 10 % with the others too)
#pragma unroll
                for (int y = 0; y < (EXACT ? 4 : 2); ++y) f[y] = k_exact(f[y], y >= 2);
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                  for (int term = QT - 1; term >= 0; --term)
                    mma_f16(acc[bl][n][w], f, qf[n][w][2 * j + p2][0][term], qf[n][w][2 * j + p2][1][term]);
              }
            }
          }
        }
        // ---------------------------------------------------------- weights, times V's scales
        uint32_t pf[STEP][N][G64][2][PT];   // second operand of the second product: rows g, keys 2 t, 2 t + 1 (+ 8)
        if constexpr (ONE) {
          // this lane's scores: of block t (of t & 1 where a tile has two), keys key0 and key0 + 8
          constexpr int MINE = BLOCKS - 1;
          const int blk = t & MINE, mypos = pos0 + blk * PA_BLOCK + key0;
          float s[2], p[2], vs[2][G64];
          bool seen[2] = {true, true};
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float ks[G64];
            load_scales<G64>(sc + blk * PA_BLOCK * SROW + s_at + y * 8 * SROW, ks);
            load_scales<G64>(sc + (VS_AT - KS_AT) + blk * PA_BLOCK * SROW + s_at + y * 8 * SROW, vs[y]);
            s[y] = 0.f;
#pragma unroll
            for (int w = 0; w < G64; ++w) {
              float v = acc[0][0][w][2 * y];
#pragma unroll
              for (int bl = 1; bl < BLOCKS; ++bl) v = blk == bl ? acc[bl][0][w][2 * y] : v;
              s[y] += v * ks[w];
            }
            s[y] *= mul[0][0];
            if (masked) {
              seen[y] = one(mypos + 8 * y);
              if (SOFTMAX && !seen[y]) s[y] = -INFINITY;
            }
          }
          if (SOFTMAX) {
            float m = fmaxf(s[0], s[1]);
            if (__any_sync(0xffffffffu, m > top[0][0] + 8.f)) {   // (2^8 does no harm to a sum)
#pragma unroll
              for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
              raise(0, 0, m);
            }
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            p[y] = SOFTMAX ? ex2(s[y] - top[0][0]) : siluf_(s[y]);
            if (SOFTMAX && (BLOCKS == 4 || t < BLOCKS)) sum[0][0] += p[y];
          }
          // two groups' weights of a key in a register, as bfloat16; then to the lanes that multiply with them
          constexpr int PAIRS = (G64 + 1) / 2;
          float x4[2][2 * PAIRS];
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int w = 0; w < 2 * PAIRS; ++w)
              x4[y][w] = w < G64 && (!masked || seen[y]) ? p[y] * vs[y][w < G64 ? w : 0] : 0.f;
#pragma unroll
          for (int term = 0; term < PT; ++term) {
            uint32_t two[2][PAIRS];
#pragma unroll
            for (int y = 0; y < 2; ++y)
#pragma unroll
              for (int w = 0; w < PAIRS; ++w) {
                two[y][w] = pack_bf16(x4[y][2 * w], x4[y][2 * w + 1]);
                if (term + 1 < PT) {
                  x4[y][2 * w] -= __uint_as_float(two[y][w] << 16);
                  x4[y][2 * w + 1] -= __uint_as_float(two[y][w] & 0xffff0000u);
                }
              }
#pragma unroll
            for (int bl = 0; bl < BLOCKS; ++bl)
#pragma unroll
              for (int y = 0; y < 2; ++y)
#pragma unroll
                for (int w = 0; w < PAIRS; ++w) {
                  const uint32_t k0 = __shfl_sync(0xffffffffu, two[y][w], 8 * t + bl);
                  const uint32_t k1 = __shfl_sync(0xffffffffu, two[y][w], 8 * t + 4 + bl);
                  pf[bl][0][2 * w][y][term] = __byte_perm(k0, k1, 0x5410);
                  if (2 * w + 1 < G64) pf[bl][0][2 * w + 1][y][term] = __byte_perm(k0, k1, 0x7632);
                }
          }
        } else {
          float s[STEP][N][4], vs[STEP][2][G64];
          uint32_t seen[STEP];
#pragma unroll
          for (int bl = 0; bl < STEP; ++bl) {
            float ks[2][G64];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              load_scales<G64>(sc + bl * PA_BLOCK * SROW + s_at + y * 8 * SROW, ks[y]);
              load_scales<G64>(sc + (VS_AT - KS_AT) + bl * PA_BLOCK * SROW + s_at + y * 8 * SROW, vs[bl][y]);
            }
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                float v = acc[bl][n][0][y] * ks[y >> 1][0];
#pragma unroll
                for (int w = 1; w < G64; ++w) v += acc[bl][n][w][y] * ks[y >> 1][w];
                s[bl][n][y] = v * mul[n][y & 1];
              }
            seen[bl] = 0;
            if (masked) {
#pragma unroll
              for (int n = 0; n < N; ++n)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                  const int *r = s_sees[n * 8 + 2 * t + (y & 1)], pos = pos0 + bl * PA_BLOCK + key0 + 8 * (y >> 1);
                  const bool v = (pos >= r[0] && pos < r[1]) || pos == r[2];
                  seen[bl] |= (uint32_t)v << (4 * n + y);
                  if (SOFTMAX && !v) s[bl][n][y] = -INFINITY;
                }
            }
          }
          if (SOFTMAX) {
            bool higher = false;
            float m[N][2];
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                m[n][y] = fmaxf(s[0][n][y], s[0][n][y + 2]);
#pragma unroll
                for (int bl = 1; bl < STEP; ++bl) m[n][y] = fmaxf(m[n][y], fmaxf(s[bl][n][y], s[bl][n][y + 2]));
                higher |= m[n][y] > top[n][y] + 8.f;   // (2^8 does no harm to a sum)
              }
            if (__any_sync(0xffffffffu, higher)) {
#pragma unroll
              for (int n = 0; n < N; ++n)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
#pragma unroll
                  for (int d = 4; d < 32; d <<= 1) m[n][y] = fmaxf(m[n][y], __shfl_xor_sync(0xffffffffu, m[n][y], d));
                  raise(n, y, m[n][y]);
                }
            }
          }
#pragma unroll
          for (int bl = 0; bl < STEP; ++bl)
#pragma unroll
            for (int n = 0; n < N; ++n) {
              float p[4], x4[G64][4];
#pragma unroll
              for (int y = 0; y < 4; ++y) {
                if (SOFTMAX) {
                  p[y] = ex2(s[bl][n][y] - top[n][y & 1]);
                  sum[n][y & 1] += p[y];
                } else {
                  p[y] = siluf_(s[bl][n][y]);
                }
#pragma unroll
                for (int w = 0; w < G64; ++w) x4[w][y] = p[y] * vs[bl][y >> 1][w];
              }
              if (masked) {   // (what lies in unseen places may be no number)
#pragma unroll
                for (int w = 0; w < G64; ++w)
#pragma unroll
                  for (int y = 0; y < 4; ++y) x4[w][y] = (seen[bl] >> (4 * n + y)) & 1 ? x4[w][y] : 0.f;
              }
#pragma unroll
              for (int w = 0; w < G64; ++w)
#pragma unroll
                for (int term = 0; term < PT; ++term)
#pragma unroll
                  for (int y = 0; y < 2; ++y) {
                    const uint32_t two = pack_bf16(x4[w][2 * y], x4[w][2 * y + 1]);
                    pf[bl][n][w][y][term] = transposed8x8(two);
                    if (term + 1 < PT) {
                      x4[w][2 * y] -= __uint_as_float(two << 16);
                      x4[w][2 * y + 1] -= __uint_as_float(two & 0xffff0000u);
                    }
                  }
            }
        }
        // ---------------------------------------------------------- second product
#pragma unroll
        for (int bl = 0; bl < STEP; ++bl)
#pragma unroll
          for (int w = 0; w < G64; ++w) {
            uint32_t c[4];   // eight codes 64 w + 8 g .. of the keys of rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
            for (int y = 0; y < 4; ++y)
              c[y] = *reinterpret_cast<const uint32_t *>(st + V_AT + (bl * PA_BLOCK + 8 * (y >> 1)) * ROW + v_at[y & 1] + 32 * w);
            const uint32_t e[4] = {__byte_perm(c[0], c[1], 0x5410), __byte_perm(c[0], c[1], 0x7632),
                                   __byte_perm(c[2], c[3], 0x5410), __byte_perm(c[2], c[3], 0x7632)};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t f[4];
#pragma unroll
              for (int y = 0; y < 4; ++y) f[y] = v_exact(v_pair(e[y] >> (4 * i)));
#pragma unroll
              for (int n = 0; n < N; ++n)
#pragma unroll
                for (int term = PT - 1; term >= 0; --term)
                  mma_bf16(o[n][w][i], f, pf[bl][n][w][0][term], pf[bl][n][w][1][term]);
            }
          }
      }
      __syncwarp();
      request(x + PA_STAGES);
    }

    // ---------------------------------------------------------------- the warps' results together
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int y = 0; y < (ONE ? 1 : 2); ++y) {
        if (SOFTMAX) {
#pragma unroll
          for (int d = ONE ? 1 : 4; d < 32; d <<= 1) sum[n][y] += __shfl_xor_sync(0xffffffffu, sum[n][y], d);
          if (ONE ? lane == 0 : g == 0) {
            s_ml[warp][ONE ? 0 : n * 8 + 2 * t + y][0] = top[n][y];
            s_ml[warp][ONE ? 0 : n * 8 + 2 * t + y][1] = sum[n][y];
          }
        }
      }
    __syncthreads();   // (the rings are free)
    float *buf = reinterpret_cast<float *>(smem);   // [warp][row][PITCH]
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int w = 0; w < G64; ++w)
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          if (ONE && ((y & 1) || t != 0)) continue;
          *reinterpret_cast<float4 *>(buf + (warp * RB + (ONE ? 0 : n * 8 + 2 * t + (y & 1))) * PITCH + 64 * w + 8 * g +
                                      4 * (y >> 1)) = make_float4(o[n][w][0][y], o[n][w][1][y], o[n][w][2][y], o[n][w][3][y]);
        }
    __syncthreads();
    const bool whole = walk.whole();
    const int slot = walk.slot();
    float *po = a.part_o + ((int64_t)blockIdx.x * 2 + slot) * RB * D;
    float *pml = a.part_ml + ((int64_t)blockIdx.x * 2 + slot) * RB * 2;
    for (int x = tid; x < nrows * (D / 4); x += PA_THREADS) {
      const int r = x / (D / 4), e = x % (D / 4) * 4;
      const RowSees sees = ONE ? one : RowSees{s_sees[r][0], s_sees[r][1], s_sees[r][2]};
      const float none = sees.past(a.cache.positions()) ? __int_as_float(0x7fffffff) : 0.f;
      float m = -3.0e38f, l = 0.f, v[4] = {none, none, none, none};
      if (SOFTMAX) {
#pragma unroll
        for (int w = 0; w < PA_WARPS; ++w) m = fmaxf(m, s_ml[w][r][0]);
      }
#pragma unroll
      for (int w = 0; w < PA_WARPS; ++w) {
        const float f = SOFTMAX ? ex2(s_ml[w][r][0] - m) : 1.f;
        if (SOFTMAX) l += s_ml[w][r][1] * f;
        const float4 y = *reinterpret_cast<const float4 *>(buf + (w * RB + r) * PITCH + e);
        v[0] += y.x * f, v[1] += y.y * f, v[2] += y.z * f, v[3] += y.w * f;
      }
      if (whole) {
        const int i = (r0 + r) / a.group, hq = h * a.group + (r0 + r) - i * a.group;
        const float f = SOFTMAX ? (l == 0.f ? 0.f : 1.f / l) : a.scale;
        T *out = static_cast<T *>(a.out) + ((int64_t)(seq.q_start + i) * a.Hq + hq) * D + e;
        T four[4];
#pragma unroll
        for (int y = 0; y < 4; ++y) four[y] = from_f32<T>(v[y] * f);
        if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<uint4 *>(four);
        else *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<uint2 *>(four);
      } else {
        *reinterpret_cast<float4 *>(po + r * D + e) = make_float4(v[0], v[1], v[2], v[3]);
        if (e == 0) pml[2 * r] = m, pml[2 * r + 1] = l;
      }
    }
    if (tid == 0) leave_join(a, walk, total, G);
    if (!walk.next(a)) break;
    ptx::fence_proxy_async();   // (the copies of the next unit go where `buf` was)
    __syncthreads();
  }
  // after a wait that gave up: the copies still under way, with a limit again
  if (s_abort != 0 && lane == 0) {
    int quiet = 0;
    for (uint32_t x = asked > PA_STAGES ? asked - PA_STAGES : 0; x < asked; ++x)
      ptx::mbar_wait_slow(&quiet, nullptr, full32 + 8 * (x % PA_STAGES), (x / PA_STAGES) & 1, 0);
  }
}

// Adds up the pieces of a unit that CTAs c - 1 (its second slot) to c1 (their first ones) have left, in this order;
// CTA (c, y) takes rows y, y + gridDim.y ..
// Few pieces of many rows are rows side by side (JOIN_FEW; 23 prompts of up to 700 x 4 rows: 9 us, 81 with the pieces
// side by side), many pieces of few rows pieces (the history of 200001: 13 us).
template <typename T, int D, bool SOFTMAX>
__global__ void __launch_bounds__(JOIN_PARTS * (D / 4)) paged_attn_join_kernel(PagedAttn a, int RB) {
  constexpr int LANES = D / 4, WARPS = JOIN_PARTS * LANES / 32;
  __shared__ float s_top[WARPS], s_l[JOIN_PARTS];
  __shared__ float4 s_o[JOIN_PARTS][LANES];
  ptx::grid_dependency_wait();
  const int c = blockIdx.x;
  const int4 j = a.joins[2 * c];
  if (j.x < 0) return;
  const int q_start = a.joins[2 * c + 1].x, lane = threadIdx.x % LANES, part = threadIdx.x / LANES;
  const int pieces = j.x - c + 2, per = (pieces + JOIN_PARTS - 1) / JOIN_PARTS;
  auto slot = [&](int x) { return x == 0 ? (int64_t)(c - 1) * 2 + 1 : (int64_t)(c - 1 + x) * 2; };
  auto write = [&](int r, const float4 &o, float l) {
    const float f = SOFTMAX ? (l == 0.f ? 0.f : 1.f / l) : a.scale;
    const int i = (j.w + r) / a.group, hq = j.z * a.group + (j.w + r) - i * a.group;
    T four[4] = {from_f32<T>(o.x * f), from_f32<T>(o.y * f), from_f32<T>(o.z * f), from_f32<T>(o.w * f)};
    T *out = static_cast<T *>(a.out) + ((int64_t)(q_start + i) * a.Hq + hq) * D + 4 * lane;
    if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(out) = *reinterpret_cast<uint4 *>(four);
    else *reinterpret_cast<uint2 *>(out) = *reinterpret_cast<uint2 *>(four);
  };
  if (pieces <= JOIN_FEW) {   // few pieces: rows side by side instead
    for (int r = blockIdx.y * JOIN_PARTS + part; r < j.y; r += gridDim.y * JOIN_PARTS) {
      float4 o[JOIN_FEW];
      float2 ml[JOIN_FEW];
#pragma unroll
      for (int x = 0; x < JOIN_FEW; ++x) {
        ml[x] = make_float2(-3.0e38f, 0.f);
        o[x] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (x >= pieces) continue;
        const int64_t at = slot(x) * RB + r;
        o[x] = *reinterpret_cast<const float4 *>(a.part_o + at * D + 4 * lane);
        if (SOFTMAX) ml[x] = *reinterpret_cast<const float2 *>(a.part_ml + at * 2);
      }
      float m = ml[0].x, l = 0.f;
#pragma unroll
      for (int x = 1; x < JOIN_FEW; ++x) m = fmaxf(m, ml[x].x);
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int x = 0; x < JOIN_FEW; ++x) {
        const float f = SOFTMAX ? ex2(ml[x].x - m) : 1.f;
        l += ml[x].y * f;
        s.x += o[x].x * f, s.y += o[x].y * f, s.z += o[x].z * f, s.w += o[x].w * f;
      }
      write(r, s, l);
    }
    return;
  }
  for (int r = blockIdx.y; r < j.y; r += gridDim.y) {
    float m = -3.0e38f, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (SOFTMAX) {
      for (int x = threadIdx.x; x < pieces; x += JOIN_PARTS * LANES) m = fmaxf(m, a.part_ml[(slot(x) * RB + r) * 2]);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      if (threadIdx.x % 32 == 0) s_top[threadIdx.x / 32] = m;
      __syncthreads();
      for (int x = 0; x < WARPS; ++x) m = fmaxf(m, s_top[x]);
    }
#pragma unroll 4
    for (int x = part * per; x < min((part + 1) * per, pieces); ++x) {
      const int64_t at = slot(x) * RB + r;
      const float4 y = *reinterpret_cast<const float4 *>(a.part_o + at * D + 4 * lane);
      float f = 1.f;
      if (SOFTMAX) {
        const float2 ml = *reinterpret_cast<const float2 *>(a.part_ml + at * 2);
        f = ex2(ml.x - m);
        l += ml.y * f;
      }
      o.x += y.x * f, o.y += y.y * f, o.z += y.z * f, o.w += y.w * f;
    }
    s_o[part][lane] = o;
    if (lane == 0) s_l[part] = l;
    __syncthreads();
    if (part == 0) {
      for (int x = 1; x < JOIN_PARTS; ++x) {
        const float4 y = s_o[x][lane];
        o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
        l += s_l[x];
      }
      write(r, o, l);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------
constexpr int SMS = 148;
constexpr int PA_MAX_CTAS = SMS * 5;
constexpr int PA_MIN_TILES = 2;   // of a CTA, where the cache may be that long
// Positions of a sequence that a CTA does by itself at most, by the width of the table: the lengths are on the device, so
// short sequences under a wide table are cut and joined.  (4 users of up to 700: 10.4 us, 12 when cut and joined; 32
// users of up to 1024 with 20 rows each: 28.7 us and 43.)
constexpr int WHOLE_UP_TO = 1024;

// Rows of a block, in eights: none of them (a single row), some where there are as many and the type's registers
// allow it, or 32, the kernel of paged_attn_sm100.cu, from TC_FROM rows a sequence on (32 users with 20 rows
// each: 28.7 us, 46 in blocks of 16).  Rows a sequence is the mean over all of the batch, those without new rows too.
constexpr int TC_EIGHTS = 32, TC_FROM = 17;
int rows_of(int nt) { return nt == 0 ? 1 : 8 * nt; }
int row_tiles(const b200_hstu_paged_attn_args &p) {
  const int64_t seqs = p.cache.B > 0 ? p.cache.B : 1, rows = (p.rows * (p.Hq / p.cache.H) + seqs - 1) / seqs;
  if (rows <= 1) return 0;
  if (rows >= TC_FROM && p.cache.d <= 128 && p.dtype != B200_HSTU_F32) return TC_EIGHTS;
  const int most = p.cache.d == 256 || p.dtype == B200_HSTU_F32 ? 1 : 2;
  int nt = 1;
  while (nt < most && 8 * nt < rows) nt *= 2;
  return nt;
}
int64_t units_of(const b200_hstu_paged_attn_args &p, int nt) {   // at most
  return ((p.rows < p.cache.B ? p.rows : p.cache.B) + p.rows * (p.Hq / p.cache.H) / rows_of(nt)) * p.cache.H;
}
int most_ctas(int nt) { return nt == TC_EIGHTS ? SMS : PA_MAX_CTAS; }
// Short sequences, and not many: whole units, so that nothing has to be joined.
bool whole_units(const b200_hstu_paged_attn_args &p, int nt) {
  return (int64_t)p.cache.table_width * p.cache.page_size <= WHOLE_UP_TO && units_of(p, nt) <= 2 * most_ctas(nt);
}
int grid_of(const b200_hstu_paged_attn_args &p, int nt) {
  const int64_t units = units_of(p, nt);
  const int64_t tile = nt == TC_EIGHTS ? 128 : PA_TILE, most = most_ctas(nt);
  const int64_t tiles = units * (((int64_t)p.cache.table_width * p.cache.page_size + tile - 1) / tile);
  int64_t n = whole_units(p, nt) ? units : (tiles + PA_MIN_TILES - 1) / PA_MIN_TILES;
  n = n < 1 ? 1 : n;
  return (int)(n < most ? n : most);
}
constexpr int64_t PA_HEADER = 256;
int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// The pieces that `grid` CTAs may have left; it waits for them where they are written, so it may be there early.
template <typename T, int D, bool SOFTMAX>
int launch_join(const PagedAttn &a, int grid, int rows, cudaStream_t st) {
  if (grid <= 1 || a.whole_units) return 0;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid, rows < 8 ? 1 : rows < 128 ? 4 : 16);
  cfg.blockDim = dim3(JOIN_PARTS * (D / 4));
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (int rc = check_cuda(cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<T, D, SOFTMAX>, a, rows), "paged_attn_join_kernel"))
    return rc;
  count_launch();
  return 0;
}

template <typename T, int D, int NT, bool SOFTMAX>
int launch(PagedAttn &a, int grid, cudaStream_t st) {
  constexpr int stage = 2 * (D == 256 ? 32 : 64) * (D / 2 + 2 * (D / 64));
  constexpr int ring = PA_WARPS * PA_STAGES * stage;
  constexpr int merge = (int)sizeof(float) * PA_WARPS * (NT == 0 ? 1 : 8 * NT) * (D + 4);
  constexpr int smem = ring > merge ? ring : merge;
  auto kernel = paged_attn_kernel<T, D, NT, SOFTMAX>;
  if (int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem),
                          "cudaFuncSetAttribute"))   // (of the current device)
    return rc;
  static std::atomic<int> known{0};   // CTAs of an SM
  int resident = known.load(std::memory_order_relaxed);
  if (resident == 0) {
    if (int rc = check_cuda(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, PA_THREADS, smem), "occupancy"))
      return rc;
    resident = resident < 1 ? 1 : resident;
    known.store(resident, std::memory_order_relaxed);
  }
  grid = grid < SMS * resident ? grid : SMS * resident;
  kernel<<<grid, PA_THREADS, smem, st>>>(a);
  count_launch();
  B200_CHECK_LAUNCH("paged_attn_kernel");
  return launch_join<T, D, SOFTMAX>(a, grid, rows_of(NT), st);
}

template <typename T, int D, int NT>
int launch_act(PagedAttn &a, bool softmax, int grid, cudaStream_t st) {
  return softmax ? launch<T, D, NT, true>(a, grid, st) : launch<T, D, NT, false>(a, grid, st);
}
template <typename T, int D>
int launch_rows(PagedAttn &a, bool softmax, int nt, int grid, cudaStream_t st) {
  if (nt == 0) return launch_act<T, D, 0>(a, softmax, grid, st);
  if constexpr (D < 256 && Terms<T>::Q < 3) {
    if (nt == 2) return launch_act<T, D, 2>(a, softmax, grid, st);
    if (nt == TC_EIGHTS) {
      if (int rc = paged_attn_tc(a, Terms<T>::BF16, softmax, grid, st)) return rc;
      return softmax ? launch_join<T, D, true>(a, grid, rows_of(nt), st) : launch_join<T, D, false>(a, grid, rows_of(nt), st);
    }
  }
  return launch_act<T, D, 1>(a, softmax, grid, st);
}
template <typename T>
int launch_dim(PagedAttn &a, bool softmax, int nt, int grid, cudaStream_t st) {
  if (a.cache.d == 64) return launch_rows<T, 64>(a, softmax, nt, grid, st);
  if (a.cache.d == 128) return launch_rows<T, 128>(a, softmax, nt, grid, st);
  return launch_rows<T, 256>(a, softmax, nt, grid, st);
}

bool sizes_ok(const b200_hstu_paged_attn_args &p) {
  return p.rows >= 0 && p.rows < (1ll << 31) && p.Hq > 0 && p.cache.H > 0 && p.Hq % p.cache.H == 0 && p.cache.d > 0 && p.cache.B >= 0 &&
         p.rows * (int64_t)p.Hq < (1ll << 31) && p.cache.table_width >= 0;
}

}  // namespace

int64_t paged_attn_workspace_bytes(const b200_hstu_paged_attn_args &p) {
  if (!sizes_ok(p) || p.rows == 0) return 0;
  const int nt = row_tiles(p), grid = grid_of(p, nt);
  return PA_HEADER + align256((int64_t)grid * 2 * sizeof(int4)) + align256((int64_t)grid * 2 * rows_of(nt) * 2 * sizeof(float)) +
         (int64_t)grid * 2 * rows_of(nt) * p.cache.d * (int64_t)sizeof(float);
}
int paged_attn_status(const b200_hstu_paged_attn_args &p, cudaStream_t st, int32_t *status) {
  *status = 0;
  if (!p.workspace || paged_attn_workspace_bytes(p) == 0) return 0;
  if (int rc = check_cuda(cudaMemcpyAsync(status, p.workspace, sizeof(int32_t), cudaMemcpyDeviceToHost, st), "status")) return rc;
  return check_cuda(cudaStreamSynchronize(st), "status");
}

int paged_attn_fwd(const b200_hstu_paged_attn_args &p, cudaStream_t st) {
  PagedAttn a = {};
  if (int rc = check_paged_cache("paged_attn", p.cache, a.cache)) return rc;
  if (p.rows < 0 || p.rows >= (1ll << 31) || p.rows * (int64_t)p.Hq >= (1ll << 31)) return fail(B200_HSTU_EINVAL, "paged_attn: bad number of rows");
  if (p.Hq <= 0 || p.Hq % p.cache.H != 0)
    return fail(B200_HSTU_EINVAL, "paged_attn: %d query heads on %d heads of the cache", p.Hq, p.cache.H);
  if (p.max_attn_len < 0 || p.contextual_seq_len < 0)
    return fail(B200_HSTU_EINVAL, "paged_attn: negative max_attn_len / contextual_seq_len");
  if (p.dtype != B200_HSTU_F32 && p.dtype != B200_HSTU_BF16 && p.dtype != B200_HSTU_F16)
    return fail(B200_HSTU_EINVAL, "unknown dtype %d", p.dtype);
  if (p.rows == 0) return 0;
  if (!p.q || !p.out || !p.q_offsets || (p.cache.B > 0 && !p.seq_lengths))
    return fail(B200_HSTU_EINVAL, "paged_attn: null tensor");
  if ((((uintptr_t)p.out | (uintptr_t)p.workspace) & 15) != 0)
    return fail(B200_HSTU_EINVAL, "paged_attn: out and workspace must be 16-byte aligned");
  a.q = p.q;
  a.out = p.out;
  a.lengths = {p.seq_lengths, (p.index_flags & B200_HSTU_LENGTHS_I64) ? 2 : 1};
  a.q_offsets = {p.q_offsets, (p.index_flags & B200_HSTU_OFFSETS_I64) ? 2 : 1};
  a.targets = {p.num_targets, (p.index_flags & B200_HSTU_TARGETS_I64) ? 2 : 1};
  a.q_rs = p.q_row_stride;
  a.q_hs = p.q_head_stride;
  a.rows = p.rows;
  a.Hq = p.Hq;
  a.group = p.Hq / p.cache.H;
  a.W = p.max_attn_len;
  a.c = p.contextual_seq_len;
  a.alpha = p.alpha;
  a.scale = p.scale;
  const int64_t size = p.dtype == B200_HSTU_F32 ? 4 : 2;
  a.q_vec = (((uintptr_t)p.q | (uintptr_t)(a.q_rs * size) | (uintptr_t)(a.q_hs * size)) & 15) == 0;
  const int nt = row_tiles(p), grid = grid_of(p, nt);
  a.whole_units = whole_units(p, nt);
  if (!p.workspace || p.workspace_bytes < paged_attn_workspace_bytes(p))
    return fail(B200_HSTU_EWORKSPACE, "paged_attn: workspace of %lld bytes needed", (long long)paged_attn_workspace_bytes(p));
  uint8_t *w = static_cast<uint8_t *>(p.workspace);
  a.status = reinterpret_cast<int *>(w);
  w += PA_HEADER;
  a.joins = reinterpret_cast<int4 *>(w);
  w += align256((int64_t)grid * 2 * sizeof(int4));
  a.part_ml = reinterpret_cast<float *>(w);
  w += align256((int64_t)grid * 2 * rows_of(nt) * 2 * sizeof(float));
  a.part_o = reinterpret_cast<float *>(w);
  ProfileScope prof(PROF_PAGED_ATTN, st);
  const bool softmax = p.softmax != 0;
  switch (p.dtype) {
    case B200_HSTU_F32: return launch_dim<float>(a, softmax, nt, grid, st);
    case B200_HSTU_BF16: return launch_dim<__nv_bfloat16>(a, softmax, nt, grid, st);
    default: return launch_dim<__half>(a, softmax, nt, grid, st);
  }
}

}  // namespace b200hstu
