// Attention of many new rows over the paged 4-bit K / V cache on Blackwell tensor cores (tcgen05 + TMEM), head
// dimension 64 or 128: pieces of a prompt, hundreds of candidates.
//
// One CTA per SM, 14 warps, on blocks of 128 rows (new rows times the heads of a group) and tiles of 128 positions:
//   warp 13      walks the units and hands out tiles through a ring of eight slots: where each 16 positions' codes
//                lie, the scales as float16, their exponent, what the tile starts or ends
//   warps 8-11   codes to float16 in shared memory, 32 positions of K and of V each, in the 128-byte swizzle that
//                tcgen05.mma reads; codes are requested two tiles ahead
//   warp 12      the products: S = Q K^T into one of two TMEM regions, O += P V with P from TMEM; S of the next tile
//                is issued before P of the present one is there
//   warps 0-3, 4-7   even and odd tiles: a row each per thread; weights from the scores (16 bits, over the scores in
//                TMEM).  The two have results and references of their own, like two pieces of a split unit, and add
//                them up at its end; then q of the next unit is in shared memory already.
//
// Rounding: (code - 8) * scale has at most 11 significant bits, so in float16 it is exact for scales from 2^12 down to
// 2^-13 (odd pairs of codes are 16 times too large and meet a sixteenth of the scale).  K's scales are divided by a
// power of two for each tile that leaves the largest at 2^12, and goes into the scores' factor; V's by one that leaves
// it at 2^9 to 2^12 and changes where a tile's scales leave that range (the results, in fp32, are multiplied by the
// difference).  So scales down to 2^-25 and 2^-22 of a tile's largest are exact, whichever rows see that one and
// whichever group of 64 values it is in; smaller ones lose a bit for each power of two.  q is scaled by a power of two
// for each row.  The weights are float16 too, so they are held at a size of their own: for softmax the largest so far
// is at 2^7 to 2^15; for SiLU 2^15 is what no score can reach, |alpha| D max |q| times the tile's largest code and
// scale, which is 2^7 or so times the usual ones.  So no finite score overflows, and weights keep their 11 bits down to
// 2^-21 of the largest (2^-29 of SiLU's bound).  What is rounded is a weight, to 11 bits, and the result; tanh.approx,
// as in the attention over 16-bit keys, is off by 2^-11 of half the score (an exponential and a reciprocal instead:
// 25 % more time, 40 % for 256 rows a history, and results as far from 64 bits, by the weights' rounding).
//
// A score costs one operation of the special-function unit (16 a clock and SM), 128 x 128 of them 1024 clocks; the
// tile's two products take 512 clocks at head dimension 128.  Neither is the bound: special functions and products are
// busy a third of the time each, and so are the issue slots.  What is, is the row warps' waiting for scores: 32 of them
// are loaded from tensor memory, waited for and worked on, then the next 32, for softmax twice (the maximum first).
// Measured at head dimension 128, 4 heads: 256 rows for each of 32 histories of 8192 221 us for SiLU (611 TFLOP/s) and
// 241 us for softmax, 128 rows each 187 us; 128 users of 320 - 8192 with 256 candidates 422 - 464 us.
#include "paged_attn.cuh"

namespace b200hstu {

using namespace ptx;

namespace {

constexpr int TC_THREADS = 448, TC_WARPS = TC_THREADS / 32;
constexpr int TC_ROWS = 128, TC_BLOCK = 2 * TC_ROWS, TC_TILE = 128;   // rows of a product, of a unit; positions of a tile
constexpr int RING_SLOTS = 8;
constexpr int RING_READERS = 13;  // 8 + 4 + 1 warps
constexpr int SCALE_AT = 12;      // exponent of the largest scale that float16 has room for (code 0: 8 * 1.99 * 2^12 < 65504)
enum { TILE_FIRST = 1, TILE_PAIR = 2, TILE_BAD = 4 };

struct __align__(16) RingSlot {
  const uint8_t *codes[8];         // K codes of 16 positions; nullptr: none
  uint16_t scales[2][TC_TILE * 2]; // float16, K and V, [position][group]
  float k_factor;                  // 2^e that K's scales were divided by
  int k_ref;                       // SiLU: the e, or a larger one, that the weights' size goes by
  int v_exp;                       // e of V's
  int flags;
  uint32_t bad[2][4];              // positions whose V is no number in a group of 64 values
};

template <int D>
struct TcSmem {
  static constexpr int CHUNKS = D / 64, CHUNK = 128 * 128, TILE = CHUNKS * CHUNK;   // 64 values of 128 rows
  static constexpr int Q = 0, K = 2 * TILE, V = 4 * TILE, RING = 6 * TILE, BARS = RING + RING_SLOTS * (int)sizeof(RingSlot);
  static constexpr int TOTAL = BARS + 320;
  // (aligned by hand; and no second CTA on an SM, each takes all of TMEM)
  static constexpr int BYTES = TOTAL + 1024 > 118 * 1024 ? TOTAL + 1024 : 118 * 1024;
};

__device__ __forceinline__ uint32_t half2_mul(uint32_t a, uint32_t b) {
  __half2 r = __hmul2(*reinterpret_cast<__half2 *>(&a), *reinterpret_cast<__half2 *>(&b));
  return *reinterpret_cast<uint32_t *>(&r);
}
// eight codes times their scale (s1) - of pairs 1 and 3 a sixteenth of it (s16); values 0 4, 1 5, 2 6, 3 7
__device__ __forceinline__ uint4 eight_values(uint32_t x, uint32_t s1, uint32_t s16) {
  uint4 r;
  r.x = half2_mul(k_exact(k_pair(x, false), false), s1);
  r.y = half2_mul(k_exact(k_pair(x, true), true), s16);
  r.z = half2_mul(k_exact(k_pair(x >> 8, false), false), s1);
  r.w = half2_mul(k_exact(k_pair(x >> 8, true), true), s16);
  return r;
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((127 + min(max(e, -126), 127)) << 23); }
__device__ __forceinline__ float pow2_far(int e) { return pow2(e / 2) * pow2(e - e / 2); }   // beyond fp32's normal numbers

// A power of two that follows those of a unit's tiles, which it may be above by `above` and below by `below` at most;
// otherwise it is set to one above by `set`.  Results are held relative to it, so it does not fall below its largest so
// far by more than `fall`: 2^44 for V and 2^30 for K together leave results of 2^50 within fp32.
struct Follow {
  int at, most;
  __device__ __forceinline__ void next(bool first, bool none, int e, int above, int below, int set, int fall) {
    if (first) at = most = -126;
    if (none) return;   // (all zeros: nothing to go by)
    if (at - e > above || e - at > below) at = max(max(e + set, most - fall), -126);
    most = max(most, at);
  }
};

// column c of a row's eight holds value ..
__device__ __forceinline__ constexpr int value_of(int c) { return (c >> 1) + 4 * (c & 1); }

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

// a barrier of the eight row warps that says whether any of them asks
__device__ __forceinline__ bool rows_any(bool asks) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.aligned.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)asks)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ uint32_t range_bits(int lo, int hi) {   // bits [lo, hi) of 32
  lo = max(lo, 0);
  hi = min(hi, 32);
  return hi <= lo ? 0u : (0xffffffffu >> (32 - hi + lo)) << lo;
}

template <typename T, int D, bool SOFTMAX>
__global__ void __launch_bounds__(TC_THREADS, 1) paged_attn_tc_kernel(PagedAttn a) {
  using SM = TcSmem<D>;
  constexpr int G64 = D / 64, ROW = D / 2, SROW = 2 * G64;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t *gen = smem_raw + (base - smem_u32(smem_raw));
  RingSlot *ring = reinterpret_cast<RingSlot *>(gen + SM::RING);
  const uint32_t bars = base + SM::BARS;
  const uint32_t ring_full = bars, ring_empty = ring_full + 8 * RING_SLOTS;
  const uint32_t k_full = ring_empty + 8 * RING_SLOTS, k_empty = k_full + 16, v_full = k_empty + 16, v_empty = v_full + 16;
  const uint32_t s_full = v_empty + 16, p_full = s_full + 16, pv_done = p_full + 16, q_full = pv_done + 16, o_empty = q_full + 8;
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(gen + SM::BARS + 304);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(gen + SM::BARS + 312);
  __shared__ RunSmem<TC_WARPS> s_run;
  __shared__ float s_top[2][TC_ROWS], s_sum[2][TC_ROWS];
  __shared__ int s_ref[2][TC_ROWS];
  __shared__ uint8_t s_lost[2][TC_ROWS];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const WaitCtx wc{abort_flag, a.status};

  allow_dependents();
  if (threadIdx.x == 0) {
    *abort_flag = 0;
    if (blockIdx.x == 0) *a.status = 0;   // (a wait gives up seconds after this)
    for (int x = 0; x < RING_SLOTS; ++x) {
      mbar_init(ring_full + 8 * x, 1);
      mbar_init(ring_empty + 8 * x, RING_READERS);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(k_full + 8 * x, 4);
      mbar_init(k_empty + 8 * x, 1);
      mbar_init(v_full + 8 * x, 4);
      mbar_init(v_empty + 8 * x, 1);
      mbar_init(s_full + 8 * x, 1);
      mbar_init(p_full + 8 * x, 4);
      mbar_init(pv_done + 8 * x, 1);
    }
    mbar_init(q_full, 8);
    mbar_init(o_empty, 8);
    fence_mbar_init();
  }
  clear_rows_of_nobody<T, D, TC_THREADS>(a);
  int64_t total;
  Walk<TC_BLOCK, TC_TILE> walk;
  const int G = find_run(a, s_run, total, walk);
  if (G == 0) return;
  if (warp == 12) {
    tmem_alloc(smem_u32(const_cast<uint32_t *>(tmem_slot)), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_o = tmem + 256;   // S and P: columns [0, 128), [128, 256); O: [256, 384), [384, 512)
  uint32_t n_tiles = (uint32_t)walk.left;
  if (a.whole_units) {
    Walk<TC_BLOCK, TC_TILE> w = walk;
    n_tiles = 0;
    do n_tiles += w.here;
    while (w.next(a));
  }
  bool ok = true;

  if (warp == 13) {
    // ---------------------------------------------------------------- tiles
    // three tiles at a time: the pages of one are looked up while the scales of the one before are on their way and
    // those before that are written
    struct Info {
      int flags;
      bool inside;             // this lane's block of 16 positions is one that the unit reads
      const uint8_t *page;     // of this lane's block (lane / 4), or nullptr
      int place;
      int pos, begin, end;     // of the tile; positions that some row sees: the scales of others count for nothing
    };
    const int blk = lane >> 2, part = lane & 3;
    bool more = true;
    auto look_up = [&](Info &f) {
      f.flags = -1;
      if (!more) return;
      const int pos = (walk.range.first_tile<TC_TILE>() + walk.tile) * TC_TILE + blk * PA_BLOCK;
      f.flags = 0;
      f.inside = pos >= walk.range.lo && pos < walk.range.hi;
      const int64_t page = f.inside ? a.cache.page_of(walk.b, pos) : -1;
      f.page = page >= 0 ? a.cache.page(page, walk.h) : nullptr;
      f.place = pos & (a.cache.page_size() - 1);
      f.pos = pos - blk * PA_BLOCK;
      f.begin = walk.range.begin;
      f.end = walk.range.end;
    };
    int done = 0;   // tiles of the unit handed out so far
    auto step = [&](Info &f) {   // flags of the tile just looked up, and on to the next
      if (!more) return;
      f.flags = (done == 0 ? TILE_FIRST : 0) | (walk.seq.rows - walk.rb * TC_BLOCK > TC_ROWS ? TILE_PAIR : 0);
      if (++done == walk.here) {
        done = 0;
        more = walk.next(a);
      } else {
        ++walk.tile;
      }
    };
    Info f[3];
    uint4 sc[3][2];
    auto request = [&](const Info &x, uint4 (&s)[2]) {
      s[0] = s[1] = make_uint4(0, 0, 0, 0);
      if (x.flags < 0 || x.page == nullptr) {
        // no such page: K is no number there; outside the unit: zeros
        if (x.flags >= 0 && x.inside) s[0] = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);
        return;
      }
      if (part < 2 * G64) {
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
          s[kv] = __ldg(reinterpret_cast<const uint4 *>(x.page + a.cache.scales_at(kv) + x.place * SROW + part * 16));
      }
    };
    look_up(f[0]);
    step(f[0]);
    look_up(f[1]);
    step(f[1]);
    request(f[0], sc[0]);
    Follow k_ref{0, 0}, v_ref{0, 0};
    auto hand_out = [&](uint32_t i, const Info &now, const uint4 (&scales)[2]) {
      RingSlot &slot = ring[i % RING_SLOTS];
      ok = mbar_wait(wc, ring_empty + 8 * (i % RING_SLOTS), ((i / RING_SLOTS) & 1) ^ 1, 961);
      if (!ok) return;
      if (part == 0)
        slot.codes[blk] = now.page == nullptr ? nullptr : now.page + now.place * ROW;
      uint32_t bad = 0;
      int exps[2];
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        uint16_t s[8];
        *reinterpret_cast<uint4 *>(s) = scales[kv];
        uint32_t most = 0;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int pos = now.pos + blk * PA_BLOCK + (part * 8 + x) / G64;
          if (pos < now.begin || pos >= now.end) s[x] = 0;
          const uint32_t size = s[x] & 0x7fffu;   // (append makes no negative scales, but they are numbers)
          if (size < 0x7f80u) most = max(most, size);
          else if (kv == 1) bad |= 1u << x, s[x] = 0;
        }
        most = __reduce_max_sync(0xffffffffu, most);
        int e = max((int)(most >> 7) - 127 - SCALE_AT, -126);
        if (kv == 0) {
          k_ref.next(now.flags & TILE_FIRST, most == 0, e, 8, 0, 1, 30);
        } else {
          v_ref.next(now.flags & TILE_FIRST, most == 0, e, 3, 0, 1, 44);
          e = v_ref.at;
        }
        exps[kv] = e;
        const float down = __int_as_float((127 - e) << 23);
        uint32_t h[4];
#pragma unroll
        for (int x = 0; x < 4; ++x)
          h[x] = pack_f16(__uint_as_float((uint32_t)s[2 * x] << 16) * down, __uint_as_float((uint32_t)s[2 * x + 1] << 16) * down);
        if (part < 2 * G64)
          *reinterpret_cast<uint4 *>(&slot.scales[kv][blk * PA_BLOCK * G64 + part * 8]) = make_uint4(h[0], h[1], h[2], h[3]);
      }
      const bool any_bad = __any_sync(0xffffffffu, bad != 0);
      if (lane < 8) slot.bad[lane >> 2][lane & 3] = 0;
      __syncwarp();
      if (any_bad && bad != 0) {
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int key = blk * PA_BLOCK + (part * 8 + x) / G64;
          if ((bad >> x) & 1) atomicOr(&slot.bad[x % G64][key >> 5], 1u << (key & 31));
        }
      }
      if (lane == 0) {
        slot.k_factor = pow2(exps[0]);
        slot.k_ref = k_ref.at;
        slot.v_exp = exps[1];
        slot.flags = now.flags | (any_bad ? TILE_BAD : 0);
      }
      __syncwarp();
      if (lane == 0) {
        asm volatile("fence.acq_rel.cta;" ::: "memory");
        mbar_arrive(ring_full + 8 * (i % RING_SLOTS));
      }
    };
    // (three in turn, unrolled: handing a load's result from one register to another would wait for it)
    for (uint32_t i0 = 0; i0 < n_tiles && ok; i0 += 3) {
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        if (i0 + k >= n_tiles || !ok) break;
        look_up(f[(k + 2) % 3]);
        step(f[(k + 2) % 3]);
        request(f[(k + 1) % 3], sc[(k + 1) % 3]);
        hand_out(i0 + k, f[k], sc[k]);
      }
    }
  } else if (warp == 12) {
    // ---------------------------------------------------------------- products
    const uint32_t idesc_s = make_idesc(0, 0, 0, 0, TC_ROWS, TC_TILE), idesc_o = make_idesc(0, 0, 0, 1, TC_ROWS, D);
    uint32_t units = 0, into = 0;          // units begun; tiles of the present one whose sums are issued
    uint32_t given[2] = {0, 0};            // weights that a side has handed over
    auto flags_of = [&](uint32_t i) {
      const uint32_t s = i % RING_SLOTS;
      ok = ok && mbar_wait(wc, ring_full + 8 * s, (i / RING_SLOTS) & 1, 962);
      const int f = *reinterpret_cast<volatile int *>(&ring[s].flags);
      __syncwarp();
      if (lane == 0) mbar_arrive(ring_empty + 8 * s);
      return f;
    };
    // scores of rows `side` (a pair) or of the only rows, into the side's region; `last`: nobody else reads K
    auto score = [&](uint32_t i, int side, int rows, bool last) {
      if (!ok) return;
      const uint64_t q = make_smem_desc(base + SM::Q + rows * SM::TILE, 16, 1024);
      const uint64_t k = make_smem_desc(base + SM::K + (i & 1) * SM::TILE, 16, 1024);
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = (ks / 4) * SM::CHUNK + (ks % 4) * 32;
          mma_ss(tmem + side * 128, desc_advance(q, off), desc_advance(k, off), idesc_s, ks > 0);
        }
        tc_commit(s_full + 8 * side);
        if (last) tc_commit(k_empty + 8 * (i & 1));
      }
      __syncwarp();
    };
    auto wait_k = [&](uint32_t i, int flags) {
      if (flags & TILE_FIRST) ok = ok && mbar_wait(wc, q_full, units++ & 1, 963);
      ok = ok && mbar_wait(wc, k_full + 8 * (i & 1), (i >> 1) & 1, 964);
      tc_fence_after();
    };
    auto scores = [&](uint32_t i, int flags) {
      wait_k(i, flags);
      if (flags & TILE_PAIR) {
        score(i, 0, 0, false);
        score(i, 1, 1, true);
      } else {
        score(i, i & 1, 0, true);
      }
    };
    auto sum = [&](uint32_t i, int side, bool fresh, bool last) {
      ok = ok && mbar_wait(wc, p_full + 8 * side, given[side]++ & 1, 967);
      if (!ok) return;
      tc_fence_after();
      const uint64_t v = make_smem_desc(base + SM::V + (i & 1) * SM::TILE, SM::CHUNK, 1024);
      if (elect_one()) {
#pragma unroll
        for (int ks = 0; ks < TC_TILE / 16; ++ks)
          mma_ts(tmem_o + side * 128, tmem + side * 128 + ks * 8, desc_advance(v, ks * 2048), idesc_o, fresh && ks == 0 ? 0u : 1u);
        if (last) tc_commit(v_empty + 8 * (i & 1));
        tc_commit(pv_done + 8 * side);
      }
      __syncwarp();
    };
    int now = flags_of(0);
    scores(0, now);
    for (uint32_t i = 0; i < n_tiles && ok; ++i) {
      const int then = i + 1 < n_tiles ? flags_of(i + 1) : TILE_FIRST;
      const bool on = !(then & TILE_FIRST);   // the unit goes on
      if (!(now & TILE_PAIR) && on) scores(i + 1, then);
      ok = ok && mbar_wait(wc, v_full + 8 * (i & 1), (i >> 1) & 1, 965);
      if (now & TILE_FIRST) {   // (the results of the unit before have been read)
        ok = ok && mbar_wait(wc, o_empty, units & 1, 966);
        into = 0;
      }
      if (now & TILE_PAIR) {    // one side's next scores while the other makes its weights
        sum(i, 0, into == 0, false);
        if (on) {
          wait_k(i + 1, then);
          score(i + 1, 0, 0, false);
        }
        sum(i, 1, into == 0, true);
        if (on) score(i + 1, 1, 1, true);
      } else {
        sum(i, i & 1, into < 2, true);
      }
      ++into;
      if (!on && i + 1 < n_tiles) scores(i + 1, then);
      now = then;
    }
  } else if (warp >= 8) {
    // ---------------------------------------------------------------- codes to numbers
    const int w = warp - 8, in8 = lane & 7, piece = lane >> 3;     // 32 positions; 8 of them, and 32 of a row's values
    const bool on = piece < 2 * G64;
    // Codes of two tiles: a tile's are asked for when those of the one two before it have been converted.
    uint4 code[2][2][4];   // [tile][K, V][positions in8, in8 + 8 ..]
    auto request = [&](uint32_t i, int kv, uint4 (&c)[4]) {
      if (i >= n_tiles) return;
      if (kv == 0) ok = ok && mbar_wait(wc, ring_full + 8 * (i % RING_SLOTS), (i / RING_SLOTS) & 1, 968);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint8_t *at = ok ? *reinterpret_cast<const uint8_t *volatile *>(&ring[i % RING_SLOTS].codes[2 * w + half]) : nullptr;
#pragma unroll
        for (int y = 0; y < 2; ++y)
          c[2 * half + y] = at != nullptr && on
                                ? __ldg(reinterpret_cast<const uint4 *>(at + a.cache.codes_at(kv) + (in8 + 8 * y) * ROW) + piece)
                                : make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
      }
    };
    // where this lane's 16-byte units of a position's 64 values lie; every eight positions 1024 bytes on
    const int chunk = piece >> 1, at0 = chunk * SM::CHUNK + (w * 32 + in8) * 128;
    int unit_at[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) unit_at[j] = at0 + ((((piece & 1) * 4 + j) ^ in8) << 4);
    auto convert = [&](uint32_t i, int kv, const uint4 (&c)[4]) {
      const uint16_t *scales = ring[i % RING_SLOTS].scales[kv] + (w * 32 + in8) * G64 + chunk;
      ok = ok && mbar_wait(wc, (kv ? v_empty : k_empty) + 8 * (i & 1), ((i >> 1) & 1) ^ 1, 969);
      if (!ok) return;
      uint8_t *tile = gen + (kv ? SM::V : SM::K) + (i & 1) * SM::TILE;
      if (on) {
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const uint32_t one = scales[8 * y * G64];
          const uint32_t s1 = one | one << 16;
          const uint32_t s16 = half2_mul(s1, 0x2c002c00u);   // 1 / 16
          const uint32_t *x = reinterpret_cast<const uint32_t *>(&c[y]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<uint4 *>(tile + unit_at[j] + 1024 * y) = eight_values(x[j], s1, s16);
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive((kv ? v_full : k_full) + 8 * (i & 1));
        if (kv) mbar_arrive(ring_empty + 8 * (i % RING_SLOTS));
      }
    };
#pragma unroll
    for (int x = 0; x < 4; ++x) request(x >> 1, x & 1, code[x >> 1][x & 1]);
    for (uint32_t i0 = 0; i0 < n_tiles && ok; i0 += 2) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t i = i0 + (x >> 1);
        if (i >= n_tiles || !ok) break;
        convert(i, x & 1, code[x >> 1][x & 1]);
        request(i + 2, x & 1, code[x >> 1][x & 1]);
      }
    }
  } else {
    // ---------------------------------------------------------------- rows
    const int side = warp >> 2, r = (warp & 3) * 32 + lane;        // even or odd tiles; row of the block, TMEM lane
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;             // (lane offset of the warp's quarter, bits 16 and up)
    const uint32_t ts = tmem + lanes + side * 128, to = tmem_o + lanes + side * 128;
    // q of a row as float16, scaled by a power of two to at most 1: of a pair each side has its own rows, otherwise each
    // writes half of a row's values.  Returns the factor of the row's scores; `bound`: they are below 2^bound times K's
    // factor of the tile.
    int bound = 0;
    auto load_q = [&]() {
      const SeqShape &seq = walk.seq;
      const bool pair = seq.rows - walk.rb * TC_BLOCK > TC_ROWS;
      const int at = walk.rb * TC_BLOCK + (pair ? side * TC_ROWS : 0) + r;
      const bool on = at < seq.rows;
      const int row_i = on ? at / a.group : 0, hq = walk.h * a.group + (on ? at - row_i * a.group : 0);
      const T *q = static_cast<const T *>(a.q) + (int64_t)(seq.q_start + row_i) * a.q_rs + (int64_t)hq * a.q_hs;
      auto eight = [&](int u, float (&x)[8]) {
        if (a.q_vec) {
          const uint4 raw = __ldg(reinterpret_cast<const uint4 *>(q + 8 * u));
#pragma unroll
          for (int y = 0; y < 8; ++y) x[y] = to_f32(reinterpret_cast<const T *>(&raw)[y]);
        } else {
#pragma unroll
          for (int y = 0; y < 8; ++y) x[y] = to_f32(q[8 * u + y]);
        }
      };
      float most = 0.f;
      if (on) {
#pragma unroll 4
        for (int u = 0; u < D / 8; ++u) {
          float x[8];
          eight(u, x);
#pragma unroll
          for (int y = 0; y < 8; ++y) most = fmaxf(most, fabsf(x[y]));
        }
      }
      if (!SOFTMAX) bound = (__float_as_int(most * fabsf(a.alpha) * (1.01f * D * 8.f * (2 << SCALE_AT))) >> 23) - 126;   // (1.01: q's rounding)
      const int e = min(max((__float_as_int(most) >> 23) - 126, -125), 125);
      const float down = __int_as_float((127 - e) << 23) * (a.alpha < 0.f ? -1.f : 1.f);
      uint8_t *tile = gen + SM::Q + (pair ? side * SM::TILE : 0) + r * 128;
      const int u0 = pair ? 0 : side * (D / 16), u1 = pair ? D / 8 : u0 + D / 16;
#pragma unroll 4
      for (int u = u0; u < u1; ++u) {
        uint4 h = make_uint4(0, 0, 0, 0);
        if (on) {
          float x[8];
          eight(u, x);
          h = make_uint4(pack_f16(x[0] * down, x[4] * down), pack_f16(x[1] * down, x[5] * down),
                         pack_f16(x[2] * down, x[6] * down), pack_f16(x[3] * down, x[7] * down));
        }
        *reinterpret_cast<uint4 *>(tile + (u >> 3) * SM::CHUNK + (((u & 7) ^ (r & 7)) << 4)) = h;
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
      return __int_as_float((127 + e) << 23) * fabsf(a.alpha) * (SOFTMAX ? 1.4426950408889634f : 0.5f);
    };
    float mul = load_q();
    uint32_t begin = 0, count = 0;   // first tile of the unit; tiles whose weights this side has made
    while (true) {   // (left at rows_any() alone, or when there is no more)
      const int here = walk.here;
      const bool pair = walk.seq.rows - walk.rb * TC_BLOCK > TC_ROWS;
      const RowSees sees = [&]() {
        const int at = walk.rb * TC_BLOCK + (pair ? side * TC_ROWS : 0) + r;
        return at < walk.seq.rows ? row_sees(walk.seq.len - walk.seq.new_rows + at / a.group, walk.seq.len, walk.seq.targets, a.c, a.W)
                                  : RowSees{0, 0, -1};
      }();
      float top = SOFTMAX ? -3.0e38f : 0.f, sum = 0.f;
      int ref = 0;          // the result so far is in units of 2^ref
      // groups of 64 values in which the row sees a V that is no number
      uint32_t lost = sees.past(a.cache.positions()) ? 3 : 0;
      const uint32_t end = begin + here, before = count;
      const int first_pos = (walk.range.first_tile<TC_TILE>() + walk.tile) * TC_TILE;
      for (uint32_t i = begin; i < end && ok; ++i) {
        const RingSlot &slot = ring[i % RING_SLOTS];
        ok = mbar_wait(wc, ring_full + 8 * (i % RING_SLOTS), (i / RING_SLOTS) & 1, 970);
        if (!pair && (int)(i & 1) != side) {   // the other side's
          __syncwarp();
          if (lane == 0) mbar_arrive(ring_empty + 8 * (i % RING_SLOTS));
          continue;
        }
        ok = ok && mbar_wait(wc, s_full + 8 * side, count & 1, 971);
        if (!ok) break;
        tc_fence_after();
        float factor = mul * slot.k_factor;
        if (SOFTMAX) factor = fmaxf(factor, 1.2e-38f);   // (above 0: an unseen score stays -inf)
        const int v_exp = slot.v_exp;
        const int pos0 = first_pos + (int)(i - begin) * TC_TILE;
        const bool masked = pos0 < walk.range.all_lo || pos0 + TC_TILE > walk.range.all_hi;
        auto seen_bits = [&](int c) {   // of 32 columns
          const int at = pos0 + 32 * c;
          return range_bits(sees.lo - at, sees.hi - at) | range_bits(sees.self - at, sees.self - at + 1);
        };
        if (slot.flags & TILE_BAD) {   // (those V are zeros in the product)
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int g = 0; g < G64; ++g) lost |= (seen_bits(c) & slot.bad[g][c]) != 0 ? 1u << g : 0u;
          }
        }
        // scores of 32 columns; unseen ones to `none`
        uint32_t s[32];
        auto load = [&](int c, float none) {
          tmem_ld32(ts + 32 * c, s);
          tc_wait_ld();
          if (masked) {
            const uint32_t bits = seen_bits(c);
#pragma unroll
            for (int x = 0; x < 32; ++x)
              if (!((bits >> x) & 1)) s[x] = __float_as_uint(none);
          }
        };
        // this side's sum before: its end is waited for before the next can begin (a parity says which of two phases
        // is over, so nobody may be two behind)
        auto wait_sum = [&]() {
          if (count > 0) ok = ok && mbar_wait(wc, pv_done + 8 * side, (count - 1) & 1, 972);
        };
        auto rescale = [&](float by) {   // multiplies this row of O
          wait_sum();
          if (!ok || count == before) return;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(to + 16 * c, o);
            tc_wait_ld();
#pragma unroll
            for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * by);
            tmem_st16(to + 16 * c, o);
          }
          tc_wait_st();
        };
        float p_factor = 1.f, shift = 0.f;
        if (SOFTMAX) {
          float m = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            load(c, -INFINITY);
#pragma unroll
            for (int x = 0; x < 32; x += 2) m = fmaxf(m, fmaxf(__uint_as_float(s[x]), __uint_as_float(s[x + 1])));
          }
          m *= factor;
          const bool higher = __any_sync(0xffffffffu, m > top + 8.f);
          if (higher || v_exp != ref) {
            m = higher ? fmaxf(m, top) : top;
            const float by = ex2(top - m);
            rescale(by * pow2(ref - v_exp));
            sum *= by;
            top = m;
            ref = v_exp;
          }
          shift = 7.f - top;
        } else {
          const int t = min(max(15 - bound - slot.k_ref, -126), 126), now = v_exp - t;
          if (__any_sync(0xffffffffu, now != ref)) {
            rescale(pow2(ref - now));
            ref = now;
          }
          p_factor = pow2(t);
        }
        float part0 = 0.f, part1 = 0.f;
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          load(c, SOFTMAX ? -INFINITY : 0.f);
          uint32_t p[16];
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            float s0, s1;
            if (SOFTMAX) {
              fma2(__uint_as_float(s[2 * x]), __uint_as_float(s[2 * x + 1]), factor, factor, shift, shift, s0, s1);
              s0 = ex2(s0);
              s1 = ex2(s1);
              fma2(s0, s1, 1.f, 1.f, part0, part1, part0, part1);
            } else {
              float h0, h1, g0, g1;
              mul2(__uint_as_float(s[2 * x]), __uint_as_float(s[2 * x + 1]), factor, h0, h1);   // half of x
              mul2(h0, h1, p_factor, g0, g1);
              fma2(g0, g1, tanh_approx(h0), tanh_approx(h1), g0, g1, s0, s1);                   // x / (1 + e^-x)
            }
            p[x] = pack_f16(s0, s1);
          }
          tmem_st16(ts + 16 * c, p);
        }
        if (SOFTMAX) sum += part0 + part1;
        tc_wait_st();
        tc_fence_before();
        wait_sum();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(p_full + 8 * side);
          mbar_arrive(ring_empty + 8 * (i % RING_SLOTS));
        }
        ++count;
      }
      // ---------------------------------------------------------- q of the next unit, then the result of this one
      const Walk<TC_BLOCK, TC_TILE> done = walk;
      if (count != before && ok) ok = mbar_wait(wc, pv_done + 8 * side, (count - 1) & 1, 974);
      s_top[side][r] = top;
      s_sum[side][r] = sum;
      s_ref[side][r] = ref;
      s_lost[side][r] = (uint8_t)lost;
      tc_fence_before();
      if (rows_any(!ok)) break;        // (all eight warps or none: whoever gave up still comes here)
      tc_fence_after();
      const bool more = walk.next(a);
      if (more) mul = load_q();        // (the scores of this unit are all there, its q has had its day)
      {
        const bool both = !pair && here > 1;   // (the side of a unit's only tile has it all)
        const int lead = pair ? side : begin & 1;
        float f0 = pow2_far(s_ref[lead][r]), f1 = pow2_far(s_ref[lead ^ 1][r]), m = 0.f, l = 0.f;
        if (SOFTMAX) {   // (weights of up to 2^15 are numbers of up to 1 from here on)
          const float t0 = s_top[lead][r], t1 = s_top[lead ^ 1][r];
          m = both ? fmaxf(t0, t1) : t0;
          const float w0 = ex2(t0 - m) * 0x1p-15f, w1 = ex2(t1 - m) * 0x1p-15f;
          l = s_sum[lead][r] * w0 + (both ? s_sum[lead ^ 1][r] * w1 : 0.f);
          f0 *= w0;
          f1 *= w1;
        }
        const bool whole = done.whole();
        const int at = done.rb * TC_BLOCK + (pair ? side * TC_ROWS : 0) + r;
        const bool on = at < done.seq.rows;
        const int row_i = on ? at / a.group : 0, hq = done.h * a.group + (on ? at - row_i * a.group : 0);
        const int64_t slot_row = ((int64_t)blockIdx.x * 2 + done.slot()) * TC_BLOCK + at - done.rb * TC_BLOCK;
        const float last = !whole ? 1.f : !SOFTMAX ? a.scale : l == 0.f ? 0.f : 1.f / l;
        f0 *= last;
        f1 *= last;
        lost = s_lost[lead][r] | (both ? s_lost[lead ^ 1][r] : 0);
        T *out = static_cast<T *>(a.out) + ((int64_t)(done.seq.q_start + row_i) * a.Hq + hq) * D;
#pragma unroll 1
        for (int c = pair ? 0 : side * (D / 32); c < (pair ? D / 16 : (side + 1) * (D / 32)); ++c) {   // 16 columns at a time
          uint32_t o[16], o1[16];
          tmem_ld16(tmem_o + lanes + lead * 128 + 16 * c, o);
          if (both) tmem_ld16(tmem_o + lanes + (lead ^ 1) * 128 + 16 * c, o1);
          tc_wait_ld();
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            float x[8];
#pragma unroll
            for (int y = 0; y < 8; ++y) {
              x[value_of(y)] = __uint_as_float(o[8 * u + y]) * ((lost >> (c / 4)) & 1 ? __int_as_float(0x7fffffff) : f0);
              if (both) x[value_of(y)] += __uint_as_float(o1[8 * u + y]) * f1;
            }
            if (on && whole) {
              uint4 raw;
#pragma unroll
              for (int y = 0; y < 8; ++y) reinterpret_cast<T *>(&raw)[y] = from_f32<T>(x[y]);
              *reinterpret_cast<uint4 *>(out + 16 * c + 8 * u) = raw;
            } else if (on) {
              float4 *dst = reinterpret_cast<float4 *>(a.part_o + slot_row * D + 16 * c + 8 * u);
              dst[0] = make_float4(x[0], x[1], x[2], x[3]);
              dst[1] = make_float4(x[4], x[5], x[6], x[7]);
            }
          }
        }
        if (on && !whole && (pair || side == 0)) {
          a.part_ml[2 * slot_row] = m;
          a.part_ml[2 * slot_row + 1] = l;
        }
      }
      tc_fence_before();
      asm volatile("bar.sync 1, 256;" ::: "memory");   // (s_top, s_sum, s_ref and s_lost are free)
      if (lane == 0) mbar_arrive(o_empty);
      if (threadIdx.x == 0) leave_join(a, done, total, G);
      begin = end;
      if (!more) break;
    }
  }

  // ------------------------------------------------------------------ exit (all data came by plain loads)
  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <typename T, int D, bool SOFTMAX>
int launch_tc(const PagedAttn &a, int grid, cudaStream_t st) {
  auto kernel = paged_attn_tc_kernel<T, D, SOFTMAX>;
  if (int rc = check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TcSmem<D>::BYTES),
                          "cudaFuncSetAttribute"))   // (of the current device)
    return rc;
  kernel<<<grid, TC_THREADS, TcSmem<D>::BYTES, st>>>(a);
  count_launch();
  B200_CHECK_LAUNCH("paged_attn_tc_kernel");
  return 0;
}
template <typename T>
int launch_tc_type(const PagedAttn &a, bool softmax, int grid, cudaStream_t st) {
  if (a.cache.d == 64) return softmax ? launch_tc<T, 64, true>(a, grid, st) : launch_tc<T, 64, false>(a, grid, st);
  return softmax ? launch_tc<T, 128, true>(a, grid, st) : launch_tc<T, 128, false>(a, grid, st);
}

}  // namespace

int paged_attn_tc(const PagedAttn &a, bool bf16, bool softmax, int grid, cudaStream_t st) {
  return bf16 ? launch_tc_type<__nv_bfloat16>(a, softmax, grid, st) : launch_tc_type<__half>(a, softmax, grid, st);
}

}  // namespace b200hstu
