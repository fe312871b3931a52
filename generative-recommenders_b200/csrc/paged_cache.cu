// Rows into and out of the paged 4-bit K / V cache.
//
// append: K is normed and rotated on the way (both optional), then K and V are rounded to codes of their group
// of 64 values:  scale = bfloat16(max |x| / 7),  code = 8 + clamp(round(x / scale), -7, 7).
// read: (code - 8) * scale.
#include "paged.cuh"
#include "rows8.cuh"

namespace b200hstu {

int check_rotation(const char *what, const float *cos, const float *sin, int64_t table_rows, int rotary, int interleaved,
                   int d, Rotation &out);

int check_paged_cache(const char *what, const b200_hstu_paged_cache &c, PagedCache &out) {
  if (c.B < 0 || c.H <= 0 || c.num_pages < 0 || c.table_width < 0)
    return fail(B200_HSTU_EINVAL, "%s: bad size of the cache", what);
  if (c.d != 64 && c.d != 128 && c.d != 256)
    return fail(B200_HSTU_EUNSUPPORTED, "%s: the cache's head dimension is 64, 128 or 256, not %d", what, c.d);
  int shift = 4;
  while (shift < 8 && (1 << shift) != c.page_size) ++shift;
  if ((1 << shift) != c.page_size)
    return fail(B200_HSTU_EUNSUPPORTED, "%s: a page has 16, 32, 64, 128 or 256 positions, not %d", what, c.page_size);
  if (((uintptr_t)c.pages & 15) != 0) return fail(B200_HSTU_EINVAL, "%s: pages must be 16-byte aligned", what);
  if ((c.num_pages > 0 && !c.pages) || (c.B > 0 && c.table_width > 0 && !c.page_table))
    return fail(B200_HSTU_EINVAL, "%s: null cache or page table", what);
  out.pages = c.pages;
  out.table = c.page_table;
  out.num_pages = c.num_pages;
  out.table_stride = c.table_stride;
  out.B = c.B;
  out.H = c.H;
  out.d = c.d;
  out.width = c.table_width;
  out.page_shift = shift;
  return 0;
}

namespace {

constexpr int PC_THREADS = 256;
constexpr int PC_MAX_ROWS = 32;   // of a block: 2^5
constexpr int PC_HEADS = 4;       // that a lane group takes in turn, at most

struct Append {
  PagedCache cache;
  const void *x[2];               // K, V
  int64_t rs[2], hs[2];
  IndexTensor cached, offsets;
  const void *w;
  bool w_f32;
  Rotation rot;
  int64_t rows;
  int row_shift;                  // log2 of the rows of a block
  int heads;                      // of a lane group
  float eps;
};

// max |x| of the 8 lanes that hold a group; infinity where one of its values is no finite number
__device__ __forceinline__ float group_top(const float (&f)[8], uint32_t mates) {
  float m = 0.f, none = 0.f;   // (x * 0 is a NaN for those, and sums keep it)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    m = fmaxf(m, fabsf(f[i]));
    none = fmaf(f[i], 0.f, none);
  }
  if (none != none) m = INFINITY;
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = fmaxf(m, __shfl_xor_sync(mates, m, o));
  return m;
}

// Whole numbers c of -7 to 7, nearest to the values, as eight codes c + 8 in the nibbles of a word.  A sum with
// 1.5 * 2^23 + 8 rounds to the nearest and has c + 8 in its low bits (a conversion takes eight times as long); the
// words' upper bits, the same for all, come off at the end.
__device__ __forceinline__ uint32_t eight_codes(const float (&f)[8], float inverse) {
  constexpr uint32_t REST = 0x4b400000u * 0x11111111u;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) codes = codes * 16u + __float_as_uint(__fadd_rn(__fmul_rn(f[i], inverse), 12582920.f));
  return codes - REST;
}

// A block takes 2^row_shift rows: one thread for each finds its place, then LANES = d / 8 lanes take up to PC_HEADS heads
// of K or V of a row with one set of angles, neighbouring groups neighbouring rows.  The arithmetic is written with
// explicit roundings (and the sum of squares neighbours first), so that a row has one set of codes whatever block it
// falls into.
// Bound by the instructions of rotating and rounding, which are scalar (issue slots 62 %, DRAM 21 % of the time), not by
// bytes: 100 histories of 37 - 2001 rows of 8 heads of 64 in
// fp16 take 45 - 50 us (2.5 TB/s), 32 single rows 13 us with the call.  Four heads a group share a row's place and angles
// (that history in 96 us with reading back, 140 with one head each); where rows are few, one head each: the single rows
// 13.7 us, 16.8 with four.
template <typename T, int LANES, int MODE, bool VEC>
__global__ void __launch_bounds__(PC_THREADS, 3) paged_append_kernel(Append a) {
  constexpr int D = 8 * LANES, GROUPS = PC_THREADS / LANES;
  __shared__ int64_t s_page[PC_MAX_ROWS], s_pos[PC_MAX_ROWS];
  const int R = 1 << a.row_shift, H = a.cache.H, chunks = (H + a.heads - 1) / a.heads;
  const int64_t row0 = (int64_t)blockIdx.x * R;
  if ((int)threadIdx.x < R) {
    const int64_t row = row0 + threadIdx.x;
    int64_t page = -1, pos = 0;
    if (row < a.rows) {
      const int b = sequence_of(a.offsets, a.cache.B, row);
      if (b < a.cache.B && a.offsets[b] <= row) {
        pos = (int64_t)a.cached[b] + (row - a.offsets[b]);
        page = a.cache.page_of(b, pos);
      }
    }
    s_page[threadIdx.x] = page;
    s_pos[threadIdx.x] = pos;
  }
  __syncthreads();
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, e0 = lane * 8;
  const uint32_t mates = (LANES == 32 ? 0xffffffffu : ((1u << LANES) - 1)) << ((threadIdx.x & 31) / LANES * LANES);
  Rotation rot = a.rot;
  rot.mode = MODE;
  const int partner_lane = (threadIdx.x & 31) - lane + (MODE == ROTATE_HALVES ? partner_of(e0, rot) >> 3 : lane);
  for (int item = group; item < 2 * chunks * R; item += GROUPS) {   // (the lanes of a group stay together)
    const int r = item & (R - 1), hk = item >> a.row_shift, kv = hk >= chunks, h0 = (kv ? hk - chunks : hk) * a.heads;
    const int64_t page = s_page[r], pos = s_pos[r];
    if (page < 0) continue;
    const int hn = min(a.heads, H - h0);
    const int64_t hs = kv ? a.hs[1] : a.hs[0];
    const T *x0 = static_cast<const T *>(kv ? a.x[1] : a.x[0]) + (row0 + r) * (kv ? a.rs[1] : a.rs[0]) + h0 * hs;
    Raw8<T> own[PC_HEADS];
#pragma unroll
    for (int h = 0; h < PC_HEADS; ++h)
      if (h < hn) own[h] = load8<T, VEC>(x0 + h * hs + e0);
    float c[8], s[8];
    if (MODE != ROTATE_NONE && kv == 0) angles8<VEC>(rot, pos, e0, c, s);
    uint8_t *at = a.cache.page(page, h0);
    const int place = (int)(pos & (a.cache.page_size() - 1));
#pragma unroll
    for (int h = 0; h < PC_HEADS; ++h) {
      if (h >= hn) break;
      float f[8];
      values8<T>(own[h], f);
      if (kv == 0) {
        float t[8];
        if (MODE == ROTATE_HALVES && VEC) {   // (whose partner lane is itself uses none of it)
          values8<T>(exchanged(mates, own[h], partner_lane), t);
        } else if (MODE == ROTATE_HALVES) {
#pragma unroll
          for (int i = 0; i < 8; ++i) t[i] = to_f32(x0[h * hs + partner_of(e0 + i, rot)]);
        }
        if (a.w != nullptr) {
          float q[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) q[i] = __fmul_rn(f[i], f[i]);
          float ss = __fadd_rn(__fadd_rn(__fadd_rn(q[0], q[1]), __fadd_rn(q[2], q[3])),
                               __fadd_rn(__fadd_rn(q[4], q[5]), __fadd_rn(q[6], q[7])));
#pragma unroll
          for (int o = 1; o < LANES; o <<= 1) ss = __fadd_rn(ss, __shfl_xor_sync(mates, ss, o));
          const float rstd = __frcp_rn(__fsqrt_rn(__fadd_rn(__fmul_rn(ss, 1.f / D), a.eps)));
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            f[i] = __fmul_rn(__fmul_rn(f[i], rstd), weight_at<T>(a.w, a.w_f32, e0 + i));
            if (MODE == ROTATE_HALVES)
              t[i] = __fmul_rn(__fmul_rn(t[i], rstd), weight_at<T>(a.w, a.w_f32, partner_of(e0 + i, rot)));
          }
        }
        if (MODE != ROTATE_NONE) {
          if (MODE == ROTATE_NEIGHBOURS) {
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = f[i ^ 1];
          }
#pragma unroll
          for (int i = 0; i < 8; ++i)
            f[i] = e0 + i < rot.rotary ? __fadd_rn(__fmul_rn(f[i], c[i]), __fmul_rn(t[i], s[i])) : __fmul_rn(f[i], c[i]);
        }
      }
      const float top = group_top(f, mates);
      const bool finite = top < INFINITY;
      __nv_bfloat16 scale = __float2bfloat16_rn(__fmul_rn(top, 1.f / 7.f));
      const float step = __bfloat162float(scale);
      const bool zero = step < 1.17549435e-38f;
      uint32_t codes = 0x88888888u;
      if (!finite) scale = __ushort_as_bfloat16(0x7fff);
      else if (zero) scale = __ushort_as_bfloat16(0);
      // (the scale is within 2^-8 of top / 7, so no value is more than 7.03 steps)
      else codes = eight_codes(f, __frcp_rn(step));
      uint8_t *to = at + (int64_t)h * a.cache.page_bytes();
      reinterpret_cast<uint32_t *>(to + a.cache.codes_at(kv) + place * (D / 2))[lane] = codes;
      if ((lane & 7) == 0)
        reinterpret_cast<__nv_bfloat16 *>(to + a.cache.scales_at(kv) + place * (2 * D / PAGED_GROUP))[lane >> 3] = scale;
    }
  }
}

struct Read {
  PagedCache cache;
  void *out[2];
  IndexTensor offsets;
  int64_t rows;
  int row_shift, heads;   // (as for Append)
};

// (the history above: 23 us)
template <typename T, int LANES>
__global__ void __launch_bounds__(PC_THREADS) paged_read_kernel(Read a) {
  constexpr int D = 8 * LANES, GROUPS = PC_THREADS / LANES;
  __shared__ int64_t s_page[PC_MAX_ROWS];
  __shared__ int s_place[PC_MAX_ROWS];
  const int R = 1 << a.row_shift, H = a.cache.H;
  const int64_t row0 = (int64_t)blockIdx.x * R;
  if ((int)threadIdx.x < R) {
    const int64_t row = row0 + threadIdx.x;
    int64_t page = -2;   // no row; -1: a row without a page
    int place = 0;
    if (row < a.rows) {
      const int b = sequence_of(a.offsets, a.cache.B, row);
      if (b < a.cache.B && a.offsets[b] <= row) {
        const int64_t pos = row - a.offsets[b];
        page = a.cache.page_of(b, pos);
        place = (int)(pos & (a.cache.page_size() - 1));
      }
    }
    s_page[threadIdx.x] = page;
    s_place[threadIdx.x] = place;
  }
  __syncthreads();
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, chunks = (H + a.heads - 1) / a.heads;
  const int rows = (int)min((int64_t)R, a.rows - row0);
  const int64_t step = a.cache.page_bytes();
  for (int item = group; item < 2 * chunks * R; item += GROUPS) {   // up to PC_HEADS heads of K or V of a row
    const int r = item & (R - 1), hk = item >> a.row_shift, kv = hk >= chunks, h0 = (kv ? hk - chunks : hk) * a.heads;
    if (r >= rows) continue;
    const int64_t page = s_page[r];
    const int hn = min(a.heads, H - h0);
    uint32_t codes[PC_HEADS];
    float scale[PC_HEADS];
    const uint8_t *at = a.cache.page(page >= 0 ? page : 0, h0);
    const uint8_t *cp = at + a.cache.codes_at(kv) + s_place[r] * (D / 2) + 4 * lane;
    const uint8_t *sp = at + a.cache.scales_at(kv) + s_place[r] * (2 * D / PAGED_GROUP) + 2 * (lane >> 3);
#pragma unroll
    for (int h = 0; h < PC_HEADS; ++h) {
      codes[h] = 0x88888888u;
      scale[h] = page == -2 ? 0.f : __int_as_float(0x7fffffff);
      if (h >= hn || page < 0) continue;
      codes[h] = __ldg(reinterpret_cast<const uint32_t *>(cp + h * step));
      scale[h] = __bfloat162float(__ldg(reinterpret_cast<const __nv_bfloat16 *>(sp + h * step)));
    }
    T *out = static_cast<T *>(kv ? a.out[1] : a.out[0]) + ((row0 + r) * H + h0) * D + lane * 8;
#pragma unroll
    for (int h = 0; h < PC_HEADS; ++h) {
      if (h >= hn) break;
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)   // (a code in the low bits of 2^23: a conversion takes eight times as long)
        f[i] = (__uint_as_float(((codes[h] >> (4 * i)) & 15u) | 0x4b000000u) - 8388616.f) * scale[h];
      store8<T>(out + h * D, f);
    }
  }
}

// Rows of a block: many where there are many (one search per row, neighbouring rows of a page together), few
// where the grid would not fill the card.
int row_shift_for(int64_t rows) {
  int s = 5;
  while (s > 0 && ((rows - 1) >> s) + 1 < 2 * 148) --s;
  return s;
}

template <typename T, int LANES>
void launch_append(const Append &a, bool vec, unsigned blocks, cudaStream_t st) {
#define B200_APPEND(MODE)                                                                       \
  if (vec) paged_append_kernel<T, LANES, MODE, true><<<blocks, PC_THREADS, 0, st>>>(a);          \
  else paged_append_kernel<T, LANES, MODE, false><<<blocks, PC_THREADS, 0, st>>>(a)
  if (a.rot.mode == ROTATE_NONE) { B200_APPEND(ROTATE_NONE); }
  else if (a.rot.mode == ROTATE_HALVES) { B200_APPEND(ROTATE_HALVES); }
  else { B200_APPEND(ROTATE_NEIGHBOURS); }
#undef B200_APPEND
}

template <typename T>
int append_type(const Append &a, bool vec, cudaStream_t st) {
  const unsigned blocks = (unsigned)(((a.rows - 1) >> a.row_shift) + 1);
  if (a.cache.d == 64) launch_append<T, 8>(a, vec, blocks, st);
  else if (a.cache.d == 128) launch_append<T, 16>(a, vec, blocks, st);
  else launch_append<T, 32>(a, vec, blocks, st);
  count_launch();
  B200_CHECK_LAUNCH("paged_append_kernel");
  return 0;
}

template <typename T>
int read_type(const Read &a, cudaStream_t st) {
  const unsigned blocks = (unsigned)(((a.rows - 1) >> a.row_shift) + 1);
  if (a.cache.d == 64) paged_read_kernel<T, 8><<<blocks, PC_THREADS, 0, st>>>(a);
  else if (a.cache.d == 128) paged_read_kernel<T, 16><<<blocks, PC_THREADS, 0, st>>>(a);
  else paged_read_kernel<T, 32><<<blocks, PC_THREADS, 0, st>>>(a);
  count_launch();
  B200_CHECK_LAUNCH("paged_read_kernel");
  return 0;
}

}  // namespace

int paged_append(const b200_hstu_paged_append_args &p, cudaStream_t st) {
  Append a = {};
  if (int rc = check_paged_cache("paged_append", p.cache, a.cache)) return rc;
  if (p.rows < 0 || p.rows >= (1ll << 31)) return fail(B200_HSTU_EINVAL, "paged_append: bad number of rows");
  if (p.cos || p.sin) {
    if (int rc = check_rotation("paged_append", p.cos, p.sin, p.table_rows, p.rotary, p.interleaved, p.cache.d, a.rot))
      return rc;
  }
  if (p.k_weight && p.k_weight_dtype != B200_HSTU_F32 && p.k_weight_dtype != p.dtype)
    return fail(B200_HSTU_EINVAL, "paged_append: the weight must be float32 or of the rows' type");
  if (p.dtype != B200_HSTU_F32 && p.dtype != B200_HSTU_BF16 && p.dtype != B200_HSTU_F16)
    return fail(B200_HSTU_EINVAL, "unknown dtype %d", p.dtype);
  if (p.rows == 0 || p.cache.B == 0) return 0;
  if (!p.k || !p.v || !p.cached_lengths || !p.new_offsets) return fail(B200_HSTU_EINVAL, "paged_append: null tensor");
  a.x[0] = p.k, a.x[1] = p.v;
  a.rs[0] = p.k_row_stride, a.rs[1] = p.v_row_stride;
  a.hs[0] = p.k_head_stride, a.hs[1] = p.v_head_stride;
  a.cached = {p.cached_lengths, (p.index_flags & B200_HSTU_LENGTHS_I64) ? 2 : 1};
  a.offsets = {p.new_offsets, (p.index_flags & B200_HSTU_OFFSETS_I64) ? 2 : 1};
  a.w = p.k_weight;
  a.w_f32 = p.k_weight_dtype == B200_HSTU_F32;
  a.rows = p.rows;
  a.row_shift = row_shift_for(p.rows);
  // (one head each where the rows would not fill the card: a step's latency goes with the heads in turn)
  a.heads = a.row_shift > 0 ? PC_HEADS : 1;
  a.eps = p.eps;
  const int64_t size = p.dtype == B200_HSTU_F32 ? 4 : 2;
  uintptr_t align = 0;
  for (int i = 0; i < 2; ++i) align |= (uintptr_t)a.x[i] | (uintptr_t)(a.rs[i] * size) | (uintptr_t)(a.hs[i] * size);
  if (a.rot.mode != ROTATE_NONE) align |= (uintptr_t)a.rot.cos | (uintptr_t)a.rot.sin | (uintptr_t)(a.rot.rotary % 16);
  ProfileScope prof(PROF_PAGED_APPEND, st);
  switch (p.dtype) {
    case B200_HSTU_F32: return append_type<float>(a, (align & 15) == 0, st);
    case B200_HSTU_BF16: return append_type<__nv_bfloat16>(a, (align & 15) == 0, st);
    default: return append_type<__half>(a, (align & 15) == 0, st);
  }
}

int paged_read(const b200_hstu_paged_read_args &p, cudaStream_t st) {
  Read a = {};
  if (int rc = check_paged_cache("paged_read", p.cache, a.cache)) return rc;
  if (p.rows < 0 || p.rows >= (1ll << 31)) return fail(B200_HSTU_EINVAL, "paged_read: bad number of rows");
  if (p.rows == 0) return 0;
  if (!p.k || !p.v || !p.seq_offsets) return fail(B200_HSTU_EINVAL, "paged_read: null tensor");
  if ((((uintptr_t)p.k | (uintptr_t)p.v) & 15) != 0) return fail(B200_HSTU_EINVAL, "paged_read: k and v must be 16-byte aligned");
  a.out[0] = p.k, a.out[1] = p.v;
  a.offsets = {p.seq_offsets, (p.index_flags & B200_HSTU_OFFSETS_I64) ? 2 : 1};
  a.rows = p.rows;
  a.row_shift = row_shift_for(p.rows);
  a.heads = a.row_shift > 0 ? PC_HEADS : 1;
  ProfileScope prof(PROF_PAGED_READ, st);
  switch (p.dtype) {
    case B200_HSTU_F32: return read_type<float>(a, st);
    case B200_HSTU_BF16: return read_type<__nv_bfloat16>(a, st);
    case B200_HSTU_F16: return read_type<__half>(a, st);
    default: return fail(B200_HSTU_EINVAL, "unknown dtype %d", p.dtype);
  }
}

}  // namespace b200hstu
