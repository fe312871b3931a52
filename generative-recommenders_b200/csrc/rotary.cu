// RMS norm of every head of q and k and the rotation of its leading values by the row's position, in one pass:
//
//   y = R(pos) (x rstd w),   rstd = 1 / sqrt(mean(x^2) + eps)
//   g = R(-pos) dy,   dw = sum g x rstd,   dx = rstd (g w - x rstd mean(g w x rstd))
//
// The backward takes rstd from x again, so the forward keeps nothing beside its inputs.
#include "rows8.cuh"
#include "sm100_ptx.cuh"   // packed fp32 arithmetic

namespace b200hstu {

namespace {

constexpr int NR_THREADS = 256;
constexpr int NR_HEADS = 4;     // heads of a row that a lane group takes in turn with one set of angles
constexpr int nr_ctas(bool bwd) { return bwd ? 2 : 4; }       // of an SM
constexpr int NR_MAX_BLOCKS = 148 * 8;

struct NormRotary {
  const void *x[2], *dy[2], *w[2];
  void *y[2], *dx[2];
  float *partial;               // bwd: [blocks][d]
  int blocks[2];                // CTAs that work on q, and those after them on k: by the number of heads
  int64_t x_rs[2], x_hs[2], dy_rs[2], dy_hs[2];
  int H[2];
  bool w_f32[2];
  const int32_t *positions;
  int pos_step;                 // 32-bit words of a position
  int64_t rows;
  int d;
  float eps;
  Rotation rot;
};

__device__ __forceinline__ int64_t position_of(const NormRotary &a, int64_t row) {
  if (a.rot.mode == ROTATE_NONE) return 0;
  return a.pos_step == 2 ? reinterpret_cast<const int64_t *>(a.positions)[row] : (int64_t)a.positions[row];
}

template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// a * b + c on eight values, two at a time
__device__ __forceinline__ void fma8(const float (&a)[8], const float (&b)[8], const float (&c)[8], float (&d)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) fma2(a[i], a[i + 1], b[i], b[i + 1], c[i], c[i + 1], d[i], d[i + 1]);
}
__device__ __forceinline__ void mul8(const float (&a)[8], const float (&b)[8], float (&d)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) mul2v(a[i], a[i + 1], b[i], b[i + 1], d[i], d[i + 1]);
}
__device__ __forceinline__ void mul8(const float (&a)[8], float b, float (&d)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i += 2) mul2(a[i], a[i + 1], b, d[i], d[i + 1]);
}
__device__ __forceinline__ float dot8(const float (&a)[8], const float (&b)[8]) {
  float s0, s1;
  mul2v(a[0], a[1], b[0], b[1], s0, s1);
#pragma unroll
  for (int i = 2; i < 8; i += 2) fma2(a[i], a[i + 1], b[i], b[i + 1], s0, s1, s0, s1);
  return s0 + s1;
}

// d = 8 * LANES.  blockIdx.y: q or k.  A group of LANES lanes takes NR_HEADS heads of one row; forward the weights meet
// the angles once for all of them: y = rstd (x (w cos) + x' (w' sin)).  A value's partner comes from its lane, as loaded,
// not by a load of its own.  What limits it is that an item's loads, arithmetic and stores follow one another: warps wait
// for loads most (issue slots 63 % forward, 53 % backward, DRAM 35 % and 44 % of the time), and no load of the next item
// is under way meanwhile.
// Measured, bf16, 36865 rows of 4 + 4 heads of 128: forward 39 - 42 us (3.6 TB/s), backward 56 - 63 us (3.6 TB/s) and the
// sum of dweight's parts 5 - 9 us; fp16, 200003 rows of 8 + 2 heads of 64: 127 and 195 us (4.0 TB/s).
template <typename T, int LANES, int MODE, bool VEC, bool BWD>
__global__ void __launch_bounds__(NR_THREADS, nr_ctas(BWD)) norm_rotary_kernel(NormRotary a) {
  constexpr int D = 8 * LANES, GROUPS = NR_THREADS / LANES;
  __shared__ float s_w[D];
  const int which = (int)blockIdx.x >= a.blocks[0], block = blockIdx.x - (which ? a.blocks[0] : 0), H = a.H[which];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES, e0 = lane * 8;
  const int chunks = (H + NR_HEADS - 1) / NR_HEADS;
  const int64_t items = a.rows * chunks, stride = (int64_t)a.blocks[which] * GROUPS;
  const bool norm = a.w[which] != nullptr, few = items < (1ll << 32);
  const T *x = static_cast<const T *>(a.x[which]);
  const T *dy = BWD ? static_cast<const T *>(a.dy[which]) : nullptr;
  T *out = static_cast<T *>(BWD ? a.dx[which] : a.y[which]);
  const T *turned = BWD ? dy : x;   // what the rotation is applied to
  const int64_t x_rs = a.x_rs[which], x_hs = a.x_hs[which];
  const int64_t turned_rs = BWD ? a.dy_rs[which] : x_rs, turned_hs = BWD ? a.dy_hs[which] : x_hs;
  Rotation rot = a.rot;
  rot.mode = MODE;
  const bool far = MODE == ROTATE_HALVES && e0 < rot.rotary;   // partners are another lane's values
  const int p0 = VEC && far ? partner_of(e0, rot) : e0, partner_lane = (threadIdx.x & 31) - lane + (p0 >> 3);
  for (int e = threadIdx.x; e < D; e += NR_THREADS) s_w[e] = norm ? weight_at<T>(a.w[which], a.w_f32[which], e) : 1.f;
  __syncthreads();

  float dw[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = 0.f;

  // the lanes of a warp stay together: sums go through the whole warp's shuffles
  const int64_t first = (int64_t)block * GROUPS + group, warp_first = first - (group % (32 / LANES));
  for (int64_t n = 0; warp_first + n < items; n += stride) {
    const int64_t item = first + n;
    const bool live = item < items;
    const int64_t row = !live ? 0 : chunks == 1 ? item : few ? (int64_t)((uint32_t)item / (uint32_t)chunks) : item / chunks;
    const int h0 = live ? (int)(item - row * chunks) * NR_HEADS : 0, hn = live ? min(NR_HEADS, H - h0) : 0;
    Raw8<T> own[NR_HEADS], grad[NR_HEADS];
    const T *xr = x + row * x_rs + h0 * x_hs + e0, *tr = turned + row * turned_rs + h0 * turned_hs;
#pragma unroll
    for (int h = 0; h < NR_HEADS; ++h) {
      if (h >= hn) continue;
      own[h] = load8<T, VEC>(xr + h * x_hs);
      if (BWD) grad[h] = load8<T, VEC>(tr + h * turned_hs + e0);
    }
    float c[8], s[8], w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = s_w[e0 + i], c[i] = 1.f, s[i] = 0.f;
    if (MODE != ROTATE_NONE) angles8<VEC>(rot, live ? position_of(a, row) : 0, e0, c, s);
    if (!BWD) {
      mul8(c, w, c);
      if (MODE != ROTATE_NONE) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          s[i] *= s_w[MODE == ROTATE_NEIGHBOURS ? (e0 + i < rot.rotary ? (e0 + i) ^ 1 : e0 + i)
                                                : VEC ? p0 + i : partner_of(e0 + i, rot)];
      }
    }
#pragma unroll
    for (int h = 0; h < NR_HEADS; ++h) {
      // (hn may differ between the groups of a warp)
      if (!__any_sync(0xffffffffu, h < hn)) break;
      const bool on = h < hn;
      float v[8], f[8], t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = f[i] = t[i] = 0.f;   // (t: what is not rotated has no partner)
      if (on) {
        values8<T>(own[h], v);
        if (BWD) values8<T>(grad[h], f);
      }
      if (MODE == ROTATE_HALVES && VEC) {
        const Raw8<T> other = exchanged(0xffffffffu, BWD ? grad[h] : own[h], partner_lane);
        if (on && far) values8<T>(other, t);
      } else if (MODE == ROTATE_HALVES) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (on && e0 + i < rot.rotary) t[i] = to_f32(tr[h * turned_hs + partner_of(e0 + i, rot)]);
      } else if (MODE == ROTATE_NEIGHBOURS) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e0 + i < rot.rotary) t[i] = BWD ? f[i ^ 1] : v[i ^ 1];
      }
      if (!BWD) {
        float rstd = 1.f;
        if (norm) rstd = rsqrtf(group_sum<LANES>(dot8(v, v)) * (1.f / D) + a.eps);
        if (MODE != ROTATE_NONE) {
          mul8(t, s, f);
          fma8(v, c, f, f);
        } else {
          mul8(v, c, f);
        }
        mul8(f, rstd, f);
      } else {
        if (MODE != ROTATE_NONE) {   // back by the same angle
          mul8(t, s, t);
#pragma unroll
          for (int i = 0; i < 8; ++i) t[i] = -t[i];
          fma8(f, c, t, f);
        }
        if (norm) {
          mul8(f, w, t);             // the gradient of x / |x|
          const float ss = group_sum<LANES>(dot8(v, v)), dot = group_sum<LANES>(dot8(t, v));
          const float rstd = rsqrtf(ss * (1.f / D) + a.eps);
          mul8(v, rstd, v);
          fma8(f, v, dw, dw);
          const float mean = -dot * rstd * (1.f / D);
#pragma unroll
          for (int i = 0; i < 8; i += 2) fma2(v[i], v[i + 1], mean, mean, t[i], t[i + 1], f[i], f[i + 1]);
          mul8(f, rstd, f);
        }
      }
      if (on) store8<T>(out + (row * H + h0 + h) * D + e0, f);
    }
  }
  if (BWD && norm) {   // the block's sum of every weight's gradient, its groups in order
    __shared__ float sums[GROUPS][D + 1];
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[group][e0 + i] = dw[i];
    __syncthreads();
    for (int e = threadIdx.x; e < D; e += NR_THREADS) {
      float t = 0.f;
      for (int g = 0; g < GROUPS; ++g) t += sums[g][e];
      a.partial[(int64_t)blockIdx.x * D + e] = t;
    }
  }
}

// Any d and any rotated part: a warp for every head, its values walked twice.
template <typename T, bool BWD>
__global__ void __launch_bounds__(NR_THREADS) norm_rotary_any_kernel(NormRotary a) {
  extern __shared__ float sums[];   // bwd: [warps][d]
  const int which = (int)blockIdx.x >= a.blocks[0], block = blockIdx.x - (which ? a.blocks[0] : 0), H = a.H[which], d = a.d;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool norm = a.w[which] != nullptr, rotate = a.rot.mode != ROTATE_NONE;
  const void *wt = a.w[which];
  const bool wf = a.w_f32[which];
  float *dw = sums + warp * d;
  if (BWD && norm) {
    for (int e = lane; e < d; e += 32) dw[e] = 0.f;
  }
  for (int64_t item = (int64_t)block * (NR_THREADS / 32) + warp; item < a.rows * H;
       item += (int64_t)a.blocks[which] * (NR_THREADS / 32)) {
    const int64_t row = item / H;
    const int h = (int)(item - row * H);
    const T *x = static_cast<const T *>(a.x[which]) + row * a.x_rs[which] + h * a.x_hs[which];
    const T *dy = BWD ? static_cast<const T *>(a.dy[which]) + row * a.dy_rs[which] + h * a.dy_hs[which] : nullptr;
    const int64_t pos = position_of(a, row);
    const bool in = pos >= 0 && pos < a.rot.table_rows;
    const float nan = __int_as_float(0x7fffffff);
    auto turned = [&](int e, auto value, float back) {   // value(e) of the rotated row; back: -1 for the inverse
      float f = value(e);
      if (rotate && e < a.rot.rotary) {
        const int k = angle_of(e, a.rot);
        const float c = in ? a.rot.cos[pos * (a.rot.rotary >> 1) + k] : nan;
        const float s = (in ? a.rot.sin[pos * (a.rot.rotary >> 1) + k] : nan) * (leads(e, a.rot) ? -back : back);
        f = f * c + value(partner_of(e, a.rot)) * s;
      } else if (rotate && !in) {
        f = nan;
      }
      return f;
    };
    float ss = 0.f, dot = 0.f, rstd = 1.f, mean = 0.f;
    if (norm) {
      for (int e = lane; e < d; e += 32) {
        const float v = to_f32(x[e]);
        ss += v * v;
        if (BWD) dot += turned(e, [&](int i) { return to_f32(dy[i]); }, -1.f) * weight_at<T>(wt, wf, e) * v;
      }
      rstd = rsqrtf(group_sum<32>(ss) / d + a.eps);
      if (BWD) mean = group_sum<32>(dot) * rstd / d;
    }
    T *out = static_cast<T *>(BWD ? a.dx[which] : a.y[which]) + item * d;
    for (int e = lane; e < d; e += 32) {
      float f;
      if (!BWD) {
        f = turned(e, [&](int i) { return norm ? to_f32(x[i]) * rstd * weight_at<T>(wt, wf, i) : to_f32(x[i]); }, 1.f);
      } else {
        f = turned(e, [&](int i) { return to_f32(dy[i]); }, -1.f);
        if (norm) {
          const float unit = to_f32(x[e]) * rstd;
          dw[e] += f * unit;
          f = rstd * (f * weight_at<T>(wt, wf, e) - unit * mean);
        }
      }
      out[e] = from_f32<T>(f);
    }
  }
  if (BWD && norm) {
    __syncthreads();
    for (int e = threadIdx.x; e < d; e += NR_THREADS) {
      float t = 0.f;
      for (int w = 0; w < NR_THREADS / 32; ++w) t += sums[w * d + e];
      a.partial[(int64_t)blockIdx.x * d + e] = t;
    }
  }
}

// dweight = sum of the blocks' rows of `partial`, in an order that depends on their number alone
__global__ void __launch_bounds__(1024) norm_rotary_dw_kernel(const float *partial, float *dq_w, float *dk_w, int blocks_q,
                                                             int blocks_k, int d) {
  __shared__ float sums[32][33];
  float *out = blockIdx.y == 0 ? dq_w : dk_w;
  if (out == nullptr) return;
  const int e = blockIdx.x * 32 + threadIdx.x;
  float t = 0.f;
  if (e < d) {
    const int blocks = blockIdx.y ? blocks_k : blocks_q;
    const float *p = partial + (int64_t)(blockIdx.y ? blocks_q : 0) * d + e;
#pragma unroll 8
    for (int b = threadIdx.y; b < blocks; b += 32) t += p[(int64_t)b * d];
  }
  sums[threadIdx.y][threadIdx.x] = t;
  __syncthreads();
  t = group_sum<32>(sums[threadIdx.x][threadIdx.y]);
  if (threadIdx.x == 0 && blockIdx.x * 32 + threadIdx.y < d) out[blockIdx.x * 32 + threadIdx.y] = t;
}

template <typename T, int LANES, int MODE, bool BWD>
void launch_lanes(const NormRotary &a, bool vec, cudaStream_t st) {
  const int grid = a.blocks[0] + a.blocks[1];
  if (vec) norm_rotary_kernel<T, LANES, MODE, true, BWD><<<grid, NR_THREADS, 0, st>>>(a);
  else norm_rotary_kernel<T, LANES, MODE, false, BWD><<<grid, NR_THREADS, 0, st>>>(a);
}
template <typename T, int LANES, bool BWD>
void launch_mode(const NormRotary &a, bool vec, cudaStream_t st) {
  if (a.rot.mode == ROTATE_NONE) return launch_lanes<T, LANES, ROTATE_NONE, BWD>(a, vec, st);
  if (a.rot.mode == ROTATE_HALVES) return launch_lanes<T, LANES, ROTATE_HALVES, BWD>(a, vec, st);
  launch_lanes<T, LANES, ROTATE_NEIGHBOURS, BWD>(a, vec, st);
}

template <typename T, bool BWD>
int launch_type(NormRotary &a, const b200_hstu_norm_rotary_args &p, cudaStream_t st) {
  uintptr_t align = 0;
  for (int i = 0; i < 2; ++i) {
    if (a.H[i] == 0) continue;
    align |= (uintptr_t)a.x[i] | (uintptr_t)(a.x_rs[i] * (int64_t)sizeof(T)) | (uintptr_t)(a.x_hs[i] * (int64_t)sizeof(T));
    if (BWD)
      align |= (uintptr_t)a.dy[i] | (uintptr_t)(a.dy_rs[i] * (int64_t)sizeof(T)) |
               (uintptr_t)(a.dy_hs[i] * (int64_t)sizeof(T));
  }
  if (a.rot.mode != ROTATE_NONE) align |= (uintptr_t)a.rot.cos | (uintptr_t)a.rot.sin | (uintptr_t)(a.rot.rotary % 16);
  const bool vec = (align & 15) == 0, lanes = a.d == 64 || a.d == 128 || a.d == 256;
  // one wave of CTAs (two where no partial sums follow), q's and k's by their shares of the work (an item of h heads costs about 2 + h), no more than
  // there are items for
  const int most = 148 * (lanes ? nr_ctas(BWD) * (BWD ? 1 : 2) : 4), per = lanes ? NR_THREADS / (a.d / 8) : NR_THREADS / 32;
  auto cost = [&](int i) { return (int64_t)2 * ((a.H[i] + NR_HEADS - 1) / NR_HEADS) + a.H[i]; };
  for (int i = 0; i < 2; ++i) {
    const int64_t items = a.rows * (lanes ? (a.H[i] + NR_HEADS - 1) / NR_HEADS : a.H[i]), want = (items + per - 1) / per;
    const int64_t share = a.H[i] == 0 ? 0 : (most * cost(i) + cost(0) + cost(1) - 1) / (cost(0) + cost(1));
    a.blocks[i] = (int)(want < share ? want : share);
  }
  if (a.d == 64) {
    launch_mode<T, 8, BWD>(a, vec, st);
  } else if (a.d == 128) {
    launch_mode<T, 16, BWD>(a, vec, st);
  } else if (a.d == 256) {
    launch_mode<T, 32, BWD>(a, vec, st);
  } else {
    const size_t smem = BWD ? (NR_THREADS / 32) * a.d * sizeof(float) : 0;
    norm_rotary_any_kernel<T, BWD><<<a.blocks[0] + a.blocks[1], NR_THREADS, smem, st>>>(a);
  }
  count_launch();
  B200_CHECK_LAUNCH("norm_rotary_kernel");
  if (BWD && (a.w[0] || a.w[1])) {
    norm_rotary_dw_kernel<<<dim3((a.d + 31) / 32, 2), dim3(32, 32), 0, st>>>(a.partial, a.w[0] ? p.dweight[0] : nullptr,
                                                                           a.w[1] ? p.dweight[1] : nullptr, a.blocks[0],
                                                                           a.blocks[1], a.d);
    count_launch();
    B200_CHECK_LAUNCH("norm_rotary_dw_kernel");
  }
  return 0;
}

}  // namespace

int64_t norm_rotary_bwd_workspace_bytes(int d) { return (int64_t)(NR_MAX_BLOCKS + 2) * d * (int64_t)sizeof(float); }

int check_rotation(const char *what, const float *cos, const float *sin, int64_t table_rows, int rotary, int interleaved,
                   int d, Rotation &out) {
  out.cos = cos;
  out.sin = sin;
  out.table_rows = table_rows;
  out.rotary = rotary;
  out.mode = interleaved ? ROTATE_NEIGHBOURS : ROTATE_HALVES;
  if (!cos || !sin) return fail(B200_HSTU_EINVAL, "%s: a rotation needs both tables", what);
  if (rotary <= 0 || rotary > d || rotary % 2 != 0 || table_rows <= 0)
    return fail(B200_HSTU_EINVAL, "%s: the rotated part must be even, positive and at most the head dimension", what);
  return 0;
}

int norm_rotary(const b200_hstu_norm_rotary_args &p, bool bwd, cudaStream_t st) {
  NormRotary a = {};
  if (p.rows < 0 || p.H[0] < 0 || p.H[1] < 0 || p.d <= 0) return fail(B200_HSTU_EINVAL, "norm_rotary: bad size");
  if (p.d > 1024) return fail(B200_HSTU_EUNSUPPORTED, "norm_rotary: heads of more than 1024 values");
  a.rows = p.rows;
  a.d = p.d;
  a.eps = p.eps;
  a.positions = static_cast<const int32_t *>(p.positions);
  a.pos_step = (p.index_flags & B200_HSTU_OFFSETS_I64) ? 2 : 1;
  if (p.positions || p.cos || p.sin) {
    if (!p.positions && p.rows > 0) return fail(B200_HSTU_EINVAL, "norm_rotary: a rotation needs positions");
    if (int rc = check_rotation("norm_rotary", p.cos, p.sin, p.table_rows, p.rotary, p.interleaved, p.d, a.rot)) return rc;
  }
  for (int i = 0; i < 2; ++i) {
    a.H[i] = p.H[i];
    a.x[i] = p.x[i], a.y[i] = p.y[i], a.dy[i] = p.dy[i], a.dx[i] = p.dx[i], a.w[i] = p.H[i] > 0 ? p.weight[i] : nullptr;
    a.x_rs[i] = p.x_row_stride[i], a.x_hs[i] = p.x_head_stride[i];
    a.dy_rs[i] = p.dy_row_stride[i], a.dy_hs[i] = p.dy_head_stride[i];
    a.w_f32[i] = p.weight_dtype[i] == B200_HSTU_F32;
    if (a.w[i] && p.weight_dtype[i] != B200_HSTU_F32 && p.weight_dtype[i] != p.dtype)
      return fail(B200_HSTU_EINVAL, "norm_rotary: weights must be float32 or of the activations' type");
    if (p.H[i] > 0 && p.rows > 0 && (!p.x[i] || (bwd ? !p.dy[i] || !p.dx[i] : !p.y[i])))
      return fail(B200_HSTU_EINVAL, "norm_rotary: null tensor");
    if (p.H[i] > 0 && p.rows > 0 && ((uintptr_t)(bwd ? p.dx[i] : p.y[i]) & 15) != 0)
      return fail(B200_HSTU_EINVAL, "norm_rotary: results must be 16-byte aligned");
    if (bwd && a.w[i] && !p.dweight[i]) return fail(B200_HSTU_EINVAL, "norm_rotary: null tensor");
  }
  for (int i = 0; bwd && i < 2; ++i) {   // a sum over nothing
    if (!p.weight[i] || !p.dweight[i] || (p.rows > 0 && p.H[i] > 0)) continue;
    if (int rc = check_cuda(cudaMemsetAsync(p.dweight[i], 0, p.d * sizeof(float), st), "cudaMemsetAsync")) return rc;
  }
  if (p.rows == 0 || p.H[0] + p.H[1] == 0) return 0;
  if (bwd && (a.w[0] || a.w[1])) {
    a.partial = static_cast<float *>(p.workspace);
    if (!p.workspace || p.workspace_bytes < norm_rotary_bwd_workspace_bytes(p.d))
      return fail(B200_HSTU_EWORKSPACE, "norm_rotary: workspace of %lld bytes needed",
                  (long long)norm_rotary_bwd_workspace_bytes(p.d));
  }
  ProfileScope prof(bwd ? PROF_NORM_ROTARY_BWD : PROF_NORM_ROTARY_FWD, st);
  switch (p.dtype) {
    case B200_HSTU_F32: return bwd ? launch_type<float, true>(a, p, st) : launch_type<float, false>(a, p, st);
    case B200_HSTU_BF16: return bwd ? launch_type<__nv_bfloat16, true>(a, p, st) : launch_type<__nv_bfloat16, false>(a, p, st);
    case B200_HSTU_F16: return bwd ? launch_type<__half, true>(a, p, st) : launch_type<__half, false>(a, p, st);
    default: return fail(B200_HSTU_EINVAL, "unknown dtype %d", p.dtype);
  }
}

}  // namespace b200hstu
