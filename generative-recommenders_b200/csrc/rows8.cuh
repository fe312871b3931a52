// Pieces of eight consecutive values of a row, which the kernels over heads (rotary.cu, paged_cache.cu) give
// each lane: loads and stores, the rotation of pairs, and the sequence that a row of a jagged batch is in.
#pragma once

#include "common.cuh"

namespace b200hstu {

// 16 bytes of a 16-bit type, 32 bytes of float
template <typename T> struct Raw8 { uint4 v[sizeof(T) / 2]; };

// VEC: the address is 16-byte aligned
template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load8(const T *p) {
  Raw8<T> r;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
  } else {
    T *e = reinterpret_cast<T *>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i];
  }
  return r;
}
// another lane's piece; all lanes of `mask` call
template <typename T>
__device__ __forceinline__ Raw8<T> exchanged(uint32_t mask, const Raw8<T> &r, int from) {
  Raw8<T> o;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
    o.v[i].x = __shfl_sync(mask, r.v[i].x, from);
    o.v[i].y = __shfl_sync(mask, r.v[i].y, from);
    o.v[i].z = __shfl_sync(mask, r.v[i].z, from);
    o.v[i].w = __shfl_sync(mask, r.v[i].w, from);
  }
  return o;
}
template <typename T>
__device__ __forceinline__ void values8(const Raw8<T> &r, float (&f)[8]) {
  const T *e = reinterpret_cast<const T *>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32(e[i]);
}
template <typename T>   // (16-byte aligned)
__device__ __forceinline__ void store8(T *p, const float (&f)[8]) {
  Raw8<T> r;
  T *e = reinterpret_cast<T *>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(f[i]);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4 *>(p)[i] = r.v[i];
}

// weights: float32 or the activations' type
template <typename T>
__device__ __forceinline__ float weight_at(const void *w, bool is_f32, int i) {
  return is_f32 ? static_cast<const float *>(w)[i] : to_f32(static_cast<const T *>(w)[i]);
}

// How the leading values of a head are rotated.  Values e < rotary have a partner and share one angle with it:
// HALVES: e and e +- rotary / 2, angle e mod rotary / 2; NEIGHBOURS: 2i and 2i + 1, angle i.
enum { ROTATE_NONE = 0, ROTATE_HALVES = 1, ROTATE_NEIGHBOURS = 2 };
struct Rotation {
  const float *cos, *sin;
  int64_t table_rows;
  int rotary, mode;
};
__device__ __forceinline__ int partner_of(int e, const Rotation &r) {
  if (e >= r.rotary) return e;
  if (r.mode == ROTATE_NEIGHBOURS) return e ^ 1;
  const int h = r.rotary >> 1;
  return e < h ? e + h : e - h;
}
__device__ __forceinline__ int angle_of(int e, const Rotation &r) {
  if (r.mode == ROTATE_NEIGHBOURS) return e >> 1;
  const int h = r.rotary >> 1;
  return e < h ? e : e - h;
}
// the first of its pair?  (a cos - b sin; the second is b cos + a sin)
__device__ __forceinline__ bool leads(int e, const Rotation &r) {
  return r.mode == ROTATE_NEIGHBOURS ? (e & 1) == 0 : e < (r.rotary >> 1);
}

// Cosines, and sines with the sign that they have in `own * c + partner * s`, of a lane's eight values;
// positions outside the tables give NaN, as cosines of values that are not rotated too.  VEC: rotary is a multiple of 16 and the tables are 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ void angles8(const Rotation &r, int64_t pos, int e0, float (&c)[8], float (&s)[8]) {
  const bool in = pos >= 0 && pos < r.table_rows;
  const int64_t row = (in ? pos : 0) * (r.rotary >> 1);
  const float nan = __int_as_float(0x7fffffff);
  if (VEC && e0 < r.rotary) {   // (all eight are rotated)
    const int first = angle_of(e0, r);
    if (r.mode == ROTATE_NEIGHBOURS) {
      const float4 a = __ldg(reinterpret_cast<const float4 *>(r.cos + row + first));
      const float4 b = __ldg(reinterpret_cast<const float4 *>(r.sin + row + first));
      c[0] = c[1] = a.x, c[2] = c[3] = a.y, c[4] = c[5] = a.z, c[6] = c[7] = a.w;
      s[0] = -b.x, s[1] = b.x, s[2] = -b.y, s[3] = b.y, s[4] = -b.z, s[5] = b.z, s[6] = -b.w, s[7] = b.w;
    } else {
      const float sign = leads(e0, r) ? -1.f : 1.f;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 a = __ldg(reinterpret_cast<const float4 *>(r.cos + row + first) + i);
        const float4 b = __ldg(reinterpret_cast<const float4 *>(r.sin + row + first) + i);
        c[4 * i] = a.x, c[4 * i + 1] = a.y, c[4 * i + 2] = a.z, c[4 * i + 3] = a.w;
        s[4 * i] = sign * b.x, s[4 * i + 1] = sign * b.y, s[4 * i + 2] = sign * b.z, s[4 * i + 3] = sign * b.w;
      }
    }
    if (!in) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = s[i] = nan;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = e0 + i;
    c[i] = in ? 1.f : nan, s[i] = 0.f;
    if (e < r.rotary) {
      const int k = angle_of(e, r);
      c[i] = in ? r.cos[row + k] : nan;
      s[i] = in ? (leads(e, r) ? -r.sin[row + k] : r.sin[row + k]) : nan;
    }
  }
}

// The sequence of row i of a jagged batch: the last b with offsets[b] <= i; B where i lies past the end.
__device__ __forceinline__ int sequence_of(const IndexTensor &offsets, int B, int64_t i) {
  int lo = 0, hi = B + 1;   // offsets[lo] <= i < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= i) lo = mid; else hi = mid;
  }
  return lo;
}

}  // namespace b200hstu
