// The per-head transform of queries and keys, shared by the kernels that norm and rotate rows of a dense tensor
// (rotary.cu) and by the one that does so on the way into a key/value cache (kv_cache.cu):
//
//     h = x / sqrt(mean(x^2) + eps) * gain                       (normalize != 0)
//     (y_a, y_b) = (h_a cos t - h_b sin t,  h_b cos t + h_a sin t),   t = position[axis(i)] * frequency[i]
//
// for every rotated pair i, whose two elements are (i, i + pairs) or, interleaved, (2 i, 2 i + 1); the elements behind
// 2 * pairs pass through.  The pairs are dealt to the position axes in consecutive sections.
//
// A row of d elements belongs to a group of LPR lanes, four pairs ("slots") and so eight elements a lane: both elements
// of a pair sit in one lane, and the row's sum of squares is the only exchange.  Slot j's elements are those of pair j;
// slots j >= pairs hold the pass-through elements 2 j, 2 j + 1 with cos = 1, sin = 0.
//
// The angle is reduced in turns in f64: position * (frequency / 2 pi) minus its nearest whole number loses
// 2^-53 * |turns|, nothing that f32 sees for any 32-bit position; the remainder's sine and cosine are f32.
// Statistics and products are f32; the one rounding to f16 is the store's.
#pragma once
#include "common.cuh"

namespace b200 {
namespace heads {

constexpr int MAX_D = 256;
constexpr int AXES = 3;

struct Transform {
  const double* freq = nullptr;    // pairs radians per position
  int pairs = 0;
  int end0 = 0, end1 = 0;          // pairs [0, end0) turn with axis 0, [end0, end1) with axis 1, the others with axis 2
  int normalize = 0;
  float eps = 0.f;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(__half* p, float x) { *p = __float2half_rn(x); }

// Four consecutive elements: 8 bytes of f16, 16 of f32.
__device__ __forceinline__ void load4(const __half* p, float (&v)[4]) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&raw.x));
  const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
  v[0] = x.x; v[1] = x.y; v[2] = y.x; v[3] = y.y;
}
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 x = *reinterpret_cast<const float4*>(p);
  v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
}
__device__ __forceinline__ void store4(__half* p, const float (&v)[4]) {
  const __half2 x = __floats2half2_rn(v[0], v[1]), y = __floats2half2_rn(v[2], v[3]);
  uint2 raw;
  raw.x = *reinterpret_cast<const uint32_t*>(&x);
  raw.y = *reinterpret_cast<const uint32_t*>(&y);
  *reinterpret_cast<uint2*>(p) = raw;
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}

// Where a lane's eight elements lie.  u and v are the two runs of four that a vector access moves (VEC); a and b the
// pairs' elements.  Interleaved, the lane's eight elements are consecutive and a, b alternate through them.
template <bool INTER, bool VEC>
struct Lane {
  int j0, d, pairs, off_u, off_v;
  bool live;                       // the lane has elements
  __device__ __forceinline__ Lane(int lane, int d_, int pairs_) : j0(lane * 4), d(d_), pairs(pairs_) {
    const bool split = !INTER && j0 < pairs;
    off_u = split ? j0 : 2 * j0;
    off_v = split ? j0 + pairs : 2 * j0 + 4;
    live = 2 * j0 < d;
  }
  __device__ __forceinline__ int at_a(int e) const { return (!INTER && j0 + e < pairs) ? j0 + e : 2 * (j0 + e); }
  __device__ __forceinline__ int at_b(int e) const { return (!INTER && j0 + e < pairs) ? j0 + e + pairs : 2 * (j0 + e) + 1; }
  __device__ __forceinline__ bool has(int e) const { return 2 * (j0 + e) < d; }
  // the element behind the lane's e-th register: a[0..3], then b[0..3].  A vector access leaves a pass-through lane's
  // two runs as they lie; nothing there depends on which of the two a register belongs to.
  __device__ __forceinline__ int at(int e) const {
    if constexpr (VEC && !INTER) return (e < 4 ? off_u : off_v) + (e & 3);
    return e < 4 ? at_a(e) : at_b(e - 4);
  }

  template <typename T>
  __device__ __forceinline__ void load(const T* row, float (&a)[4], float (&b)[4]) const {
    if constexpr (VEC) {
      float u[4], v[4];
      load4(row + off_u, u);
      load4(row + off_v, v);
      if constexpr (INTER) {
        a[0] = u[0]; b[0] = u[1]; a[1] = u[2]; b[1] = u[3]; a[2] = v[0]; b[2] = v[1]; a[3] = v[2]; b[3] = v[3];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) { a[e] = u[e]; b[e] = v[e]; }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        a[e] = has(e) ? to_f(row[at_a(e)]) : 0.f;
        b[e] = has(e) ? to_f(row[at_b(e)]) : 0.f;
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&a)[4], const float (&b)[4]) const {
    if constexpr (VEC) {
      if constexpr (INTER) {
        const float u[4] = {a[0], b[0], a[1], b[1]}, v[4] = {a[2], b[2], a[3], b[3]};
        store4(row + off_u, u);
        store4(row + off_v, v);
      } else {
        store4(row + off_u, a);
        store4(row + off_v, b);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (has(e)) { put(row + at_a(e), a[e]); put(row + at_b(e), b[e]); }
    }
  }
};

// Turns per position of a lane's four slots (0 for slots that do not rotate) and the axis each turns with.
struct Turns {
  double per_pos[4];
  int axis[4];
  __device__ __forceinline__ void init(const Transform& t, int j0) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int j = j0 + e;
      per_pos[e] = j < t.pairs ? t.freq[j] * 0.15915494309189535 : 0.0;
      axis[e] = j < t.end0 ? 0 : j < t.end1 ? 1 : 2;
    }
  }
  __device__ __forceinline__ void at(int p0, int p1, int p2, float (&c)[4], float (&s)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      double x = (double)(axis[e] == 0 ? p0 : axis[e] == 1 ? p1 : p2) * per_pos[e];
      x -= rint(x);
      sincospif(2.f * (float)x, &s[e], &c[e]);
    }
  }
};

template <int LPR>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
template <int LPR>
__device__ __forceinline__ float group_max(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float sum8(const float (&a)[4], const float (&b)[4], const float (&c)[4], const float (&d)[4]) {
  float x = a[0] * c[0], y = b[0] * d[0];
#pragma unroll
  for (int e = 1; e < 4; ++e) { x = fmaf(a[e], c[e], x); y = fmaf(b[e], d[e], y); }
  return x + y;
}

// Turns slots [0, n) of the lane's four by the angle whose cosine and sine are given; `BACK` by its negative.  The other
// slots are left alone rather than turned by 0: an infinity among pass-through elements would make its neighbour NaN.
template <bool BACK>
__device__ __forceinline__ void turn(float (&a)[4], float (&b)[4], const float (&c)[4], const float (&s)[4], int n) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float x = a[e], y = b[e], t = BACK ? -s[e] : s[e];
    const float ta = fmaf(x, c[e], -(y * t)), tb = fmaf(y, c[e], x * t);
    a[e] = e < n ? ta : x;
    b[e] = e < n ? tb : y;
  }
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
// Checks a b200_head_op against the head size and takes it apart.  `axes`: how many position axes it reads.
inline int parse(const b200_head_op* op, size_t d, Transform* t, int* axes) {
  if (!op) return B200_ERR_NULL;
  size_t pairs = 0;
  *axes = 0;
  for (int a = 0; a < AXES; ++a) {
    if (op->axis_pairs[a] > MAX_D) return B200_ERR_SHAPE;
    pairs += op->axis_pairs[a];
    if (op->axis_pairs[a]) *axes = a + 1;
  }
  if (2 * pairs > d) return B200_ERR_SHAPE;
  if (pairs && !op->frequencies) return B200_ERR_NULL;
  if (!op->normalize && (op->q_gain || op->k_gain)) return B200_ERR_UNSUPPORTED;   // a gain belongs to the norm
  t->freq = op->frequencies;
  t->pairs = (int)pairs;
  t->end0 = (int)op->axis_pairs[0];
  t->end1 = (int)(op->axis_pairs[0] + op->axis_pairs[1]);
  t->normalize = op->normalize != 0;
  t->eps = (float)op->epsilon;
  return B200_OK;
}

inline int lanes_per_row(int64_t d) { return d <= 64 ? 8 : d <= 128 ? 16 : 32; }

}  // namespace heads
}  // namespace b200
