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

// Two f32 in one register pair: Blackwell's packed multiply, add and multiply-add take one issue slot for both.
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack(f2 v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 both(float x) { return pack(x, x); }
__device__ __forceinline__ f2 neg2(f2 v) { return v ^ 0x8000000080000000ull; }

// A lane's eight elements of a row: the pairs' first elements a = (a0, a1), (a2, a3) and their second ones b.
struct Row {
  f2 a[2], b[2];
};
__device__ __forceinline__ f2 dot(const Row& x, const Row& y) {      // two partial sums
  return fma2(x.b[1], y.b[1], fma2(x.b[0], y.b[0], fma2(x.a[1], y.a[1], mul2(x.a[0], y.a[0]))));
}
__device__ __forceinline__ Row times(const Row& x, const Row& y) {
  return {{mul2(x.a[0], y.a[0]), mul2(x.a[1], y.a[1])}, {mul2(x.b[0], y.b[0]), mul2(x.b[1], y.b[1])}};
}
__device__ __forceinline__ Row scaled(const Row& x, float f) {
  const f2 w = both(f);
  return {{mul2(x.a[0], w), mul2(x.a[1], w)}, {mul2(x.b[0], w), mul2(x.b[1], w)}};
}

// A row's elements as they were loaded: two runs of four (VEC), f16 still packed.  Holding these rather than the f32
// values lets a lane have four rows of f16 on their way in 16 registers.
template <typename T, bool VEC> struct Raw { float x[8]; };
template <> struct Raw<__half, true> { uint2 u, v; };
template <> struct Raw<float, true> { float4 u, v; };

__device__ __forceinline__ float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t half2_of(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Where a lane's eight elements lie.  off_u and off_v start the two runs of four that a vector access moves (VEC, whole
// lanes rotate or none of it: the number of pairs is a multiple of 4); a and b are the pairs' elements.  Interleaved, the
// eight elements are consecutive and a, b alternate through them.
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
  // the element behind the lane's e-th value: a0..a3, then b0..b3.  A vector access leaves a pass-through lane's two runs
  // as they lie; nothing there depends on which of the two a value belongs to.
  __device__ __forceinline__ int at(int e) const {
    if constexpr (VEC && !INTER) return (e < 4 ? off_u : off_v) + (e & 3);
    return e < 4 ? at_a(e) : at_b(e - 4);
  }

  template <typename T>
  __device__ __forceinline__ void load(const T* row, Raw<T, VEC>& r) const {
    if constexpr (!VEC) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r.x[e] = has(e & 3) ? to_f(row[at(e)]) : 0.f;
    } else if constexpr (sizeof(T) == 2) {
      r.u = *reinterpret_cast<const uint2*>(row + off_u);
      r.v = *reinterpret_cast<const uint2*>(row + off_v);
    } else {
      r.u = *reinterpret_cast<const float4*>(row + off_u);
      r.v = *reinterpret_cast<const float4*>(row + off_v);
    }
  }
  template <typename T>
  __device__ __forceinline__ void clear(Raw<T, VEC>& r) const {
    if constexpr (!VEC) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r.x[e] = 0.f;
    } else if constexpr (sizeof(T) == 2) {
      r.u = r.v = make_uint2(0, 0);
    } else {
      r.u = r.v = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
  template <typename T>
  __device__ __forceinline__ Row row(const Raw<T, VEC>& r) const {
    float u[4], v[4];
    if constexpr (!VEC) return {{pack(r.x[0], r.x[1]), pack(r.x[2], r.x[3])}, {pack(r.x[4], r.x[5]), pack(r.x[6], r.x[7])}};
    else if constexpr (sizeof(T) == 2) {
      const float2 w = halves(r.u.x), x = halves(r.u.y), y = halves(r.v.x), z = halves(r.v.y);
      u[0] = w.x; u[1] = w.y; u[2] = x.x; u[3] = x.y;
      v[0] = y.x; v[1] = y.y; v[2] = z.x; v[3] = z.y;
    } else {
      u[0] = r.u.x; u[1] = r.u.y; u[2] = r.u.z; u[3] = r.u.w;
      v[0] = r.v.x; v[1] = r.v.y; v[2] = r.v.z; v[3] = r.v.w;
    }
    if constexpr (INTER) return {{pack(u[0], u[2]), pack(v[0], v[2])}, {pack(u[1], u[3]), pack(v[1], v[3])}};
    return {{pack(u[0], u[1]), pack(u[2], u[3])}, {pack(v[0], v[1]), pack(v[2], v[3])}};
  }
  // the values in run order (VEC): u0..u3, v0..v3; otherwise a0..a3, b0..b3
  __device__ __forceinline__ void values(const Row& x, float (&u)[4], float (&v)[4]) const {
    if constexpr (INTER && VEC) {
      unpack(x.a[0], u[0], u[2]); unpack(x.b[0], u[1], u[3]);
      unpack(x.a[1], v[0], v[2]); unpack(x.b[1], v[1], v[3]);
    } else {
      unpack(x.a[0], u[0], u[1]); unpack(x.a[1], u[2], u[3]);
      unpack(x.b[0], v[0], v[1]); unpack(x.b[1], v[2], v[3]);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const Row& x) const {
    float u[4], v[4];
    values(x, u, v);
    if constexpr (!VEC) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (has(e)) { put(row + at(e), u[e]); put(row + at(4 + e), v[e]); }
    } else if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint2*>(row + off_u) = make_uint2(half2_of(u[0], u[1]), half2_of(u[2], u[3]));
      *reinterpret_cast<uint2*>(row + off_v) = make_uint2(half2_of(v[0], v[1]), half2_of(v[2], v[3]));
    } else {
      *reinterpret_cast<float4*>(row + off_u) = make_float4(u[0], u[1], u[2], u[3]);
      *reinterpret_cast<float4*>(row + off_v) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  template <typename T>
  __device__ __forceinline__ Row gain(const T* g) const {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = g && has(e & 3) ? to_f(g[at(e)]) : 1.f;
    return ordered(x);
  }
  // eight values in at()'s order as a Row
  __device__ __forceinline__ Row ordered(const float (&x)[8]) const {
    return {{pack(x[0], x[1]), pack(x[2], x[3])}, {pack(x[4], x[5]), pack(x[6], x[7])}};
  }
};

// cos and sin of a lane's four slots at a token's positions, c as (c0, c1), (c2, c3); 1 and 0 where nothing rotates.
struct Angle {
  f2 c[2], s[2];
};
__device__ __forceinline__ Angle angle_at(const Transform& t, int j0, int p0, int p1, int p2) {
  float c[4], s[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int j = j0 + e;
    c[e] = 1.f;
    s[e] = 0.f;
    if (j < t.pairs) {
      double x = (double)(j < t.end0 ? p0 : j < t.end1 ? p1 : p2) * (__ldg(t.freq + j) * 0.15915494309189535);
      x -= rint(x);
      sincospif(2.f * (float)x, &s[e], &c[e]);
    }
  }
  return {{pack(c[0], c[1]), pack(c[2], c[3])}, {pack(s[0], s[1]), pack(s[2], s[3])}};
}

// x turned by the angle.  Slots that do not rotate are left alone rather than turned by 0: an infinity among pass-through
// elements would make its neighbour NaN.  VEC lanes rotate as a whole or not at all.
template <bool VEC>
__device__ __forceinline__ Row turned(const Row& x, const f2 (&c)[2], const f2 (&s)[2], int j0, int pairs) {
  if (VEC && j0 >= pairs) return x;
  Row y;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    y.a[e] = fma2(x.b[e], neg2(s[e]), mul2(x.a[e], c[e]));
    y.b[e] = fma2(x.a[e], s[e], mul2(x.b[e], c[e]));
    if constexpr (!VEC) {
      float ya[2], yb[2], xa[2], xb[2];
      unpack(y.a[e], ya[0], ya[1]); unpack(y.b[e], yb[0], yb[1]);
      unpack(x.a[e], xa[0], xa[1]); unpack(x.b[e], xb[0], xb[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (j0 + 2 * e + i >= pairs) { ya[i] = xa[i]; yb[i] = xb[i]; }
      y.a[e] = pack(ya[0], ya[1]); y.b[e] = pack(yb[0], yb[1]);
    }
  }
  return y;
}

template <int LPR>
__device__ __forceinline__ float group_sum(f2 v) {
  float x, y;
  unpack(v, x, y);
  x += y;
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
// Two sums at once.
template <int LPR>
__device__ __forceinline__ void group_sum_pair(f2 v, f2 w, float& x, float& y) {
  float a, b, c, d;
  unpack(v, a, b);
  unpack(w, c, d);
  f2 z = add2(pack(a, c), pack(b, d));
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) z = add2(z, __shfl_xor_sync(0xffffffffu, z, o));
  unpack(z, x, y);
}

template <int LPR>
__device__ __forceinline__ float group_max(float x) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// gain * x / sqrt(mean(x^2) + eps), then the turn: the whole forward transform of a row.  The gain is folded into the
// angle by the caller (coef): what is left is one scale by the reciprocal root.
struct Coef {
  f2 ac[2], bs[2], bc[2], as[2];   // gain_a cos, -gain_b sin, gain_b cos, gain_a sin
};
__device__ __forceinline__ Coef coef(const Angle& t, const Row& gain) {
  Coef k;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    k.ac[e] = mul2(gain.a[e], t.c[e]);
    k.as[e] = mul2(gain.a[e], t.s[e]);
    k.bc[e] = mul2(gain.b[e], t.c[e]);
    k.bs[e] = neg2(mul2(gain.b[e], t.s[e]));
  }
  return k;
}
template <int LPR, bool VEC>
__device__ __forceinline__ Row transformed(const Row& x, const Coef& k, const Transform& t, int j0, float inv_d) {
  Row y;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    y.a[e] = mul2(x.a[e], k.ac[e]);                        // slots that do not rotate: cos is 1, this is all
    y.b[e] = mul2(x.b[e], k.bc[e]);
    if (VEC && j0 >= t.pairs) continue;
    const f2 ta = fma2(x.b[e], k.bs[e], y.a[e]), tb = fma2(x.a[e], k.as[e], y.b[e]);
    if constexpr (VEC) {
      y.a[e] = ta;
      y.b[e] = tb;
    } else {
      float ya[2], yb[2], za[2], zb[2];
      unpack(y.a[e], ya[0], ya[1]); unpack(y.b[e], yb[0], yb[1]);
      unpack(ta, za[0], za[1]); unpack(tb, zb[0], zb[1]);
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (j0 + 2 * e + i < t.pairs) { ya[i] = za[i]; yb[i] = zb[i]; }
      y.a[e] = pack(ya[0], ya[1]); y.b[e] = pack(yb[0], yb[1]);
    }
  }
  if (t.normalize) y = scaled(y, rsqrtf(group_sum<LPR>(dot(x, x)) * inv_d + t.eps));
  return y;
}

// Positions of a token on the axes: pos is axes x n, or null for the one index on every axis.
struct Place { int p0, p1, p2; };
__device__ __forceinline__ Place place_of(const int* pos, int axes, long long n, long long tok, int index) {
  Place p;
  p.p0 = pos ? __ldg(pos + tok) : index;
  p.p1 = pos && axes > 1 ? __ldg(pos + n + tok) : p.p0;
  p.p2 = pos && axes > 2 ? __ldg(pos + 2 * n + tok) : p.p0;
  return p;
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
