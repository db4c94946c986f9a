// The per-head transform of queries and keys, shared by the kernels that norm and rotate rows of a dense tensor
// (rotary.cu) and by the one that does so on the way into a key/value cache (kv_cache.cu):
//
//     h = x / sqrt(mean(x^2) + eps) * gain                       (normalize != 0)
//     (y_a, y_b) = (h_a cos t - h_b sin t,  h_b cos t + h_a sin t),   t = position[axis(i)] * frequency[i]
//
// for every rotated pair i, whose two elements are (i, i + pairs) or, interleaved, (2 i, 2 i + 1); the elements behind
// 2 * pairs pass through.  The pairs are dealt to the position axes in consecutive sections.
//
// A row of d elements belongs to a group of LPR lanes with S pairs ("slots"), 2 S elements, a lane: both elements of a pair
// sit in one lane, and the row's sum of squares is the only exchange.  Slot j's elements are those of pair j; slots
// j >= pairs hold the pass-through elements 2 j, 2 j + 1 with cos = 1, sin = 0.  S is 8 in the forward of f16 rows that
// 16-byte accesses fit, else 4.
//
// The angle is reduced in turns: position * (frequency / 2 pi) minus its nearest whole number, the quotient in two f64
// parts and the product fused with the subtraction.  (With the quotient and the product rounded to f64 the remainder is off
// by up to 2^-52 * |turns|: 5e-7 radians at position 2^31 and frequency 1, and more with the frequency.)  What is left is
// below 2^-50 turns at any 32-bit position and frequencies up to 2^20.  Sine and cosine are those of the remainder's f32
// part, with the rest's share added: 1.5 * 2^-24.  (Without the rest, off by up to 1.6 * 2^-24 more, 291 of 133 million keys
// came to lie on the other side of a code's boundary than exact ones, with it 176; it costs the append 0.5 of 77 us.)
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

// Two f32 side by side.  (Blackwell's packed f32x2 instructions were tried here: what they save in arithmetic goes into
// moving values into register pairs, 70 us against 66 for the forward of 16384 tokens, 40 heads of 128.)
struct f2 { float x, y; };
__device__ __forceinline__ f2 pack(float x, float y) { return {x, y}; }
__device__ __forceinline__ void unpack(f2 v, float& x, float& y) { x = v.x; y = v.y; }
__device__ __forceinline__ f2 mul2(f2 a, f2 b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ f2 add2(f2 a, f2 b) { return {a.x + b.x, a.y + b.y}; }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) { return {fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)}; }
__device__ __forceinline__ f2 neg2(f2 v) { return {-v.x, -v.y}; }

// A lane's 2 S elements of a row: the pairs' first elements a = (a0, a1), (a2, a3), ... and their second ones b.
template <int S> struct Row {
  f2 a[S / 2], b[S / 2];
};
template <int S>
__device__ __forceinline__ f2 dot(const Row<S>& x, const Row<S>& y) {          // two partial sums
  f2 r = mul2(x.a[0], y.a[0]), t = mul2(x.b[0], y.b[0]);
#pragma unroll
  for (int e = 1; e < S / 2; ++e) { r = fma2(x.a[e], y.a[e], r); t = fma2(x.b[e], y.b[e], t); }
  return add2(r, t);
}
template <int S>
__device__ __forceinline__ Row<S> times(const Row<S>& x, const Row<S>& y) {
  Row<S> r;
#pragma unroll
  for (int e = 0; e < S / 2; ++e) { r.a[e] = mul2(x.a[e], y.a[e]); r.b[e] = mul2(x.b[e], y.b[e]); }
  return r;
}

// A row's elements as they were loaded: two runs of S (VEC), f16 still packed.  Holding these rather than the f32 values
// lets a lane have several rows on their way in few registers.
template <typename T, int S, bool VEC> struct Raw { float x[2 * S]; };
template <> struct Raw<__half, 8, true> { uint4 u, v; };
template <> struct Raw<__half, 4, true> { uint2 u, v; };
template <> struct Raw<float, 4, true> { uint4 u, v; };

__device__ __forceinline__ float2 halves(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ uint32_t half2_of(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Where a lane's 2 S elements lie.  off_u and off_v start the two runs of S that a vector access moves (VEC: whole lanes
// rotate or none of it, the number of pairs being a multiple of S); a and b are the pairs' elements.  Interleaved, the
// elements are consecutive and a, b alternate through them.
template <typename T, int S, bool INTER, bool VEC>
struct Lane {
  int j0, d, pairs, off_u, off_v;
  bool live;                       // the lane has elements
  __device__ __forceinline__ Lane(int lane, int d_, int pairs_) : j0(lane * S), d(d_), pairs(pairs_) {
    const bool split = !INTER && j0 < pairs;
    off_u = split ? j0 : 2 * j0;
    off_v = split ? j0 + pairs : 2 * j0 + S;
    live = 2 * j0 < d;
  }
  __device__ __forceinline__ int at_a(int e) const { return (!INTER && j0 + e < pairs) ? j0 + e : 2 * (j0 + e); }
  __device__ __forceinline__ int at_b(int e) const { return (!INTER && j0 + e < pairs) ? j0 + e + pairs : 2 * (j0 + e) + 1; }
  __device__ __forceinline__ bool has(int e) const { return 2 * (j0 + e) < d; }
  // the element behind the lane's e-th value: the a, then the b.  A vector access leaves a pass-through lane's two runs as
  // they lie; nothing there depends on which of the two a value belongs to.
  __device__ __forceinline__ int at(int e) const {
    if constexpr (VEC && !INTER) return (e < S ? off_u : off_v) + e % S;
    return e < S ? at_a(e) : at_b(e - S);
  }

  typedef Raw<T, S, VEC> R;
  __device__ __forceinline__ void clear(R& r) const {      // what a lane without elements holds
    if constexpr (VEC && sizeof(T) * S == 8) {
      r.u = r.v = make_uint2(0, 0);
    } else if constexpr (VEC) {
      r.u = r.v = make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 2 * S; ++e) r.x[e] = 0.f;
    }
  }
  __device__ __forceinline__ void load(const T* row, R& r) const {
    if constexpr (VEC) {
      if (!live) return;
      r.u = *reinterpret_cast<const decltype(r.u)*>(row + off_u);
      r.v = *reinterpret_cast<const decltype(r.v)*>(row + off_v);
    } else {
#pragma unroll
      for (int e = 0; e < 2 * S; ++e)
        if (has(e % S)) r.x[e] = to_f(row[at(e)]);
    }
  }
  __device__ __forceinline__ Row<S> row(const R& r) const {
    Row<S> x;
    if constexpr (!VEC) {
#pragma unroll
      for (int e = 0; e < S / 2; ++e) { x.a[e] = pack(r.x[2 * e], r.x[2 * e + 1]); x.b[e] = pack(r.x[S + 2 * e], r.x[S + 2 * e + 1]); }
    } else {
      float u[S], v[S];
      if constexpr (sizeof(T) == 2) {
        const float2 p = halves(r.u.x), q = halves(r.u.y), w = halves(r.v.x), z = halves(r.v.y);
        u[0] = p.x; u[1] = p.y; u[2] = q.x; u[3] = q.y;
        v[0] = w.x; v[1] = w.y; v[2] = z.x; v[3] = z.y;
        if constexpr (S == 8) {
          const float2 p2 = halves(r.u.z), q2 = halves(r.u.w), w2 = halves(r.v.z), z2 = halves(r.v.w);
          u[4] = p2.x; u[5] = p2.y; u[6] = q2.x; u[7] = q2.y;
          v[4] = w2.x; v[5] = w2.y; v[6] = z2.x; v[7] = z2.y;
        }
      } else {
        u[0] = __uint_as_float(r.u.x); u[1] = __uint_as_float(r.u.y); u[2] = __uint_as_float(r.u.z); u[3] = __uint_as_float(r.u.w);
        v[0] = __uint_as_float(r.v.x); v[1] = __uint_as_float(r.v.y); v[2] = __uint_as_float(r.v.z); v[3] = __uint_as_float(r.v.w);
      }
#pragma unroll
      for (int e = 0; e < S / 2; ++e) {
        if constexpr (INTER) {                             // u, v in sequence: a0 b0 a1 b1 ...
          const float* w = 4 * e < S ? u + 4 * e : v + 4 * e - S;
          x.a[e] = pack(w[0], w[2]);
          x.b[e] = pack(w[1], w[3]);
        } else {
          x.a[e] = pack(u[2 * e], u[2 * e + 1]);
          x.b[e] = pack(v[2 * e], v[2 * e + 1]);
        }
      }
    }
    return x;
  }
  // the values in the runs' order (VEC); otherwise the a, then the b
  __device__ __forceinline__ void values(const Row<S>& x, float (&u)[S], float (&v)[S]) const {
#pragma unroll
    for (int e = 0; e < S / 2; ++e) {
      if constexpr (INTER && VEC) {
        float* w = 4 * e < S ? u + 4 * e : v + 4 * e - S;
        unpack(x.a[e], w[0], w[2]);
        unpack(x.b[e], w[1], w[3]);
      } else {
        unpack(x.a[e], u[2 * e], u[2 * e + 1]);
        unpack(x.b[e], v[2 * e], v[2 * e + 1]);
      }
    }
  }
  __device__ __forceinline__ void store(T* row, const Row<S>& x) const {
    float u[S], v[S];
    values(x, u, v);
    if constexpr (!VEC) {
#pragma unroll
      for (int e = 0; e < S; ++e)
        if (has(e)) { put(row + at(e), u[e]); put(row + at(S + e), v[e]); }
    } else if constexpr (sizeof(T) == 2) {
      if (!live) return;
      if constexpr (S == 8) {
        *reinterpret_cast<uint4*>(row + off_u) = make_uint4(half2_of(u[0], u[1]), half2_of(u[2], u[3]), half2_of(u[4], u[5]), half2_of(u[6], u[7]));
        *reinterpret_cast<uint4*>(row + off_v) = make_uint4(half2_of(v[0], v[1]), half2_of(v[2], v[3]), half2_of(v[4], v[5]), half2_of(v[6], v[7]));
      } else {
        *reinterpret_cast<uint2*>(row + off_u) = make_uint2(half2_of(u[0], u[1]), half2_of(u[2], u[3]));
        *reinterpret_cast<uint2*>(row + off_v) = make_uint2(half2_of(v[0], v[1]), half2_of(v[2], v[3]));
      }
    } else {
      if (!live) return;
      *reinterpret_cast<float4*>(row + off_u) = make_float4(u[0], u[1], u[2], u[3]);
      *reinterpret_cast<float4*>(row + off_v) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  __device__ __forceinline__ Row<S> gain(const void* p) const {
    const T* g = reinterpret_cast<const T*>(p);
    float x[2 * S];
#pragma unroll
    for (int e = 0; e < 2 * S; ++e) x[e] = g && has(e % S) ? to_f(g[at(e)]) : 1.f;
    Row<S> r;
#pragma unroll
    for (int e = 0; e < S / 2; ++e) { r.a[e] = pack(x[2 * e], x[2 * e + 1]); r.b[e] = pack(x[S + 2 * e], x[S + 2 * e + 1]); }
    return r;
  }
};

// cos and sin of a lane's slots at a token's positions; 1 and 0 where nothing rotates.
template <int S> struct Angle {
  f2 c[S / 2], s[S / 2];
};
struct Place { int p0, p1, p2; };
// cos and sin of pair j at a place, from the pair's turns per position (a sum of two).
struct Turns { double hi, lo; };
__device__ __forceinline__ Turns turns_of(const Transform& t, int j) {
  constexpr double INV = 0.15915494309189535, INV_REST = -9.839338337591243e-18;   // 1 / 2 pi
  const double f = __ldg(t.freq + j), hi = f * INV;
  return {hi, fma(f, INV_REST, fma(f, INV, -hi))};
}
__device__ __forceinline__ float2 cos_sin(const Transform& t, int j, const Turns& per_pos, const Place& p) {
  const double n = (double)(j < t.end0 ? p.p0 : j < t.end1 ? p.p1 : p.p2);
  constexpr double WHOLE = 6755399441055744.0;             // 1.5 * 2^52: what is added to it is rounded to a whole number
  const double turns = fma(n, per_pos.hi, WHOLE) - WHOLE;
  const double x = fma(n, per_pos.lo, fma(n, per_pos.hi, -turns));
  const float near = (float)x, rest = 6.2831853f * (float)(x - (double)near);
  float s, c;
  sincospif(2.f * near, &s, &c);
  return make_float2(fmaf(-s, rest, c), fmaf(c, rest, s));
}
// Fills table[i * pairs + j] with cos and sin of pair j at place_at(i) for i < n: a thread keeps to one pair.
template <int NT, typename At>
__device__ __forceinline__ void fill_table(const Transform& t, float2* table, int n, At place_at) {
  if (t.pairs == 0) return;
  const int lead = t.pairs < NT ? t.pairs : NT;            // pairs at a time; the threads beyond take further places
  const int j0 = threadIdx.x % lead, i0 = threadIdx.x / lead, stride = NT / lead;
  if (i0 >= stride) return;
  for (int j = j0; j < t.pairs; j += lead) {
    const Turns per_pos = turns_of(t, j);
    for (int i = i0; i < n; i += stride) table[i * t.pairs + j] = cos_sin(t, j, per_pos, place_at(i));
  }
}
// A lane's from a table of all pairs of one place.
template <int S>
__device__ __forceinline__ Angle<S> angle_from(const float2* table, int j0, int pairs) {
  Angle<S> r;
#pragma unroll
  for (int i = 0; i < S / 2; ++i) {
    const int j = j0 + 2 * i;
    const float2 x = j < pairs ? table[j] : make_float2(1.f, 0.f), y = j + 1 < pairs ? table[j + 1] : make_float2(1.f, 0.f);
    r.c[i] = pack(x.x, y.x);
    r.s[i] = pack(x.y, y.y);
  }
  return r;
}

// Keeps the slots that do not rotate as `plain` has them: slots of a lane that does not rotate as a whole (no VEC).  They
// are left alone rather than turned by 0, since an infinity among them would make its neighbour NaN.
__device__ __forceinline__ f2 kept(f2 turned, f2 plain, int j, int pairs) {
  float t[2], p[2];
  unpack(turned, t[0], t[1]);
  unpack(plain, p[0], p[1]);
  return pack(j < pairs ? t[0] : p[0], j + 1 < pairs ? t[1] : p[1]);
}

template <int S, bool VEC>
__device__ __forceinline__ Row<S> turned(const Row<S>& x, const Angle<S>& t, int j0, int pairs) {
  if (VEC && j0 >= pairs) return x;
  Row<S> y;
#pragma unroll
  for (int e = 0; e < S / 2; ++e) {
    y.a[e] = fma2(x.b[e], neg2(t.s[e]), mul2(x.a[e], t.c[e]));
    y.b[e] = fma2(x.a[e], t.s[e], mul2(x.b[e], t.c[e]));
    if constexpr (!VEC) {
      y.a[e] = kept(y.a[e], x.a[e], j0 + 2 * e, pairs);
      y.b[e] = kept(y.b[e], x.b[e], j0 + 2 * e, pairs);
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
  for (int o = LPR / 2; o > 0; o >>= 1) z = add2(z, f2{__shfl_xor_sync(0xffffffffu, z.x, o), __shfl_xor_sync(0xffffffffu, z.y, o)});
  unpack(z, x, y);
}
__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

// gain * x / sqrt(mean(x^2) + eps), then the turn: the whole forward transform of a row.  The gain is folded into the
// angle, which serves all heads of a token: what is left is one scale by the reciprocal root.
template <int S> struct Coef {
  f2 ac[S / 2], bs[S / 2], bc[S / 2], as[S / 2];           // gain_a cos, -gain_b sin, gain_b cos, gain_a sin
};
template <int S>
__device__ __forceinline__ Coef<S> coef(const Angle<S>& t, const Row<S>& gain) {
  Coef<S> k;
#pragma unroll
  for (int e = 0; e < S / 2; ++e) {
    k.ac[e] = mul2(gain.a[e], t.c[e]);
    k.as[e] = mul2(gain.a[e], t.s[e]);
    k.bc[e] = mul2(gain.b[e], t.c[e]);
    k.bs[e] = neg2(mul2(gain.b[e], t.s[e]));
  }
  return k;
}
template <int S, int LPR, bool VEC>
__device__ __forceinline__ Row<S> transformed(const Row<S>& x, const Coef<S>& k, const Transform& t, int j0, float inv_d) {
  Row<S> y;
  f2 rs = {0.f, 0.f};
  if (t.normalize) {
    const float r = rsqrtf(group_sum<LPR>(dot(x, x)) * inv_d + t.eps);
    rs = pack(r, r);
  }
#pragma unroll
  for (int e = 0; e < S / 2; ++e) {
    y.a[e] = mul2(x.a[e], k.ac[e]);                        // slots that do not rotate: cos is 1, this is all
    y.b[e] = mul2(x.b[e], k.bc[e]);
    if (!VEC || j0 < t.pairs) {
      const f2 ta = fma2(x.b[e], k.bs[e], y.a[e]), tb = fma2(x.a[e], k.as[e], y.b[e]);
      y.a[e] = VEC ? ta : kept(ta, y.a[e], j0 + 2 * e, t.pairs);
      y.b[e] = VEC ? tb : kept(tb, y.b[e], j0 + 2 * e, t.pairs);
    }
    if (t.normalize) { y.a[e] = mul2(y.a[e], rs); y.b[e] = mul2(y.b[e], rs); }
  }
  return y;
}

// Positions of a token on the axes: pos is axes x n, or null for the one index on every axis.
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

// Whether the rows of an operand can be moved n elements at a time.
inline bool vec_ok(int n, int64_t es, const void* p, int64_t s0, int64_t s1, int64_t s2) {
  return ((uintptr_t)p % (n * es)) == 0 && s0 % n == 0 && s1 % n == 0 && s2 % n == 0;
}
// Lanes that share a row.
inline int lanes_per_row(int64_t d, int slots) {
  int n = 4;
  while (n * 2 * slots < d) n *= 2;
  return n;
}

// How many of a CTA's groups of lanes share a token, a power of two: fewer compute the sines and addresses for more heads,
// more leave the last CTAs less uneven and a small batch not idle.  A CTA costs a group's rows, taken `ahead` at a time,
// and what it does once a token, measured at about four rows.  CTAs that stay and loop (`looping`) all take the most
// rounds that one of them has; others follow one another, and half a CTA's time goes by at the end.
inline int groups_per_token(int64_t tokens, int rows, int groups, int64_t resident, int ahead, bool looping) {
  int best = 1;
  int64_t least = 0;
  for (int p = 1; p <= groups; p *= 2) {
    const int64_t ctas = (tokens + groups / p - 1) / (groups / p);
    const int64_t each = 4 + (rows + p * ahead - 1) / (p * ahead) * ahead;
    const int64_t cost = (looping || ctas <= resident ? (ctas + resident - 1) / resident * resident : ctas + resident / 2) * each;
    if (p == 1 || cost < least) {
      best = p;
      least = cost;
    }
  }
  return best;
}

}  // namespace heads
}  // namespace b200
