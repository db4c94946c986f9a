// Norm of every query and key head with the position rotation in the same pass, forward and backward
// (head_transform.cuh has the formulas).  Both are bound by HBM: forward reads and writes each element once, backward
// reads x and the upstream gradient once and writes the gradient once; the norm's statistics are recomputed from the
// row that the backward holds anyway, so nothing is saved between the two.
//
//   qk_forward_kernel   a group of LPR lanes owns a token and walks its heads (queries, then keys) `per_token` groups
//                       apart: the angles' sines are computed once per token and group and serve all its heads.
//   qk_backward_kernel  the same walk.  With h' = R^T g the gradient before the rotation,
//                         dgain += h' * xhat,   dx = r (h' gain - xhat mean(h' gain xhat)),   xhat = x r.
//                       The gains' sums stay in f32 registers over all rows of a lane, are added up per CTA in a fixed
//                       order and leave as one row of partial sums per CTA.
//   gain_sum_kernel     adds the CTAs' rows in a fixed order: no atomics, the same bits in every run.
#include "head_transform.cuh"

namespace b200 {

namespace {

using namespace heads;

struct QkArgs {
  Transform t;
  long long tokens;                // batch * tokens
  int seq, q_heads, rows;          // rows = q_heads + k_heads of one token
  int d, axes, per_token;          // groups that share a token
  const int* pos;                  // axes x tokens, or nullptr: the index in the sequence on every axis
  const void *q, *k, *gq, *gk;     // inputs; upstream gradients (backward)
  void *q_out, *k_out;             // outputs; gradients (backward)
  long long qb, qt, qh, kb, kt, kh;          // element strides of the batch, token and head axes
  long long gqb, gqt, gqh, gkb, gkt, gkh;
  long long qob, qot, qoh, kob, kot, koh;
  const void *q_gain, *k_gain;
  float* partial;                  // backward: gridDim.x rows of 2 * d sums, or nullptr
};

constexpr int THREADS = 256;

template <typename T, int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(THREADS, 3) qk_forward_kernel(const QkArgs g) {
  constexpr int GROUPS = THREADS / LPR, U = !VEC ? 1 : sizeof(T) == 2 ? 4 : 2;   // rows on their way per group
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const Lane<INTER, VEC> ln(lane, g.d, g.t.pairs);
  const int per_cta = GROUPS / g.per_token, part = group % g.per_token;
  const float inv_d = 1.f / (float)g.d;
  const long long tok = (long long)blockIdx.x * per_cta + group / g.per_token;
  const bool on = tok < g.tokens && ln.live;
  const int tc = tok < g.tokens ? (int)tok : 0;
  const int ib = tc / g.seq, is = tc % g.seq;
  const Place at = place_of(g.pos, g.axes, g.tokens, tc, is);
  Angle angle;
#pragma unroll
  for (int w = 0; w < 2; ++w) {                            // queries, then keys; the next group begins where the last ended
    const T* src = w == 0 ? reinterpret_cast<const T*>(g.q) + ib * g.qb + is * g.qt : reinterpret_cast<const T*>(g.k) + ib * g.kb + is * g.kt;
    T* dst = w == 0 ? reinterpret_cast<T*>(g.q_out) + ib * g.qob + is * g.qot : reinterpret_cast<T*>(g.k_out) + ib * g.kob + is * g.kot;
    const long long sh = w == 0 ? g.qh : g.kh, dh = w == 0 ? g.qoh : g.koh;
    const int heads = w == 0 ? g.q_heads : g.rows - g.q_heads;
    const int first = w == 0 ? part : (part - g.q_heads) & (g.per_token - 1);
    Coef k;
    for (int r0 = 0; r0 < heads; r0 += U * g.per_token) {  // the same trip count in every group
      Raw<T, VEC> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * g.per_token + first;
        ln.clear(raw[u]);
        if (on && r < heads) ln.load(src + r * sh, raw[u]);
      }
      if (r0 == 0) {                                       // under the first loads
        if (w == 0 || g.q_heads == 0) angle = angle_at(g.t, ln.j0, at.p0, at.p1, at.p2);
        k = coef(angle, ln.gain(reinterpret_cast<const T*>(w == 0 ? g.q_gain : g.k_gain)));
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * g.per_token + first;
        const Row y = transformed<LPR, VEC>(ln.row(raw[u]), k, g.t, ln.j0, inv_d);
        if (on && r < heads) ln.store(dst + r * dh, y);
      }
    }
  }
}

template <typename T, int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) qk_backward_kernel(const QkArgs g) {
  constexpr int GROUPS = THREADS / LPR, U = VEC ? 2 : 1;
  __shared__ float sums[THREADS * 8];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const Lane<INTER, VEC> ln(lane, g.d, g.t.pairs);
  const int per_cta = GROUPS / g.per_token, part = group % g.per_token;
  const float inv_d = 1.f / (float)g.d;
  const Row zero = {{0, 0}, {0, 0}};
  Row acc[2] = {zero, zero};                               // the gains' gradients: queries, keys
  for (long long t0 = (long long)blockIdx.x * per_cta; t0 < g.tokens; t0 += (long long)gridDim.x * per_cta) {
    const long long tok = t0 + group / g.per_token;
    const bool on = tok < g.tokens && ln.live;
    const int tc = tok < g.tokens ? (int)tok : 0;
    const int ib = tc / g.seq, is = tc % g.seq;
    const Place at = place_of(g.pos, g.axes, g.tokens, tc, is);
    Angle angle;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const T* src = w == 0 ? reinterpret_cast<const T*>(g.q) + ib * g.qb + is * g.qt : reinterpret_cast<const T*>(g.k) + ib * g.kb + is * g.kt;
      const T* up = w == 0 ? reinterpret_cast<const T*>(g.gq) + ib * g.gqb + is * g.gqt : reinterpret_cast<const T*>(g.gk) + ib * g.gkb + is * g.gkt;
      T* dst = w == 0 ? reinterpret_cast<T*>(g.q_out) + ib * g.qob + is * g.qot : reinterpret_cast<T*>(g.k_out) + ib * g.kob + is * g.kot;
      const long long sh = w == 0 ? g.qh : g.kh, uh = w == 0 ? g.gqh : g.gkh, dh = w == 0 ? g.qoh : g.koh;
      const int heads = w == 0 ? g.q_heads : g.rows - g.q_heads;
      const int first = w == 0 ? part : (part - g.q_heads) & (g.per_token - 1);
      Row gain;
      for (int r0 = 0; r0 < heads; r0 += U * g.per_token) {
        Raw<T, VEC> rx[U], rg[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * g.per_token + first;
          ln.clear(rx[u]);
          ln.clear(rg[u]);
          if (on && r < heads) {
            if (g.t.normalize) ln.load(src + r * sh, rx[u]);
            ln.load(up + r * uh, rg[u]);
          }
        }
        if (r0 == 0) {
          if (w == 0 || g.q_heads == 0) {
            angle = angle_at(g.t, ln.j0, at.p0, at.p1, at.p2);
#pragma unroll
            for (int e = 0; e < 2; ++e) angle.s[e] = neg2(angle.s[e]);       // the gradient turns back
          }
          if (g.t.normalize) gain = ln.gain(reinterpret_cast<const T*>(w == 0 ? g.q_gain : g.k_gain));
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * g.per_token + first;
          Row h = turned<VEC>(ln.row(rg[u]), angle.c, angle.s, ln.j0, g.t.pairs);
          if (g.t.normalize) {
            // both sums before the reciprocal root is known:  sum x^2  and  sum h gain x
            const Row x = ln.row(rx[u]), hx = times(h, x);
            float sq, hg;
            group_sum_pair<LPR>(dot(x, x), dot(hx, gain), sq, hg);
            const float rs = rsqrtf(sq * inv_d + g.t.eps);
            const f2 rs2 = both(rs), back = both(-(hg * inv_d) * rs * rs * rs);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              acc[w].a[e] = fma2(hx.a[e], rs2, acc[w].a[e]);
              acc[w].b[e] = fma2(hx.b[e], rs2, acc[w].b[e]);
              h.a[e] = fma2(h.a[e], mul2(gain.a[e], rs2), mul2(x.a[e], back));
              h.b[e] = fma2(h.b[e], mul2(gain.b[e], rs2), mul2(x.b[e], back));
            }
          }
          if (on && r < heads) ln.store(dst + r * dh, h);
        }
      }
    }
  }
  if (!g.partial) return;
  float* out = g.partial + (long long)blockIdx.x * 2 * g.d;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float x[8];
    unpack(acc[w].a[0], x[0], x[1]); unpack(acc[w].a[1], x[2], x[3]);
    unpack(acc[w].b[0], x[4], x[5]); unpack(acc[w].b[1], x[6], x[7]);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[(group * 8 + e) * LPR + lane] = x[e];
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * LPR; i += THREADS) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) sum += sums[j * 8 * LPR + i];
      const int e = i / LPR;
      // INTER: a Row's values are a0..a3, b0..b3 whatever the runs' order
      const Lane<INTER, VEC> who(i % LPR, g.d, g.t.pairs);
      if (who.has(e & 3)) out[w * g.d + who.at(e)] = sum;
    }
  }
}

// out[w][j] (+)= sum over the CTAs' rows, 8 rows at a time and their sums in order.
__global__ void __launch_bounds__(256) gain_sum_kernel(const float* __restrict__ partial, int parts, int d,
                                                       float* __restrict__ gq, float* __restrict__ gk, int accumulate) {
  __shared__ float sh[8][33];
  const int j = blockIdx.x * 32 + (threadIdx.x & 31), y = threadIdx.x >> 5;
  float x = 0.f;
  if (j < 2 * d)
    for (int p = y; p < parts; p += 8) x += partial[(long long)p * 2 * d + j];
  sh[y][threadIdx.x & 31] = x;
  __syncthreads();
  if (y || j >= 2 * d) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) x += sh[i][threadIdx.x];
  float* out = j < d ? gq : gk;
  if (!out) return;
  out += j < d ? j : j - d;
  *out = accumulate ? *out + x : x;
}

constexpr int MAX_PARTS = 1024;

bool vec_ok(int64_t es, const void* p, int64_t b, int64_t t, int64_t h) {
  return ((uintptr_t)p % (4 * es)) == 0 && b % 4 == 0 && t % 4 == 0 && h % 4 == 0;
}

template <typename T, int LPR, bool INTER, bool VEC>
int launch_one(const QkArgs& g, bool backward, unsigned grid, cudaStream_t stream) {
  if (backward) qk_backward_kernel<T, LPR, INTER, VEC><<<grid, THREADS, 0, stream>>>(g);
  else qk_forward_kernel<T, LPR, INTER, VEC><<<grid, THREADS, 0, stream>>>(g);
  count_launch(false);
  return note_cuda_error(cudaGetLastError(), "query/key norm and rotation launch");
}
template <typename T, int LPR>
int launch_lpr(const QkArgs& g, bool inter, bool vec, bool backward, unsigned grid, cudaStream_t stream) {
  if (inter) return vec ? launch_one<T, LPR, true, true>(g, backward, grid, stream) : launch_one<T, LPR, true, false>(g, backward, grid, stream);
  return vec ? launch_one<T, LPR, false, true>(g, backward, grid, stream) : launch_one<T, LPR, false, false>(g, backward, grid, stream);
}
template <typename T>
int launch_type(const QkArgs& g, bool inter, bool vec, bool backward, unsigned grid, cudaStream_t stream) {
  switch (lanes_per_row(g.d)) {
    case 8: return launch_lpr<T, 8>(g, inter, vec, backward, grid, stream);
    case 16: return launch_lpr<T, 16>(g, inter, vec, backward, grid, stream);
    default: return launch_lpr<T, 32>(g, inter, vec, backward, grid, stream);
  }
}

}  // namespace

size_t qk_norm_rotary_backward_workspace_bytes(int64_t d) { return (size_t)MAX_PARTS * 2 * (size_t)d * sizeof(float); }

// Strides are [batch, token, head] of q, k, the upstream gradients (backward) and the outputs.
int qk_norm_rotary(int dtype, const b200_head_op* op, int64_t batch, int64_t seq, int64_t q_heads, int64_t k_heads, int64_t d,
                   const void* const in[4], const int64_t in_strides[4][3], const int32_t* positions, void* const out[2],
                   const int64_t out_strides[2][3], bool backward, float* q_gain_grad, float* k_gain_grad, int accumulate,
                   void* workspace, cudaStream_t stream) {
  QkArgs g;
  const int rc = parse(op, (size_t)d, &g.t, &g.axes);
  if (rc) return rc;
  const DeviceState* ds = device_state();
  if (!ds) return note_cuda_error(cudaErrorInitializationError, "b200_init not called on this device");
  const int64_t es = dtype == B200_F32 ? 4 : 2;
  g.tokens = batch * seq;
  g.seq = (int)seq; g.q_heads = (int)q_heads; g.rows = (int)(q_heads + k_heads); g.d = (int)d;
  g.pos = positions;
  g.q = in[0]; g.k = in[1]; g.gq = in[2]; g.gk = in[3];
  g.q_out = out[0]; g.k_out = out[1];
  g.qb = in_strides[0][0]; g.qt = in_strides[0][1]; g.qh = in_strides[0][2];
  g.kb = in_strides[1][0]; g.kt = in_strides[1][1]; g.kh = in_strides[1][2];
  g.gqb = in_strides[2][0]; g.gqt = in_strides[2][1]; g.gqh = in_strides[2][2];
  g.gkb = in_strides[3][0]; g.gkt = in_strides[3][1]; g.gkh = in_strides[3][2];
  g.qob = out_strides[0][0]; g.qot = out_strides[0][1]; g.qoh = out_strides[0][2];
  g.kob = out_strides[1][0]; g.kot = out_strides[1][1]; g.koh = out_strides[1][2];
  g.q_gain = op->q_gain; g.k_gain = op->k_gain;
  const bool inter = op->interleaved != 0;
  bool vec = d % 8 == 0 && g.t.pairs % 4 == 0;
  for (int i = 0; i < (backward ? 4 : 2); ++i) vec = vec && vec_ok(es, in[i], in_strides[i][0], in_strides[i][1], in_strides[i][2]);
  for (int i = 0; i < 2; ++i) vec = vec && vec_ok(es, out[i], out_strides[i][0], out_strides[i][1], out_strides[i][2]);
  // Groups that share a token: as few as still give every SM's 2048 threads a group (the sines are then computed for
  // the most heads), and no more than the token has rows.
  const int lpr = lanes_per_row(d), groups = THREADS / lpr;
  const int64_t want = (int64_t)ds->sm_count * (2048 / lpr);
  g.per_token = 1;
  while (g.per_token < groups && g.per_token < g.rows && g.tokens * g.per_token < want) g.per_token *= 2;
  const int64_t per_cta = groups / g.per_token;
  int64_t grid = (g.tokens + per_cta - 1) / per_cta;
  const bool sums = backward && g.t.normalize && (q_gain_grad || k_gain_grad);
  g.partial = sums ? (float*)workspace : nullptr;
  if (backward && grid > (int64_t)ds->sm_count * 4) grid = (int64_t)ds->sm_count * 4;
  if (backward && grid > MAX_PARTS) grid = MAX_PARTS;
  if (grid > 0x7fffffff) grid = 0x7fffffff;
  if (g.rows == 0) grid = 0;
  int rc2 = grid == 0 ? B200_OK : dtype == B200_F32 ? launch_type<float>(g, inter, vec, backward, (unsigned)grid, stream)
                              : launch_type<__half>(g, inter, vec, backward, (unsigned)grid, stream);   // an empty batch: sums over nothing follow
  if (rc2 || !sums) return rc2;
  gain_sum_kernel<<<(unsigned)((2 * d + 31) / 32), 256, 0, stream>>>(g.partial, (int)grid, (int)d, q_gain_grad, k_gain_grad, accumulate);
  count_launch(false);
  return note_cuda_error(cudaGetLastError(), "gain gradient launch");
}

}  // namespace b200
