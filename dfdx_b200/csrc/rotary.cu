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

struct Side {                      // queries or keys
  const void *x, *up;              // input; upstream gradient (backward)
  void* y;                         // output; gradient (backward)
  const void* gain;
  int heads, per_token;            // per_token: groups that share a token
  int xh, uh, yh;                  // element strides of the head, batch and token axes
  long long xb, xt, ub, ut, yb, yt;
};
struct QkArgs {
  Transform t;
  Side side[2];
  unsigned q_ctas;                 // the CTAs behind them have keys
  int tokens, seq;                 // batch * tokens of a sequence
  int d, axes;
  const int* pos;                  // axes x tokens, or nullptr: the index in the sequence on every axis
  float* partial;                  // backward: a row of d sums per CTA, or nullptr
};

constexpr int THREADS = 128;

__device__ __forceinline__ Place place_at(const QkArgs& g, int tok) { return place_of(g.pos, g.axes, g.tokens, tok, tok % g.seq); }

// cos and sin of all pairs at the CTA's tokens t0 .. t0 + n - 1, each computed once for all its heads.
__device__ __forceinline__ void fill_table(const QkArgs& g, float2* table, int t0, int n) {
  const int pairs = g.t.pairs;
  for (int i = threadIdx.x; i < n * pairs; i += THREADS) {
    const int tok = t0 + i / pairs;
    if (tok < g.tokens) table[i] = cos_sin(g.t, i % pairs, place_at(g, tok));
  }
}

template <typename T, int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 && VEC ? 7 : 5) qk_forward_kernel(const __grid_constant__ QkArgs g) {
  constexpr int GROUPS = THREADS / LPR, U = !VEC ? 1 : sizeof(T) == 2 ? 4 : 2;   // rows on their way per group
  __shared__ float2 table[GROUPS * LPR * S];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const bool keys = blockIdx.x >= g.q_ctas;
  const Side& sd = g.side[keys];
  const Lane<T, INTER, VEC> ln(lane, g.d, g.t.pairs);
  const int per_cta = GROUPS / sd.per_token, first = group % sd.per_token, mine = group / sd.per_token;
  const int t0 = (int)(blockIdx.x - (keys ? g.q_ctas : 0)) * per_cta, tok = t0 + mine;
  const bool on = tok < g.tokens;
  const int tc = min(tok, g.tokens - 1), ib = tc / g.seq, is = tc % g.seq;   // a group without a token works on the last one
  const T* src = reinterpret_cast<const T*>(sd.x) + ib * sd.xb + is * sd.xt;
  T* dst = reinterpret_cast<T*>(sd.y) + ib * sd.yb + is * sd.yt;
  const float inv_d = 1.f / (float)g.d;
  const int step = sd.per_token, heads = sd.heads;
  Raw<T, VEC> raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    ln.clear(raw[u]);
    ln.load(src + (long long)min(u * step + first, heads - 1) * sd.xh, raw[u]);
  }
  fill_table(g, table, t0, per_cta);                       // under the first loads
  const Row gain = ln.gain(sd.gain);
  __syncthreads();
  const Coef k = coef(angle_from(table + mine * g.t.pairs, ln.j0, on ? g.t.pairs : 0), gain);
  for (int r0 = 0;;) {                                     // the same trip count in every group
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * step + first;
      const Row y = transformed<LPR, VEC>(ln.row(raw[u]), k, g.t, ln.j0, inv_d);
      if (on && r < heads) ln.store(dst + (long long)r * sd.yh, y);
    }
    r0 += U * step;
    if (r0 >= heads) break;
#pragma unroll
    for (int u = 0; u < U; ++u) ln.load(src + (long long)min(r0 + u * step + first, heads - 1) * sd.xh, raw[u]);
  }
}

template <typename T, int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 && VEC ? 5 : 4) qk_backward_kernel(const __grid_constant__ QkArgs g) {
  constexpr int GROUPS = THREADS / LPR, U = VEC ? 2 : 1;
  __shared__ float2 table[GROUPS * LPR * S];
  __shared__ float sums[THREADS * 2 * S];
  asm volatile("griddepcontrol.launch_dependents;");       // the sum of the partial rows may be brought in; it waits for this
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const bool keys = blockIdx.x >= g.q_ctas;
  const Side& sd = g.side[keys];
  const Lane<T, INTER, VEC> ln(lane, g.d, g.t.pairs);
  const int per_cta = GROUPS / sd.per_token, first = group % sd.per_token, mine = group / sd.per_token;
  const int step = sd.per_token, heads = sd.heads, pairs = g.t.pairs;
  const int cta = (int)(blockIdx.x - (keys ? g.q_ctas : 0)), ctas = (int)(keys ? gridDim.x - g.q_ctas : g.q_ctas);
  const float inv_d = 1.f / (float)g.d;
  Row acc, gain;                                           // the gain's gradient; the gain
#pragma unroll
  for (int e = 0; e < S / 2; ++e) acc.a[e] = acc.b[e] = 0;
  if (g.t.normalize) gain = ln.gain(sd.gain);
  Raw<T, VEC> rx[U], rg[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    ln.clear(rx[u]);
    ln.clear(rg[u]);
  }
  for (int t0 = cta * per_cta; t0 < g.tokens; t0 += ctas * per_cta) {
    const int tok = t0 + mine;
    const bool on = tok < g.tokens;
    const int tc = min(tok, g.tokens - 1), ib = tc / g.seq, is = tc % g.seq;
    const T* src = reinterpret_cast<const T*>(sd.x) + ib * sd.xb + is * sd.xt;
    const T* up = reinterpret_cast<const T*>(sd.up) + ib * sd.ub + is * sd.ut;
    T* dst = reinterpret_cast<T*>(sd.y) + ib * sd.yb + is * sd.yt;
    auto load = [&](int r0) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = min(r0 + u * step + first, heads - 1);
        if (g.t.normalize) ln.load(src + (long long)r * sd.xh, rx[u]);
        ln.load(up + (long long)r * sd.uh, rg[u]);
      }
    };
    load(0);
    __syncthreads();                                       // the table's last readers are done
    fill_table(g, table, t0, per_cta);
    __syncthreads();
    Angle angle = angle_from(table + mine * pairs, ln.j0, on ? pairs : 0);
#pragma unroll
    for (int e = 0; e < S / 2; ++e) angle.s[e] = neg2(angle.s[e]);           // the gradient turns back
    for (int r0 = 0;;) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * step + first;
        const bool live = on && r < heads;
        Row h = turned<VEC>(ln.row(rg[u]), angle, ln.j0, pairs);
        if (g.t.normalize) {
          // both sums before the reciprocal root is known:  sum x^2  and  sum h gain x
          const Row x = ln.row(rx[u]), hx = times(h, x);
          float sq, hg;
          group_sum_pair<LPR>(dot(x, x), dot(hx, gain), sq, hg);
          const float rs = rsqrtf(sq * inv_d + g.t.eps), b = -(hg * inv_d) * rs * rs * rs;
          const f2 rs2 = pack(rs, rs), back = pack(b, b);
#pragma unroll
          for (int e = 0; e < S / 2; ++e) {
            if (live) {
              acc.a[e] = fma2(hx.a[e], rs2, acc.a[e]);
              acc.b[e] = fma2(hx.b[e], rs2, acc.b[e]);
            }
            h.a[e] = fma2(h.a[e], mul2(gain.a[e], rs2), mul2(x.a[e], back));
            h.b[e] = fma2(h.b[e], mul2(gain.b[e], rs2), mul2(x.b[e], back));
          }
        }
        if (live) ln.store(dst + (long long)r * sd.yh, h);
      }
      r0 += U * step;
      if (r0 >= heads) break;
      load(r0);
    }
  }
  if (!g.partial) return;
  float* out = g.partial + (long long)blockIdx.x * g.d;
#pragma unroll
  for (int e = 0; e < S / 2; ++e) {
    float x, y;
    unpack(acc.a[e], x, y);
    sums[(group * 2 * S + 2 * e) * LPR + lane] = x;
    sums[(group * 2 * S + 2 * e + 1) * LPR + lane] = y;
    unpack(acc.b[e], x, y);
    sums[(group * 2 * S + S + 2 * e) * LPR + lane] = x;
    sums[(group * 2 * S + S + 2 * e + 1) * LPR + lane] = y;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * S * LPR; i += THREADS) {
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < GROUPS; ++j) sum += sums[j * 2 * S * LPR + i];
    const Lane<T, INTER, VEC> who(i % LPR, g.d, g.t.pairs);
    if (who.has(i / LPR % S)) out[who.at(i / LPR)] = sum;
  }
}

// Adds the CTAs' rows: each of 32 warps every 32nd of the queries' (or keys') rows, then the warps in order.
__global__ void __launch_bounds__(1024) gain_sum_kernel(const float* __restrict__ partial, int q_parts, int k_parts, int d,
                                                        float* __restrict__ gq, float* __restrict__ gk, int accumulate) {
  __shared__ float sh[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");       // the rows are complete and visible
  const bool keys = blockIdx.y;
  const int lane = threadIdx.x & 31, j = blockIdx.x * 32 + lane, y = threadIdx.x >> 5;
  const int parts = keys ? k_parts : q_parts;
  if (keys) partial += (long long)q_parts * d;
  float x = 0.f;
  if (j < d) {
#pragma unroll 8
    for (int p = y; p < parts; p += 32) x += partial[(long long)p * d + j];
  }
  sh[y][lane] = x;
  __syncthreads();
  float* out = keys ? gk : gq;
  if (y || j >= d || !out) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) x += sh[i][lane];
  out[j] = accumulate ? out[j] + x : x;
}

constexpr int MAX_PARTS = 2048;

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
    case 4: return launch_lpr<T, 4>(g, inter, vec, backward, grid, stream);
    case 8: return launch_lpr<T, 8>(g, inter, vec, backward, grid, stream);
    case 16: return launch_lpr<T, 16>(g, inter, vec, backward, grid, stream);
    default: return launch_lpr<T, 32>(g, inter, vec, backward, grid, stream);
  }
}

}  // namespace

size_t qk_norm_rotary_backward_workspace_bytes(int64_t d) { return (size_t)MAX_PARTS * (size_t)d * sizeof(float); }

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
  g.tokens = (int)(batch * seq);
  g.seq = (int)seq; g.d = (int)d;
  g.pos = positions;
  const bool inter = op->interleaved != 0;
  bool vec = d % 8 == 0 && g.t.pairs % 4 == 0;
  const int lpr = lanes_per_row(d), groups = THREADS / lpr;
  const int64_t want = (int64_t)ds->sm_count * (2048 / lpr);                 // groups that fill every SM
  int64_t ctas[2] = {0, 0}, work = 0;
  for (int w = 0; w < 2; ++w) {
    Side& sd = g.side[w];
    sd.x = in[w]; sd.up = in[2 + w]; sd.y = out[w];
    sd.gain = w == 0 ? op->q_gain : op->k_gain;
    sd.heads = (int)(w == 0 ? q_heads : k_heads);
    const int64_t *xs = in_strides[w], *us = in_strides[2 + w], *ys = out_strides[w];
    if (xs[2] > 0x7fffffff || us[2] > 0x7fffffff || ys[2] > 0x7fffffff) return B200_ERR_LIMIT;
    sd.xb = xs[0]; sd.xt = xs[1]; sd.xh = (int)xs[2];
    sd.ub = us[0]; sd.ut = us[1]; sd.uh = (int)us[2];
    sd.yb = ys[0]; sd.yt = ys[1]; sd.yh = (int)ys[2];
    sd.per_token = 1;
    if (sd.heads == 0 || g.tokens == 0) continue;
    vec = vec && vec_ok(es, sd.x, sd.xb, sd.xt, sd.xh) && vec_ok(es, sd.y, sd.yb, sd.yt, sd.yh);
    if (backward) vec = vec && vec_ok(es, sd.up, sd.ub, sd.ut, sd.uh);
    // Groups that share a token: at most eight heads each, so that CTAs are short and end together, and more while the
    // groups of all tokens would leave SMs without work.
    while (sd.per_token < groups && sd.per_token < sd.heads && (sd.heads > 8 * sd.per_token || (int64_t)g.tokens * sd.per_token < want))
      sd.per_token *= 2;
    ctas[w] = (g.tokens + groups / sd.per_token - 1) / (groups / sd.per_token);
    work += ctas[w];
  }
  // Backward: what is resident at once, shared out by the work; each CTA's sums are a row to add up at the end.
  const int64_t resident = (int64_t)ds->sm_count * (es == 2 && vec ? 5 : 4), most = resident < MAX_PARTS ? resident : MAX_PARTS;
  if (backward && work > most) {
    const int64_t share = ctas[0] * most / work;
    ctas[0] = ctas[0] ? (share > 0 ? share : 1) : 0;
    ctas[1] = ctas[1] ? (most - ctas[0] > 0 ? most - ctas[0] : 1) : 0;
  }
  const bool sums = backward && g.t.normalize && (q_gain_grad || k_gain_grad);
  g.partial = sums ? (float*)workspace : nullptr;
  g.q_ctas = (unsigned)ctas[0];
  const int64_t grid = ctas[0] + ctas[1];
  if (grid > 0x7fffffff) return B200_ERR_LIMIT;
  if (grid) {                                              // an empty batch: sums over nothing follow
    const int rc2 = dtype == B200_F32 ? launch_type<float>(g, inter, vec, backward, (unsigned)grid, stream)
                                      : launch_type<__half>(g, inter, vec, backward, (unsigned)grid, stream);
    if (rc2) return rc2;
  }
  if (!sums) return B200_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((d + 31) / 32), 2);
  cfg.blockDim = dim3(1024);
  cfg.stream = stream;
  cudaLaunchAttribute early;                               // its launch overlaps the end of the kernel before it
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  const int rc3 = note_cuda_error(cudaLaunchKernelEx(&cfg, gain_sum_kernel, (const float*)g.partial, (int)ctas[0], (int)ctas[1], (int)d,
                                                     q_gain_grad, k_gain_grad, accumulate), "gain gradient launch");
  count_launch(false);
  return rc3;
}

}  // namespace b200
