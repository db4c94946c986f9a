// Norm of every query and key head with the position rotation in the same pass, forward and backward
// (head_transform.cuh has the formulas).  The least that has to move is each element once in and once out forward, x and
// the upstream gradient in and the gradient out backward; the norm's statistics are recomputed from the row that the
// backward holds anyway, so nothing is saved between the two.
//
//   qk_forward_kernel   a group of LPR lanes owns a token and walks its heads (queries, then keys) `per_token` groups
//                       apart.  The angles go through f64 and are the costliest part: their sines are put into a table in
//                       shared memory once for all heads, under the first rows' loads.  Two sets of rows in registers,
//                       one on its way while the other is worked on.
//                       Bound by HBM: 16384 tokens, 40 heads of 128, f16: 63 us, 5.3 TB/s, 0.81 of a plain copy.
//   qk_backward_kernel  the same walk by CTAs that stay and loop.  With h' = R^T g the gradient before the rotation,
//                         dgain += h' * xhat,   dx = r (h' gain - xhat mean(h' gain xhat)),   xhat = x r.
//                       The gains' sums stay in f32 registers over all rows of a lane, are added up per CTA in a fixed
//                       order and leave as one row of partial sums per CTA: at 59400 rows 1.7e-7 of the sums' norm off,
//                       where f64 sums of f32 products are 7e-8 off.
//                       Bound by what 16 warps an SM (12 in f32) can have on their way and by issue (0.54 of the cycles
//                       issue): 16384 tokens, 36 heads of 128, f16: 107 us, 4.2 TB/s; 4950 tokens, 24 heads of 96, f32:
//                       37 us, 3.7 TB/s.  More warps do not fit: x, g and the sums of both gains take 119 registers.
//   gain_sum_kernel     adds the CTAs' rows in a fixed order: no atomics, the same bits in every run.  Its launch overlaps
//                       the end of the backward.
#include "head_transform.cuh"

namespace b200 {

namespace {

using namespace heads;

struct Side {                      // queries or keys
  const void *x, *up;              // input; upstream gradient (backward)
  void* y;                         // output; gradient (backward)
  const void* gain;
  int heads;
  int xh, uh, yh;                  // element strides: head axis,
  long long xb, xt, ub, ut, yb, yt;  // batch and token axes
};
struct QkArgs {
  Transform t;
  Side side[2];
  int tokens, seq;                 // batch * tokens of a sequence
  int d, axes, per_token;          // per_token: groups that share a token
  const int* pos;                  // axes x tokens, or nullptr: the index in the sequence on every axis
  float* partial;                  // backward: 2 x gridDim.x rows of d sums, or nullptr
};

constexpr int THREADS = 128;

template <typename T, int S, int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(THREADS, 4) qk_forward_kernel(const __grid_constant__ QkArgs g) {
  constexpr int GROUPS = THREADS / LPR, U = VEC ? 2 : 1;   // rows of a set
  __shared__ float2 table[GROUPS * LPR * S];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const Lane<T, S, INTER, VEC> ln(lane, g.d, g.t.pairs);
  const int step = g.per_token, per_cta = GROUPS / step, part = group % step, mine = group / step;
  const int t0 = (int)blockIdx.x * per_cta, tok = t0 + mine;
  const bool on = tok < g.tokens;
  const int tc = min(tok, g.tokens - 1), ib = tc / g.seq, is = tc % g.seq;   // a group without a token works on the last one
  const float inv_d = 1.f / (float)g.d;
  // Two sets of rows: the next ones are on their way while these are worked on.
  Raw<T, S, VEC> ra[U], rb[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    ln.clear(ra[u]);
    ln.clear(rb[u]);
  }
  int first = part;
  bool filled = false;
  for (int w = 0; w < 2; ++w) {                            // queries, then keys; the next group begins where the last ended
    const Side& sd = g.side[w];
    const int heads = sd.heads;
    if (heads == 0) continue;
    const T* src = reinterpret_cast<const T*>(sd.x) + ib * sd.xb + is * sd.xt;
    T* dst = reinterpret_cast<T*>(sd.y) + ib * sd.yb + is * sd.yt;
    auto load = [&](int r0, Raw<T, S, VEC>(&raw)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u) ln.load(src + (long long)min(r0 + u * step + first, heads - 1) * sd.xh, raw[u]);
    };
    load(0, ra);
    const Row<S> gain = ln.gain(sd.gain);
    if (!filled) {                                         // under the first loads
      fill_table<THREADS>(g.t, table, per_cta, [&](int i) {    // once for all heads
        const int x = min(t0 + i, g.tokens - 1);
        return place_of(g.pos, g.axes, g.tokens, x, x % g.seq);
      });
      __syncthreads();
      filled = true;
    }
    const Coef<S> k = coef(angle_from<S>(table + mine * g.t.pairs, ln.j0, on ? g.t.pairs : 0), gain);
    auto work = [&](int r0, const Raw<T, S, VEC>(&raw)[U]) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int r = r0 + u * step + first;
        const Row<S> y = transformed<S, LPR, VEC>(ln.row(raw[u]), k, g.t, ln.j0, inv_d);
        if (on && r < heads) ln.store(dst + (long long)r * sd.yh, y);
      }
    };
    const int stride = U * step;
    for (int r0 = 0; r0 < heads; r0 += 2 * stride) {       // the same trip count in every group
      if (r0 + stride < heads) load(r0 + stride, rb);
      work(r0, ra);
      if (r0 + stride >= heads) break;
      if (r0 + 2 * stride < heads) load(r0 + 2 * stride, ra);
      work(r0 + stride, rb);
    }
    first = (part - heads) & (step - 1);
  }
}

template <typename T, int S, int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(THREADS, sizeof(T) == 2 ? 4 : 3) qk_backward_kernel(const __grid_constant__ QkArgs g) {
  constexpr int GROUPS = THREADS / LPR, U = VEC ? 2 : 1;
  __shared__ float2 table[GROUPS * LPR * S];
  __shared__ float sums[THREADS * 2 * S];
  __shared__ __align__(16) float gains[2][LPR][2 * S];
  asm volatile("griddepcontrol.launch_dependents;");       // the sum of the partial rows may be brought in; it waits for this
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const Lane<T, S, INTER, VEC> ln(lane, g.d, g.t.pairs);
  const int step = g.per_token, per_cta = GROUPS / step, part = group % step, mine = group / step, pairs = g.t.pairs;
  const float inv_d = 1.f / (float)g.d;
  Row<S> acc[2];                                           // the gains' gradients: queries, keys
#pragma unroll
  for (int w = 0; w < 2; ++w)
#pragma unroll
    for (int e = 0; e < S / 2; ++e) acc[w].a[e] = acc[w].b[e] = f2{0.f, 0.f};
  // Two sets of rows: the next ones are on their way while these are worked on.
  Raw<T, S, VEC> ax[U], ag[U], bx[U], bg[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    ln.clear(ax[u]);
    ln.clear(ag[u]);
    ln.clear(bx[u]);
    ln.clear(bg[u]);
  }
  for (int i = threadIdx.x; i < 2 * LPR; i += THREADS) {   // the gains in f32, in the lanes' order
    const Row<S> x = Lane<T, S, INTER, VEC>(i % LPR, g.d, g.t.pairs).gain(g.side[i / LPR].gain);
#pragma unroll
    for (int e = 0; e < S / 2; ++e) {
      *reinterpret_cast<float2*>(&gains[i / LPR][i % LPR][2 * e]) = make_float2(x.a[e].x, x.a[e].y);
      *reinterpret_cast<float2*>(&gains[i / LPR][i % LPR][S + 2 * e]) = make_float2(x.b[e].x, x.b[e].y);
    }
  }
  for (int t0 = (int)blockIdx.x * per_cta; t0 < g.tokens; t0 += (int)gridDim.x * per_cta) {
    const int tok = t0 + mine;
    const bool on = tok < g.tokens;
    const int tc = min(tok, g.tokens - 1), ib = tc / g.seq, is = tc % g.seq;
    int first = part;
    bool filled = false;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const Side& sd = g.side[w];
      const int heads = sd.heads;
      if (heads == 0) continue;
      const T* src = reinterpret_cast<const T*>(sd.x) + ib * sd.xb + is * sd.xt;
      const T* up = reinterpret_cast<const T*>(sd.up) + ib * sd.ub + is * sd.ut;
      T* dst = reinterpret_cast<T*>(sd.y) + ib * sd.yb + is * sd.yt;
      auto load = [&](int r0, Raw<T, S, VEC>(&rx)[U], Raw<T, S, VEC>(&rg)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = min(r0 + u * step + first, heads - 1);
          if (g.t.normalize) ln.load(src + (long long)r * sd.xh, rx[u]);
          ln.load(up + (long long)r * sd.uh, rg[u]);
        }
      };
      load(0, ax, ag);
      if (!filled) {
        __syncthreads();                                   // the table's last readers are done
        fill_table<THREADS>(g.t, table, per_cta, [&](int i) {                 // once for all heads
          const int x = min(t0 + i, g.tokens - 1);
          return place_of(g.pos, g.axes, g.tokens, x, x % g.seq);
        });
        __syncthreads();
        filled = true;
      }
      Angle<S> angle = angle_from<S>(table + mine * pairs, ln.j0, on ? pairs : 0);
#pragma unroll
      for (int e = 0; e < S / 2; ++e) angle.s[e] = neg2(angle.s[e]);         // the gradient turns back
      auto work = [&](int r0, const Raw<T, S, VEC>(&rx)[U], const Raw<T, S, VEC>(&rg)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int r = r0 + u * step + first;
          const bool live = on && r < heads;
          Row<S> h = turned<S, VEC>(ln.row(rg[u]), angle, ln.j0, pairs);
          if (g.t.normalize) {
            // both sums before the reciprocal root is known:  sum x^2  and  sum h gain x
            Row<S> gain;
#pragma unroll
            for (int e = 0; e < S / 2; ++e) {
              const float2 p = *reinterpret_cast<const float2*>(&gains[w][lane][2 * e]), q = *reinterpret_cast<const float2*>(&gains[w][lane][S + 2 * e]);
              gain.a[e] = pack(p.x, p.y);
              gain.b[e] = pack(q.x, q.y);
            }
            const Row<S> x = ln.row(rx[u]), hx = times(h, x);
            float sq, hg;
            group_sum_pair<LPR>(dot(x, x), dot(hx, gain), sq, hg);
            const float rs = rsqrtf(sq * inv_d + g.t.eps), b = -(hg * inv_d) * rs * rs * rs;
            const f2 rs2 = pack(rs, rs), back = pack(b, b);
#pragma unroll
            for (int e = 0; e < S / 2; ++e) {
              if (live) {
                acc[w].a[e] = fma2(hx.a[e], rs2, acc[w].a[e]);
                acc[w].b[e] = fma2(hx.b[e], rs2, acc[w].b[e]);
              }
              h.a[e] = fma2(h.a[e], mul2(gain.a[e], rs2), mul2(x.a[e], back));
              h.b[e] = fma2(h.b[e], mul2(gain.b[e], rs2), mul2(x.b[e], back));
            }
          }
          if (live) ln.store(dst + (long long)r * sd.yh, h);
        }
      };
      const int stride = U * step;
      for (int r0 = 0; r0 < heads; r0 += 2 * stride) {
        if (r0 + stride < heads) load(r0 + stride, bx, bg);
        work(r0, ax, ag);
        if (r0 + stride >= heads) break;
        if (r0 + 2 * stride < heads) load(r0 + 2 * stride, ax, ag);
        work(r0 + stride, bx, bg);
      }
      first = (part - heads) & (step - 1);
    }
  }
  if (!g.partial) return;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    float* out = g.partial + ((long long)w * gridDim.x + blockIdx.x) * g.d;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < S / 2; ++e) {
      float x, y;
      unpack(acc[w].a[e], x, y);
      sums[(group * 2 * S + 2 * e) * LPR + lane] = x;
      sums[(group * 2 * S + 2 * e + 1) * LPR + lane] = y;
      unpack(acc[w].b[e], x, y);
      sums[(group * 2 * S + S + 2 * e) * LPR + lane] = x;
      sums[(group * 2 * S + S + 2 * e + 1) * LPR + lane] = y;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * S * LPR; i += THREADS) {
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < GROUPS; ++j) sum += sums[j * 2 * S * LPR + i];
      const Lane<T, S, INTER, VEC> who(i % LPR, g.d, g.t.pairs);
      if (who.has(i / LPR % S)) out[who.at(i / LPR)] = sum;
    }
  }
}

// Adds the CTAs' rows: each of 32 warps every 32nd of the queries' (or keys') rows, then the warps in order.
__global__ void __launch_bounds__(1024) gain_sum_kernel(const float* __restrict__ partial, int parts, int d,
                                                        float* __restrict__ gq, float* __restrict__ gk, int accumulate) {
  __shared__ float sh[32][33];
  asm volatile("griddepcontrol.wait;" ::: "memory");       // the rows are complete and visible
  const bool keys = blockIdx.y;
  const int lane = threadIdx.x & 31, j = blockIdx.x * 32 + lane, y = threadIdx.x >> 5;
  if (keys) partial += (long long)parts * d;
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

constexpr int MAX_PARTS = 1024;

template <typename T, int S, int LPR, bool INTER, bool VEC>
int launch_one(const QkArgs& g, bool backward, unsigned grid, cudaStream_t stream) {
  if constexpr (S == 4) {
    if (backward) qk_backward_kernel<T, S, LPR, INTER, VEC><<<grid, THREADS, 0, stream>>>(g);
  }
  if (!backward) qk_forward_kernel<T, S, LPR, INTER, VEC><<<grid, THREADS, 0, stream>>>(g);
  count_launch(false);
  return note_cuda_error(cudaGetLastError(), "query/key norm and rotation launch");
}
template <typename T, int S, bool VEC>
int launch_lpr(const QkArgs& g, bool inter, int lpr, bool backward, unsigned grid, cudaStream_t stream) {
  switch (lpr) {
    case 4: return inter ? launch_one<T, S, 4, true, VEC>(g, backward, grid, stream) : launch_one<T, S, 4, false, VEC>(g, backward, grid, stream);
    case 8: return inter ? launch_one<T, S, 8, true, VEC>(g, backward, grid, stream) : launch_one<T, S, 8, false, VEC>(g, backward, grid, stream);
    case 16: return inter ? launch_one<T, S, 16, true, VEC>(g, backward, grid, stream) : launch_one<T, S, 16, false, VEC>(g, backward, grid, stream);
    default:
      if constexpr (S == 8) return B200_ERR_LIMIT;         // 16 lanes of 16 elements hold the largest head
      else return inter ? launch_one<T, S, 32, true, VEC>(g, backward, grid, stream) : launch_one<T, S, 32, false, VEC>(g, backward, grid, stream);
  }
}
int launch(const QkArgs& g, int dtype, bool inter, int run, int lpr, bool backward, unsigned grid, cudaStream_t stream) {
  if (dtype == B200_F32) return run ? launch_lpr<float, 4, true>(g, inter, lpr, backward, grid, stream) : launch_lpr<float, 4, false>(g, inter, lpr, backward, grid, stream);
  return run == 8 ? launch_lpr<__half, 8, true>(g, inter, lpr, backward, grid, stream)
         : run == 4 ? launch_lpr<__half, 4, true>(g, inter, lpr, backward, grid, stream)
                    : launch_lpr<__half, 4, false>(g, inter, lpr, backward, grid, stream);
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
  g.tokens = (int)(batch * seq);
  g.seq = (int)seq; g.d = (int)d;
  g.pos = positions;
  const bool inter = op->interleaved != 0;
  // Elements that a lane moves at a time.  Eight of f16 (16 bytes) halve the forward's loads, stores and exchanges (63 us
  // against 85 for 16384 tokens, 40 heads of 128); the backward, with two inputs and the gains' sums in registers, would
  // lose a quarter of its warps to them (119 us against 109 for 16384 tokens, 36 heads of 128, 41 against 33 for 8192, 32 of
  // 64).
  int run = 0;
  for (int n = es == 2 && !backward ? 8 : 4; n >= 4 && !run; n /= 2) {
    bool ok = d % (2 * n) == 0 && g.t.pairs % n == 0;
    const int64_t heads[2] = {q_heads, k_heads};
    for (int i = 0; i < (backward ? 4 : 2); ++i) ok = ok && (heads[i & 1] == 0 || vec_ok(n, es, in[i], in_strides[i][0], in_strides[i][1], in_strides[i][2]));
    for (int i = 0; i < 2; ++i) ok = ok && (heads[i] == 0 || vec_ok(n, es, out[i], out_strides[i][0], out_strides[i][1], out_strides[i][2]));
    if (ok) run = n;
  }
  const int lpr = lanes_per_row(d, run ? run : 4), groups = THREADS / lpr;
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
  }
  const int rows = (int)(q_heads + k_heads);
  const int64_t resident = (int64_t)ds->sm_count * (backward && es == 4 ? 3 : 4);
  g.per_token = groups_per_token(g.tokens, rows, groups, resident, run ? 2 : 1, backward);
  int64_t grid = rows ? (g.tokens + groups / g.per_token - 1) / (groups / g.per_token) : 0;
  // Backward: what is resident at once; each CTA's sums are two rows to add up at the end.
  if (backward && grid > resident) grid = resident;
  if (backward && grid > MAX_PARTS) grid = MAX_PARTS;
  const bool sums = backward && g.t.normalize && (q_gain_grad || k_gain_grad);
  g.partial = sums ? (float*)workspace : nullptr;
  if (grid) {                                              // an empty batch: sums over nothing follow
    const int rc2 = launch(g, dtype, inter, run, lpr, backward, (unsigned)grid, stream);
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
  const int rc3 = note_cuda_error(cudaLaunchKernelEx(&cfg, gain_sum_kernel, (const float*)g.partial, (int)grid, (int)d,
                                                     q_gain_grad, k_gain_grad, accumulate), "gain gradient launch");
  count_launch(false);
  return rc3;
}

}  // namespace b200
