// Attention of new tokens over the paged 8-bit cache (kv_common.cuh):
//
//     o = softmax(alpha * q K^T) V   over the slots that the token may see,   K = ck * sk,  V = cv * sv
//
// with ck, cv the e4m3 codes and sk, sv their blocks' scales, powers of two.  The value scale goes into the exponent:
// with  s' = alpha log2(e) sk (q . ck) + log2(sv),  m' a running maximum of s',  p' = 2^(s' - m' + 14):
//
//     o = sum p' cv / l,     l = sum p' / sv,     log-sum-exp = ln 2 (m' - 14 + log2 l)
//
// so the probabilities that meet the codes lie in [0, 2^15] whatever the scales are, and one pass keeps one maximum
// (which may lag behind the largest s' by 1).  The lift by 2^14 uses f16's upper binades too: a probability keeps its 11
// bits down to 2^-28 of the largest, which matters where the most probable slot's values are small beside another's.
//
//   kv_decode_kernel    few rows: bound by reading the codes.  A CTA has one (sequence, key head), up to 8 * NQ of its
//                       rows (a row is a new token and one of the query heads that share the key head) and a range of
//                       slots; its four warps take every fourth 16 slots each, on m16n8k16 f16 matrix instructions (the
//                       fifth-generation ones take 128 rows at least, which a token's shared heads do not fill).
//                       The order of the products' summation index and of the output columns is free, and is chosen so
//                       that each lane reads whole 16-byte (d = 128) pieces of a row, a warp whole 128-byte lines, and
//                       that no lane needs what another has read: codes go from global memory to registers, a tile
//                       ahead, with no shared memory and no barrier in the loop.  (A ring in shared memory filled by
//                       asynchronous copies took 150 us where this takes 117.)
//                       Scores, maxima, sums and outputs are f32; codes are exact in f16, probabilities are rounded
//                       to f16 for the second product only (2^-12 of each, of random sign).
//                       48 sequences of 200 to 12000 slots, one token, 32 query and 8 key heads of 128: 117 us with the
//                       joining, 5.2 TB/s, 0.79 of a plain copy; one of 131000: 53 us, 5.0 TB/s.
//   kv_combine_kernel   joins the ranges of a row, in order; its launch overlaps the end of the kernel before.
// The kernel for many rows is in kv_attention_tc.cu.
// A range is a fixed number of slots, not a share of the sequence, so that ragged lengths give CTAs of equal work.
#include "kv_attention.cuh"

namespace b200 {

namespace {

using namespace kv;

constexpr int WARPS = 4;
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// How SHARE neighbouring lanes share a row of codes, N words each: in pieces of SIZE bytes (16 for N % 4 == 0, 8 for
// N % 2 == 0, else 4), piece i of all lanes side by side, so that every access covers whole 32-byte sectors.
template <int N, int SHARE> struct Words {
  static constexpr int SIZE = N % 4 == 0 ? 16 : N % 2 == 0 ? 8 : 4, PIECES = N * 4 / SIZE;
  // the code behind word w's first byte in lane `share`
  static __device__ __forceinline__ constexpr int code(int w, int share) { return (w * 4 / SIZE * SHARE + share) * SIZE + w * 4 % SIZE; }
  static __device__ __forceinline__ void load(const uint8_t* row, int share, uint32_t (&w)[N]) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const uint8_t* p = row + (i * SHARE + share) * SIZE;
      if constexpr (SIZE == 16) {
        const uint4 x = __ldg(reinterpret_cast<const uint4*>(p));
        w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
      } else if constexpr (SIZE == 8) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
        w[2 * i] = x.x; w[2 * i + 1] = x.y;
      } else {
        w[i] = __ldg(reinterpret_cast<const uint32_t*>(p));
      }
    }
  }
};
__device__ __forceinline__ uint32_t transposed(uint32_t x) {         // an 8 x 8 matrix of f16, two a lane
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// NQ: eights of rows.  The products are taken transposed, S^T = K Q^T and O^T = V^T P^T: the matrix instruction's 16-row
// side then holds slots and head elements, which there are always enough of, and its 8-column side the few rows.
template <int D, int NQ>
__global__ void __launch_bounds__(WARPS * 32, NQ == 1 ? 3 : 2) kv_decode_kernel(const __grid_constant__ AttArgs g) {
  constexpr int KS = D / 16;                               // k-steps of S^T; also 16-element tiles of O^T
  constexpr int KW = D / 16;                               // words of a key row that a lane holds (D / 4 codes)
  constexpr int VW = D / 32;                               // words of a value row that a lane holds (D / 8 codes)
  typedef Words<KW, 4> KeyWords;
  typedef Words<VW, 8> ValueWords;
  constexpr int R = 8 * NQ;
  constexpr bool Q_REGS = NQ == 1;
  __shared__ __align__(16) float sh_o[WARPS][8][D + 4];
  __shared__ float sh_m[WARPS][8], sh_l[WARPS][8];
  __shared__ __align__(16) uint2 sh_q[Q_REGS ? 1 : NQ * KS * 32];
  __shared__ int sh_nan;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, c = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;");       // the joining kernel may be brought in; it waits for this one
  Work w;
  // All sequences' first ranges, then the second ones, and so on: what runs last are the ends of the longest.  (17.2 us
  // against 17.6 sequence by sequence for 24 sequences' drafts of 2 to 5 tokens, 22.3 against 23.3 for 16 of 4.)
  const unsigned units = gridDim.x / (unsigned)g.splits, unit = blockIdx.x % units;
  const int x_range = (int)(blockIdx.x / units);
  if (!work_of<R>(g, unit, x_range, w)) return;
  const long long cta = (long long)unit * g.splits + x_range;        // its place among the partial results
  if (threadIdx.x == 0) sh_nan = 0;

  // the queries as the second operand: lane (gr, c) has four elements of row gr at each step, the same order of summation
  // in which it reads the keys
  uint2 qf[Q_REGS ? KS : 1];
  auto query_of = [&](int r) -> const __half* {
    const int row = w.tile * R + r;
    return g.q + (long long)(w.q.first + row / g.group) * g.qt + (long long)(w.head * g.group + row % g.group) * g.qh;
  };
  if constexpr (Q_REGS) {
    const __half* src = query_of(min(gr, w.rows - 1));
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = *reinterpret_cast<const uint2*>(src + KeyWords::code(ks, c));
  } else {
    for (int i = threadIdx.x; i < NQ * KS * 32; i += WARPS * 32) {
      const int l = i & 31, ks = (i >> 5) % KS, nt = (i >> 5) / KS;
      sh_q[i] = *reinterpret_cast<const uint2*>(query_of(min(nt * 8 + (l >> 2), w.rows - 1)) + KeyWords::code(ks, l & 3));
    }
  }
  // the pages and scales of a warp's next 32 tiles, one a lane; the first ones while the queries are on their way
  const int* table = g.batch.table + (long long)w.s * g.batch.table_stride;
  int id;
  float ks_l, vs_l;
  uint32_t bad_tiles;
  auto pages_from = [&](int i0) {
    const int mine = i0 + lane * WARPS;
    bool bad = false;
    id = 0;
    ks_l = 0.f;
    vs_l = 1.f;
    if (mine < w.end) {
      id = __ldg(table + ((mine << 4) >> g.cache.page_log2));
      bad = id < 0 || id >= g.cache.pages;
      if (bad) id = 0;                                     // its slots count for nothing; the caller learns of it
      ks_l = __ldg(g.cache.k_scale + (long long)id * g.cache.heads + w.head) * g.scale_log2;
      vs_l = __ldg(g.cache.v_scale + (long long)id * g.cache.heads + w.head);
    }
    bad_tiles = __ballot_sync(0xffffffffu, bad);
    if (bad_tiles && lane == 0) flag_index(g.status);
  };
  pages_from(w.begin + warp);
  __syncthreads();

  float o[NQ][KS][4];
  float m[NQ][2], l[NQ][2];                                // of rows 2 c and 2 c + 1
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
#pragma unroll
    for (int j = 0; j < KS; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][j][e] = 0.f;
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
  }

  const int in_page = g.cache.page - 1;
  for (int i0 = w.begin + warp; i0 < w.end; i0 += WARPS * 32) {
    if (i0 != w.begin + warp) pages_from(i0);
    const int n = min(32, (w.end - i0 + WARPS - 1) / WARPS);
    // Two tiles' codes in registers: the next ones load while these are worked on.
    auto load = [&](int i, uint32_t (&kw)[2][KW], uint32_t (&vw)[4][VW]) {
      const int page = __shfl_sync(0xffffffffu, id, i);
      const long long at = (((long long)page * g.cache.heads + w.head) * g.cache.page + (((i0 + i * WARPS) << 4) & in_page)) * D;
#pragma unroll
      for (int h = 0; h < 2; ++h) KeyWords::load(g.cache.k + at + (h * 8 + gr) * D, c, kw[h]);
#pragma unroll
      for (int t = 0; t < 4; ++t) ValueWords::load(g.cache.v + at + (2 * c + (t & 1) + (t >> 1) * 8) * D, gr, vw[t]);
    };
    auto step = [&](int i, uint32_t (&kw)[2][KW], uint32_t (&vw)[4][VW], uint32_t (&next_kw)[2][KW], uint32_t (&next_vw)[4][VW]) {
      if (i + 1 < n) load(i + 1, next_kw, next_vw);
      const int slot0 = (i0 + i * WARPS) << 4;
      const float sk = __shfl_sync(0xffffffffu, ks_l, i);
      const uint32_t sv = __float_as_uint(__shfl_sync(0xffffffffu, vs_l, i));
      const float lsv = (float)((int)(sv >> 23) - 127), inv_sv = __uint_as_float((254u << 23) - sv);   // a power of two
      float sc[NQ][4];
#pragma unroll
      for (int t = 0; t < NQ; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[t][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const uint2 lo = values4(kw[0][ks]), hi = values4(kw[1][ks]);
#pragma unroll
        for (int t = 0; t < NQ; ++t) {
          const uint2 b = Q_REGS ? qf[Q_REGS ? ks : 0] : sh_q[(t * KS + ks) * 32 + lane];
          mma16816(sc[t], lo.x, hi.x, lo.y, hi.y, b.x, b.y);
        }
      }

      // sc: slots gr (0, 1) and gr + 8 (2, 3), rows 2 c (0, 2) and 2 c + 1 (1, 3)
      const bool tile_bad = (bad_tiles >> i) & 1u;
      const bool edge = tile_bad || slot0 < w.lo_all || slot0 + 16 > w.hi_all;
      uint32_t pb[NQ][2];
#pragma unroll
      for (int t = 0; t < NQ; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[t][e] = fmaf(sc[t][e], sk, lsv);
        if (edge) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int r = t * 8 + 2 * c + y;
            const View v = view_of(g, w.q, w.tile * R + min(r, w.rows - 1));
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int slot = slot0 + h * 8 + gr;
              if (tile_bad || slot < v.lo || slot >= v.hi) sc[t][2 * h + y] = -INFINITY;
            }
          }
        }
        // The maximum moves only when a score passes it by more than 1: most tiles then need neither its reduction over
        // the slots nor a change of the sums, and probabilities stay below 2 * 2^LIFT.
        if (__any_sync(0xffffffffu, fmaxf(sc[t][0], sc[t][2]) > m[t][0] + 1.f || fmaxf(sc[t][1], sc[t][3]) > m[t][1] + 1.f)) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float top = fmaxf(sc[t][y], sc[t][2 + y]);
#pragma unroll
            for (int x = 4; x < 32; x *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float now = fmaxf(m[t][y], top);
            const float f = now == -INFINITY ? 1.f : ex2(m[t][y] - now);
            m[t][y] = now;
            l[t][y] *= f;
#pragma unroll
            for (int j = 0; j < KS; ++j) { o[t][j][y] *= f; o[t][j][2 + y] *= f; }
          }
        }
        float p[4];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float nm = m[t][y] == -INFINITY ? 0.f : LIFT - m[t][y];
          p[y] = ex2(sc[t][y] + nm);
          p[2 + y] = ex2(sc[t][2 + y] + nm);
          l[t][y] = fmaf(p[y] + p[2 + y], inv_sv, l[t][y]);
        }
        pb[t][0] = transposed(half2_of(p[0], p[1]));
        pb[t][1] = transposed(half2_of(p[2], p[3]));
      }
      if (edge) {
        // A NaN among values that some row does not see must not reach it through 0 * NaN: it is taken out here and put
        // back at the end where it belongs.
        uint32_t any = 0;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int x = 0; x < VW; ++x) {
            const uint32_t gone = nan_bytes(vw[t][x]);
            any |= gone;
            vw[t][x] &= ~gone;
          }
        if (any) sh_nan = 1;
      }
#pragma unroll
      for (int x = 0; x < VW; ++x)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          // codes 4 x + 2 b and + 1 of the lane's run: (slot, slot + 1) pairs side by side
          const uint32_t sel = b == 0 ? 0x5140u : 0x7362u;
          const uint32_t x0 = __byte_perm(vw[0][x], vw[1][x], sel), x1 = __byte_perm(vw[2][x], vw[3][x], sel);
          const uint2 lo = values4(x0), hi = values4(x1);
#pragma unroll
          for (int t = 0; t < NQ; ++t) mma16816(o[t][2 * x + b], lo.x, lo.y, hi.x, hi.y, pb[t][0], pb[t][1]);
        }
    };
    uint32_t ka[2][KW], va[4][VW], kb[2][KW], vb[4][VW];
    load(0, ka, va);
    for (int i = 0; i < n; i += 2) {
      step(i, ka, va, kb, vb);
      if (i + 1 < n) step(i + 1, kb, vb, ka, va);
    }
  }

  // join the warps, then write the rows or leave them as a partial result
#pragma unroll
  for (int t = 0; t < NQ; ++t) {
    __syncthreads();
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      float sum = l[t][y];
#pragma unroll
      for (int x = 4; x < 32; x *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, x);
      const int r = 2 * c + y;
      if (gr == 0) { sh_m[warp][r] = m[t][y]; sh_l[warp][r] = sum; }
      // tiles' rows gr and gr + 8 are codes 2 j and 2 j + 1 of the lane's words
#pragma unroll
      for (int j = 0; j < KS; j += 2)
        *reinterpret_cast<float4*>(&sh_o[warp][r][ValueWords::code(j / 2, gr)]) = make_float4(o[t][j][y], o[t][j][2 + y], o[t][j + 1][y], o[t][j + 1][2 + y]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * (D / 8); i += WARPS * 32) {
      const int r = i / (D / 8), j = (i % (D / 8)) * 8;
      if (t * 8 + r >= w.rows) continue;
      float top = sh_m[0][r];
#pragma unroll
      for (int x = 1; x < WARPS; ++x) top = fmaxf(top, sh_m[x][r]);
      float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < WARPS; ++x) {
        const float f = sh_m[x][r] == -INFINITY ? 0.f : ex2(sh_m[x][r] - top);
        sum = fmaf(sh_l[x][r], f, sum);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(sh_o[x][r][j + e], f, v[e]);
      }
      const int row = w.tile * R + t * 8 + r, tok = w.q.first + row / g.group, qh = w.head * g.group + row % g.group;
      if (sh_nan) nan_fixup(g, w, 1, row, j, v);
      if (w.ranges == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;    // a row that sees nothing: 0, and -inf below
        uint4 pk;
        pk.x = half2_of(v[0] * inv, v[1] * inv); pk.y = half2_of(v[2] * inv, v[3] * inv);
        pk.z = half2_of(v[4] * inv, v[5] * inv); pk.w = half2_of(v[6] * inv, v[7] * inv);
        *reinterpret_cast<uint4*>(g.out + tok * g.ot + qh * g.oh + j) = pk;
        if (g.lse && j == 0) g.lse[(long long)tok * g.q_heads + qh] = sum == 0.f ? -INFINITY : (top - LIFT + log2f(sum)) * 0.6931471805599453f;
      } else {
        float* dst = g.part_o + (cta * R + t * 8 + r) * D + j;
        *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
        if (j == 0) g.part_ml[cta * R + t * 8 + r] = make_float2(top, sum);
      }
    }
  }
}

// The ranges' partial results of a row, joined in order.  COLS lanes take a row's d elements, four each.  Up to FEW_RANGES
// ranges: these lanes hold all of a row's at once, several rows a CTA.  More: a CTA has one row, and every PARTS-th range
// goes to one of its groups of lanes.  (With the first form up to 2 ranges only: 6.5 us against 6.1 for one sequence of 900
// slots, 119.5 against 117 for 48 of up to 12000.)
constexpr int FEW_RANGES = 8;
template <int D, int R, bool FEW>
__global__ void __launch_bounds__(128) kv_combine_kernel(const AttArgs g, long long rows_all) {
  constexpr int COLS = D / 4, PARTS = 128 / COLS;          // 4, 5, 8 or 16 groups
  const int part = threadIdx.x / COLS, col = threadIdx.x % COLS;
  const long long item = FEW ? (long long)blockIdx.x * PARTS + part : blockIdx.x;
  const unsigned unit = (unsigned)(item / R);
  const int r = (int)(item % R);
  Work w;
  const bool mine = part < PARTS && item < rows_all && work_of<R>(g, unit, 0, w) && r < w.rows && w.ranges > 1;
  asm volatile("griddepcontrol.wait;" ::: "memory");       // the partial results are complete and visible
  const long long cta0 = (long long)unit * g.splits;
  float top = -INFINITY, sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if constexpr (FEW) {
    if (!mine) return;
    float2 ml[FEW_RANGES];
    float4 o[FEW_RANGES];
#pragma unroll
    for (int x = 0; x < FEW_RANGES; ++x) {
      ml[x] = make_float2(-INFINITY, 0.f);
      if (x < w.ranges) {
        ml[x] = g.part_ml[(cta0 + x) * R + r];
        o[x] = *reinterpret_cast<const float4*>(g.part_o + ((cta0 + x) * R + r) * D + col * 4);
      }
    }
#pragma unroll
    for (int x = 0; x < FEW_RANGES; ++x) top = fmaxf(top, ml[x].x);
#pragma unroll
    for (int x = 0; x < FEW_RANGES; ++x) {
      if (x >= w.ranges) continue;
      const float f = ml[x].x == -INFINITY ? 0.f : ex2(ml[x].x - top);
      sum = fmaf(ml[x].y, f, sum);
      v.x = fmaf(o[x].x, f, v.x); v.y = fmaf(o[x].y, f, v.y); v.z = fmaf(o[x].z, f, v.z); v.w = fmaf(o[x].w, f, v.w);
    }
  } else {
    __shared__ float sh_top[4];
    __shared__ float4 sh_v[PARTS][COLS];
    __shared__ float sh_sum[PARTS];
    const bool any = __syncthreads_or(mine);               // the same in all threads of a row but those behind the groups
    if (!any) return;
    if (part < PARTS) {
      for (int x = threadIdx.x; x < w.ranges; x += PARTS * COLS) top = fmaxf(top, g.part_ml[(cta0 + x) * R + r].x);
    }
#pragma unroll
    for (int x = 16; x > 0; x /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    if ((threadIdx.x & 31) == 0) sh_top[threadIdx.x >> 5] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sh_top[0], sh_top[1]), fmaxf(sh_top[2], sh_top[3]));
    if (part < PARTS) {
#pragma unroll 8
      for (int x = part; x < w.ranges; x += PARTS) {
        const float2 ml = g.part_ml[(cta0 + x) * R + r];
        const float4 o = *reinterpret_cast<const float4*>(g.part_o + ((cta0 + x) * R + r) * D + col * 4);
        const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
        sum = fmaf(ml.y, f, sum);
        v.x = fmaf(o.x, f, v.x); v.y = fmaf(o.y, f, v.y); v.z = fmaf(o.z, f, v.z); v.w = fmaf(o.w, f, v.w);
      }
      sh_v[part][col] = v;
      if (col == 0) sh_sum[part] = sum;
    }
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int x = 1; x < PARTS; ++x) {
      const float4 o = sh_v[x][col];
      sum += sh_sum[x];
      v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
    }
  }
  const int row = w.tile * R + r, tok = w.q.first + row / g.group, qh = w.head * g.group + row % g.group;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint2*>(g.out + tok * g.ot + qh * g.oh + col * 4) = make_uint2(half2_of(v.x * inv, v.y * inv), half2_of(v.z * inv, v.w * inv));
  if (g.lse && col == 0) g.lse[(long long)tok * g.q_heads + qh] = sum == 0.f ? -INFINITY : (top - LIFT + log2f(sum)) * 0.6931471805599453f;
}

struct Plan {
  bool few, many;                  // which kernels the batch may need
  int nq;                          // few rows: eights of rows of a tile
  AttArgs f, m;                    // their tiles, splits, ranges and row limits
  long long f_units, m_units;      // row tiles
  long long f_ctas() const { return f_units * f.splits; }
  long long m_ctas() const { return m_units * m.splits; }
  // partial results: rows of d + 2 floats
  size_t f_rows() const { return few && f.splits > 1 ? (size_t)f_ctas() * 8 * nq : 0; }
  size_t m_rows() const { return many && m.splits > 1 ? (size_t)m_ctas() * TC_ROWS : 0; }
};

// Sequences with up to this many rows go to the kernel for few rows.  In us, this kernel against the one for many, 32 query
// and 8 key heads: 24 sequences of 50 to 6000 slots, 20 rows of 128: 81, 93; 32 rows of 96: 83, 95; one sequence of 30000,
// 32 rows of 96: 31, 41; 64 short ones, 32 rows of 128: 61, 65.  At 32 rows of 128 the registers are used up and the two
// meet: 112, 95 for the 24 sequences, 40, 40 for the long one.
constexpr int FEW_ROWS = 32;
constexpr int ROUNDS = 4;          // 48 sequences of 200 to 12000 slots: 138 us with 3, 120 with 4, 121 with 6, 127 with 8

// How the rows and slots of a call are cut.  Everything follows from what the host knows: the lengths stay on the device,
// the page table's width bounds them.
Plan plan_of(const Cache& c, const Batch& b, int64_t q_heads, int64_t window, int causal, int sms) {
  Plan p;
  const int64_t group = q_heads / c.heads, rows = (int64_t)b.max_new * group;
  int64_t bound = (int64_t)b.max_pages << c.page_log2;
  if (bound > MAX_SLOTS) bound = MAX_SLOTS;
  if (window && causal && bound > window + b.max_new + 16) bound = window + b.max_new + 16;
  p.many = rows > FEW_ROWS;
  // One launch does where every sequence may be as long as max_new: the kernel for many rows then takes the shorter ones
  // of a padded batch too.
  p.few = !p.many || (int64_t)b.seqs * b.max_new != b.tokens;
  const int64_t few_rows = p.many ? FEW_ROWS : rows;
  p.nq = few_rows <= 8 ? 1 : few_rows <= 16 ? 2 : few_rows <= 24 ? 3 : 4;
  p.f.tiles = 1;
  p.f_units = (int64_t)b.seqs * c.heads;
  p.f.rows_over = 0;
  p.f.rows_most = FEW_ROWS;
  // Tiles are cut into ranges of slots: into as many as make one round of CTAs, which is the quickest for one sequence and
  // for short ones, where a CTA's start (about 4 us of latencies) costs more than its reading.  Where one round's ranges
  // would be longer than 1024 slots and there are several sequences, into ROUNDS rounds if all were as long as the
  // bound, no shorter than that: shorter sequences leave CTAs that return at once, and the ranges' equal length evens out
  // the others.
  auto cut = [&](AttArgs& a, int64_t units, int64_t round, int most_rounds, int64_t least, int64_t unit) {
    int64_t range = 0;
    for (int rounds = 1; rounds <= most_rounds; rounds += most_rounds > 1 ? most_rounds - 1 : 1) {
      int64_t parts = rounds * round / (units > 0 ? units : 1);
      if (parts < 1) parts = 1;
      const int64_t r = ((bound + parts - 1) / parts + unit - 1) / unit * unit;
      if (rounds == 1 || (range > 1024 && b.seqs > 1)) range = rounds == 1 || r > 1024 ? r : 1024;
    }
    if (range < least) range = least;
    a.range = (int)(range > (1 << 30) ? (1 << 30) : range);
    a.splits = (int)((bound + a.range - 1) / a.range);
    if (a.splits < 1) a.splits = 1;
  };
  cut(p.f, p.f_units, (int64_t)sms * (p.nq == 1 ? 3 : 2), ROUNDS, 256, 64);
  // Many rows: tiles of 256, cut along the slots only while there are fewer of them than SMs.
  p.m.tiles = (int)((rows + TC_ROWS - 1) / TC_ROWS);
  p.m_units = (int64_t)b.seqs * c.heads * p.m.tiles;
  p.m.rows_over = p.few ? FEW_ROWS : 0;
  p.m.rows_most = 0x7fffffff;
  cut(p.m, p.m_units, sms, 1, 1024, 128);
  return p;
}

template <int D, int R>
int combine_one(const AttArgs& g, long long units, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  const bool few = g.splits <= FEW_RANGES;
  const int per_cta = few ? 128 / (D / 4) : 1;
  cfg.gridDim = dim3((unsigned)((units * R + per_cta - 1) / per_cta));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute early;                               // its launch overlaps the end of the kernel before it
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  const int rc = note_cuda_error(few ? cudaLaunchKernelEx(&cfg, kv_combine_kernel<D, R, true>, g, units * R)
                                     : cudaLaunchKernelEx(&cfg, kv_combine_kernel<D, R, false>, g, units * R), "cache attention join launch");
  count_launch(false);
  return rc;
}
template <int D>
int combine_d(const AttArgs& g, int rows, long long units, cudaStream_t stream) {
  switch (rows) {
    case 8: return combine_one<D, 8>(g, units, stream);
    case 16: return combine_one<D, 16>(g, units, stream);
    case 24: return combine_one<D, 24>(g, units, stream);
    case 32: return combine_one<D, 32>(g, units, stream);
    default: return combine_one<D, TC_ROWS>(g, units, stream);
  }
}
int combine(const AttArgs& g, int rows, long long units, cudaStream_t stream) {
  switch (g.cache.d) {
    case 32: return combine_d<32>(g, rows, units, stream);
    case 64: return combine_d<64>(g, rows, units, stream);
    case 96: return combine_d<96>(g, rows, units, stream);
    default: return combine_d<128>(g, rows, units, stream);
  }
}

template <int D, int NQ>
int launch_few(const AttArgs& g, long long ctas, cudaStream_t stream) {
  kv_decode_kernel<D, NQ><<<(unsigned)ctas, WARPS * 32, 0, stream>>>(g);
  count_launch(true);
  return note_cuda_error(cudaGetLastError(), "cache attention launch");
}
template <int D>
int launch_few_d(const AttArgs& g, int nq, long long ctas, cudaStream_t stream) {
  switch (nq) {
    case 1: return launch_few<D, 1>(g, ctas, stream);
    case 2: return launch_few<D, 2>(g, ctas, stream);
    case 3: return launch_few<D, 3>(g, ctas, stream);
    default: return launch_few<D, 4>(g, ctas, stream);
  }
}

}  // namespace

int kv_attention_setup_device() { return kv::setup_attention_tc(); }

size_t kv_cache_attention_workspace_bytes(const b200_kv_cache* cache, const b200_kv_batch* batch, int64_t q_heads, int64_t window, int causal) {
  Cache c;
  Batch b;
  if (parse_cache(cache, &c) || parse_batch(batch, &b) || q_heads <= 0 || q_heads % c.heads) return 0;
  if (c.pages == 0) b.max_pages = 0;
  const DeviceState* ds = device_state();
  const Plan p = plan_of(c, b, q_heads, window, causal, ds ? ds->sm_count : 148);
  return (p.f_rows() + p.m_rows()) * (c.d + 2) * sizeof(float);
}

int kv_cache_attention(int dtype, const b200_kv_cache* cache, const b200_kv_batch* batch, int64_t q_heads, const void* q,
                       const int64_t qs[2], double alpha, int causal, int64_t window, void* out, const int64_t os[2], float* lse,
                       void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  if (dtype != B200_F16 && dtype != B200_AMP_F16) return B200_ERR_UNSUPPORTED;
  AttArgs g;
  int rc = parse_cache(cache, &g.cache);
  if (rc) return rc;
  if ((rc = parse_batch(batch, &g.batch))) return rc;
  if (g.cache.pages == 0) g.batch.max_pages = 0;           // no page can be named: only empty sequences pass
  if (q_heads <= 0 || q_heads % g.cache.heads) return B200_ERR_SHAPE;
  if (window > 0x3fffffff || q_heads > 0x3fffffff) return B200_ERR_LIMIT;
  if (window && !causal) return B200_ERR_UNSUPPORTED;      // a window reaches back from the token's own slot
  if (g.batch.seqs == 0 || g.batch.tokens == 0 || g.batch.max_new == 0) return B200_OK;
  if (!q || !out) return B200_ERR_NULL;
  const DeviceState* ds = device_state();
  if (!ds) return note_cuda_error(cudaErrorInitializationError, "b200_init not called on this device");
  if (((uintptr_t)q | (uintptr_t)out) & 15) return B200_ERR_UNSUPPORTED;
  if (qs[0] % 8 || qs[1] % 8 || os[0] % 8 || os[1] % 8) return B200_ERR_UNSUPPORTED;
  const Plan p = plan_of(g.cache, g.batch, q_heads, window, causal, ds->sm_count);
  if ((int64_t)g.batch.max_new * (q_heads / g.cache.heads) > 0x3fffffff || p.f_ctas() * 8 * p.nq > 0x7fffffff || p.m_ctas() > 0x7fffffff ||
      p.m_units * TC_ROWS > 0x7fffffff)
    return B200_ERR_LIMIT;
  const size_t need = (p.f_rows() + p.m_rows()) * (g.cache.d + 2) * sizeof(float);
  if (need && (!workspace || ((uintptr_t)workspace & 15))) return B200_ERR_NULL;
  if (workspace_bytes < need) return B200_ERR_WORKSPACE;
  g.q_heads = (int)q_heads; g.group = (int)(q_heads / g.cache.heads);
  g.causal = causal != 0; g.window = (int)window;
  g.scale_log2 = (float)(alpha * 1.4426950408889634);
  g.q = (const __half*)q; g.qt = qs[0]; g.qh = qs[1];
  g.out = (__half*)out; g.ot = os[0]; g.oh = os[1];
  g.lse = lse;
  g.status = ds->status;
  auto with = [&](const AttArgs& cut, float* part, size_t rows) {
    AttArgs a = g;
    a.tiles = cut.tiles; a.splits = cut.splits; a.range = cut.range;
    a.rows_over = cut.rows_over; a.rows_most = cut.rows_most;
    a.part_o = part;
    a.part_ml = (float2*)(part + rows * g.cache.d);
    return a;
  };
  float* part = (float*)workspace;
  if (p.many) {
    const AttArgs a = with(p.m, part, p.m_rows());
    // One CTA runs on an SM.  In two to four rounds of them the order decides how late the last ones end: 244 us against
    // 253 for prompts of 511, 957 and 1024 tokens behind up to 6000, 134 against 148 for one of 3000 (32 query heads, 8 key
    // heads of 128).  In more rounds what the order costs every CTA, about 2 us, is not won back: 236 us against 207 for 60
    // prompts of 40 to 250 tokens in 13 rounds.
    const bool sort = p.m_ctas() > ds->sm_count && p.m_ctas() <= 4 * (int64_t)ds->sm_count;
    if ((rc = launch_attention_tc(a, p.m_ctas(), sort, stream))) return rc;
    if (a.splits > 1 && (rc = combine(a, TC_ROWS, p.m_units, stream))) return rc;
    part += p.m_rows() * (g.cache.d + 2);
  }
  if (p.few) {
    const AttArgs a = with(p.f, part, p.f_rows());
    switch (g.cache.d) {
      case 32: rc = launch_few_d<32>(a, p.nq, p.f_ctas(), stream); break;
      case 64: rc = launch_few_d<64>(a, p.nq, p.f_ctas(), stream); break;
      case 96: rc = launch_few_d<96>(a, p.nq, p.f_ctas(), stream); break;
      default: rc = launch_few_d<128>(a, p.nq, p.f_ctas(), stream);
    }
    if (rc) return rc;
    if (a.splits > 1 && (rc = combine(a, 8 * p.nq, p.f_units, stream))) return rc;
  }
  return B200_OK;
}

}  // namespace b200
