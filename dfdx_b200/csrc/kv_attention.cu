// Attention of new tokens over the paged 8-bit cache (kv_common.cuh):
//
//     o = softmax(alpha * q K^T) V   over the slots that the token may see,   K = ck * sk,  V = cv * sv
//
// with ck, cv the e4m3 codes and sk, sv their blocks' scales, powers of two.  The value scale goes into the exponent:
// with  s' = alpha log2(e) sk (q . ck) + log2(sv),  m' a running maximum of s',  p' = 2^(s' - m' + 15):
//
//     o = sum p' cv / l,     l = sum p' / sv,     log-sum-exp = ln 2 (m' - 15 + log2 l)
//
// so the probabilities that meet the codes lie in [0, 2^15] whatever the scales are, and one pass keeps one maximum.
// The lift by 2^15 uses f16's upper binades too: a probability keeps its 11 bits down to 2^-29 of the largest, which
// matters where the most probable slot's values are small beside another's.
//
//   kv_decode_kernel    few rows: bound by reading the codes.  A CTA has one (sequence, key head), up to 16 * MT of its
//                       rows (a row is a new token and one of the query heads that share the key head) and a range of
//                       slots; each of its four warps walks 16 slots at a time on m16n8k16 f16 matrix instructions.
//                       Codes go from global memory to registers directly: the order of the products' summation index
//                       and of the output columns is free, and is chosen so that each lane reads whole 16-byte (d = 128)
//                       pieces of a row, a warp whole 128-byte lines, with no shared memory and no barrier in the loop.
//                       The next tile's keys load under this tile's softmax, the next values under its scores.
//                       Scores, maxima, sums and outputs are f32; codes are exact in f16, probabilities are rounded
//                       to f16 for the second product only (2^-12 of each, of random sign).
//   kv_combine_kernel   joins the ranges of a row, in order.
// A range is a fixed number of slots, not a share of the sequence, so that ragged lengths give CTAs of equal work.
#include "kv_common.cuh"

namespace b200 {

namespace {

using namespace kv;

struct AttArgs {
  Cache cache;
  Batch batch;
  int q_heads, group;              // group = q_heads / cache.heads
  int tiles;                       // row tiles of a (sequence, key head)
  int splits, range;               // ranges per row tile (at most), slots per range
  int causal, window;
  float scale_log2;                // alpha * log2(e)
  const __half* q;
  long long qt, qh;
  __half* out;
  long long ot, oh;
  float* lse;                      // tokens x q_heads, or nullptr
  float* part_o;                   // [cta][row][d] unnormalised outputs
  float2* part_ml;                 // [cta][row] maximum, sum
  int* status;
};

constexpr int WARPS = 4;
constexpr float LIFT = 15.f;       // log2 of the largest probability as the second product sees it

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// N words from an address aligned to 16 bytes (N % 4 == 0), 8 bytes (N % 2 == 0) or 4.  Codes are read once per CTA.
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const uint4 x = __ldg(reinterpret_cast<const uint4*>(p) + i);
      w[4 * i] = x.x; w[4 * i + 1] = x.y; w[4 * i + 2] = x.z; w[4 * i + 3] = x.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const uint2 x = __ldg(reinterpret_cast<const uint2*>(p) + i);
      w[2 * i] = x.x; w[2 * i + 1] = x.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
  }
}
__device__ __forceinline__ bool has_nan(uint32_t codes) {  // a byte that is 0x7f but for its sign
  const uint32_t x = (codes & 0x7f7f7f7fu) + 0x01010101u;
  return (x & 0x80808080u) != 0;
}
__device__ __forceinline__ uint32_t nan_bytes(uint32_t codes) {    // 0xff where the code is NaN
  const uint32_t x = (((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return x * 0xffu;
}

// The slots that row r of a sequence sees: [lo, hi).
struct View { int lo, hi; };
__device__ __forceinline__ View view_of(const AttArgs& g, const Seq& q, int r) {
  const int pos = q.len - q.m + r / g.group;
  View v;
  v.hi = g.causal ? max(pos + 1, 0) : q.len;
  v.lo = g.window ? max(pos + 1 - g.window, 0) : 0;
  return v;
}

template <int D, int MT>
__global__ void __launch_bounds__(WARPS * 32) kv_decode_kernel(const AttArgs g) {
  constexpr int KS = D / 16;                               // k-steps of the scores' product
  constexpr int NT = D / 8;                                // column tiles of the output
  constexpr int KW = D / 16;                               // words of a key row that a lane holds (D / 4 codes)
  constexpr int VW = D / 32;                               // words of a value row that a lane holds (D / 8 codes)
  constexpr int R = 16 * MT;
  __shared__ __align__(16) float sh_o[WARPS][16][D + 4];
  __shared__ float sh_m[WARPS][16], sh_l[WARPS][16];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gr = lane >> 2, c = lane & 3;
  unsigned rest = blockIdx.x;
  const int x = (int)(rest % (unsigned)g.splits); rest /= (unsigned)g.splits;
  const int tile = (int)(rest % (unsigned)g.tiles); rest /= (unsigned)g.tiles;
  const int head = (int)(rest % (unsigned)g.cache.heads), s = (int)(rest / (unsigned)g.cache.heads);
  const Seq q = load_seq(g.batch, g.cache, s);
  if (!q.ok) {
    if (threadIdx.x == 0) flag_index(g.status);
    return;
  }
  const int rows = min(q.m * g.group - tile * R, R);       // of this tile
  if (rows <= 0) return;
  const int lo_tile = view_of(g, q, tile * R).lo, hi_tile = view_of(g, q, tile * R + rows - 1).hi;
  const int first_range = lo_tile / g.range;
  const int ranges = hi_tile > lo_tile ? (hi_tile - 1) / g.range - first_range + 1 : 1;
  if (x >= ranges) return;
  const int begin = max(lo_tile, (first_range + x) * g.range) >> 4;          // in 16-slot tiles
  const int end = hi_tile > lo_tile ? (min(hi_tile, (first_range + x + 1) * g.range) + 15) >> 4 : begin;

  // this lane's rows: gr and gr + 8 of every 16
  uint32_t qf[MT][KS][4];
  int lo[MT][2], hi[MT][2];
  int lo_all = 0, hi_all = 0x7fffffff;                     // slots [lo_all, hi_all) are seen by every row of the tile
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = t * 16 + h * 8 + gr;
      View v = {0, 0};
      if (r < rows) {
        const int row = tile * R + r;
        v = view_of(g, q, row);
        const __half* src = g.q + (long long)(q.first + row / g.group) * g.qt + (long long)(head * g.group + row % g.group) * g.qh + c * (D / 4);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const uint2 w = *reinterpret_cast<const uint2*>(src + ks * 4);
          qf[t][ks][h] = w.x;
          qf[t][ks][2 + h] = w.y;
        }
      } else {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) qf[t][ks][h] = qf[t][ks][2 + h] = 0;
      }
      lo[t][h] = v.lo; hi[t][h] = v.hi;
    }
  lo_all = view_of(g, q, tile * R + rows - 1).lo;
  hi_all = view_of(g, q, tile * R).hi;

  float o[MT][NT][4];
  float m[MT][2], l[MT][2];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][j][e] = 0.f;
    m[t][0] = m[t][1] = -INFINITY;
    l[t][0] = l[t][1] = 0.f;
  }

  const int* table = g.batch.table + (long long)s * g.batch.table_stride;
  const int in_page = g.cache.page - 1, shift = g.cache.page_log2;
  for (int i0 = begin + warp; i0 < end; i0 += WARPS * 32) {
    // the pages and scales of the warp's next 32 tiles, one a lane
    const int mine = i0 + lane * WARPS;
    int id = 0;
    float ks_l = 0.f, vs_l = 1.f;
    bool bad = false;
    if (mine < end) {
      id = table[(mine << 4) >> shift];
      bad = id < 0 || id >= g.cache.pages;
      if (!bad) {
        ks_l = g.cache.k_scale[(long long)id * g.cache.heads + head];
        vs_l = g.cache.v_scale[(long long)id * g.cache.heads + head];
      }
    }
    if (__any_sync(0xffffffffu, bad)) {                    // its slots count for nothing; the caller learns of it
      if (lane == 0) flag_index(g.status);
    }
    const int n = min(32, (end - i0 + WARPS - 1) / WARPS);
    uint32_t kw[2][KW], vw[4][VW];
    auto base_of = [&](int i) -> long long {               // byte offset of tile i's first row
      const int page = max(__shfl_sync(0xffffffffu, bad ? -1 : id, i), 0);
      return (((long long)page * g.cache.heads + head) * g.cache.page + (((i0 + i * WARPS) << 4) & in_page)) * D;
    };
    auto load_k = [&](long long at) {
#pragma unroll
      for (int h = 0; h < 2; ++h) load_words<KW>(g.cache.k + at + (h * 8 + gr) * D + c * (D / 4), kw[h]);
    };
    auto load_v = [&](long long at) {
#pragma unroll
      for (int t = 0; t < 4; ++t) load_words<VW>(g.cache.v + at + (2 * c + (t & 1) + (t >> 1) * 8) * D + gr * (D / 8), vw[t]);
    };
    long long at = base_of(0);
    load_k(at);
    load_v(at);
    for (int i = 0; i < n; ++i) {
      const int slot0 = (i0 + i * WARPS) << 4;
      const bool tile_bad = __shfl_sync(0xffffffffu, (int)bad, i) != 0;
      const float sk = __shfl_sync(0xffffffffu, ks_l, i) * g.scale_log2, sv = __shfl_sync(0xffffffffu, vs_l, i);
      const float lsv = log2f(sv), inv_sv = 1.f / sv;      // sv is a power of two: both exact
      float sc[MT][2][4];
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[t][h][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t b0 = values2(kw[h][ks]), b1 = values2(kw[h][ks] >> 16);
#pragma unroll
          for (int t = 0; t < MT; ++t) mma16816(sc[t][h], qf[t][ks][0], qf[t][ks][1], qf[t][ks][2], qf[t][ks][3], b0, b1);
        }
      const long long next = i + 1 < n ? base_of(i + 1) : at;
      if (i + 1 < n) load_k(next);

      const bool edge = tile_bad || slot0 < lo_all || slot0 + 16 > hi_all;
      uint32_t p[MT][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[t][h][e] = fmaf(sc[t][h][e], sk, lsv);
        if (edge) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int slot = slot0 + h * 8 + 2 * c + (e & 1);
              if (tile_bad || slot < lo[t][e >> 1] || slot >= hi[t][e >> 1]) sc[t][h][e] = -INFINITY;
            }
        }
        float top[2];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          top[y] = fmaxf(fmaxf(sc[t][0][2 * y], sc[t][0][2 * y + 1]), fmaxf(sc[t][1][2 * y], sc[t][1][2 * y + 1]));
          top[y] = fmaxf(top[y], __shfl_xor_sync(0xffffffffu, top[y], 1));
          top[y] = fmaxf(top[y], __shfl_xor_sync(0xffffffffu, top[y], 2));
        }
        if (__any_sync(0xffffffffu, top[0] > m[t][0] || top[1] > m[t][1])) {
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float now = fmaxf(m[t][y], top[y]);
            const float f = now == -INFINITY ? 1.f : ex2(m[t][y] - now);
            m[t][y] = now;
            l[t][y] *= f;
#pragma unroll
            for (int j = 0; j < NT; ++j) { o[t][j][2 * y] *= f; o[t][j][2 * y + 1] *= f; }
          }
        }
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const float nm = m[t][y] == -INFINITY ? 0.f : LIFT - m[t][y];
          float sum = 0.f;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float p0 = ex2(sc[t][h][2 * y] + nm), p1 = ex2(sc[t][h][2 * y + 1] + nm);
            sum += p0 + p1;
            p[t][2 * h + y] = half2_of(p0, p1);
          }
          l[t][y] = fmaf(sum, inv_sv, l[t][y]);
        }
      }
      if (edge) {
        // A NaN among values that some row does not see must not reach it through 0 * NaN: such codes become 0 here, and
        // a second product of "sees the slot" with "is NaN" finds the outputs that are NaN by right.
        bool any = false;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int w = 0; w < VW; ++w) any |= has_nan(vw[t][w]);
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            uint32_t sees[4];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const int slot = slot0 + h * 8 + 2 * c;
                const bool s0 = !tile_bad && slot >= lo[t][y] && slot < hi[t][y];
                const bool s1 = !tile_bad && slot + 1 >= lo[t][y] && slot + 1 < hi[t][y];
                sees[2 * h + y] = half2_of(s0 ? 1.f : 0.f, s1 ? 1.f : 0.f);
              }
#pragma unroll
            for (int w = 0; w < VW; ++w)
#pragma unroll
              for (int b = 0; b < 4; ++b) {
                uint32_t f[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) f[k] = (nan_bytes(vw[k][w]) >> (8 * b)) & 1u;
                float hit[4] = {0.f, 0.f, 0.f, 0.f};
                mma16816(hit, sees[0], sees[1], sees[2], sees[3], f[0] * 0x3c00u | f[1] * 0x3c000000u, f[2] * 0x3c00u | f[3] * 0x3c000000u);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (hit[e] != 0.f) o[t][w * 4 + b][e] = NAN;
              }
          }
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int w = 0; w < VW; ++w) vw[t][w] &= ~nan_bytes(vw[t][w]);
        }
      }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int b = 0; b < 4; b += 2) {
          // codes of columns 4 w + b and + 1: (slot, slot + 1) pairs side by side
          const uint32_t sel = b == 0 ? 0x5140u : 0x7362u;
          const uint32_t x0 = __byte_perm(vw[0][w], vw[1][w], sel), x1 = __byte_perm(vw[2][w], vw[3][w], sel);
          const uint32_t f0 = values2(x0), f1 = values2(x1), f2 = values2(x0 >> 16), f3 = values2(x1 >> 16);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            mma16816(o[t][w * 4 + b], p[t][0], p[t][1], p[t][2], p[t][3], f0, f1);
            mma16816(o[t][w * 4 + b + 1], p[t][0], p[t][1], p[t][2], p[t][3], f2, f3);
          }
        }
      if (i + 1 < n) load_v(next);
      at = next;
    }
  }

  // join the warps, then write the rows or leave them as a partial result
  const bool whole = ranges == 1;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    __syncthreads();
#pragma unroll
    for (int y = 0; y < 2; ++y) {
      float sum = l[t][y];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int r = y * 8 + gr;
      if (c == 0) { sh_m[warp][r] = m[t][y]; sh_l[warp][r] = sum; }
      // columns 2 c and 2 c + 1 of the column tiles are D / 4 consecutive elements of the row
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < NT; j += 4)
          *reinterpret_cast<float4*>(&sh_o[warp][r][(2 * c + e) * (D / 8) + j]) =
              make_float4(o[t][j][2 * y + e], o[t][j + 1][2 * y + e], o[t][j + 2][2 * y + e], o[t][j + 3][2 * y + e]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 8); i += WARPS * 32) {
      const int r = i / (D / 8), j = (i % (D / 8)) * 8;
      if (t * 16 + r >= rows) continue;
      float top = sh_m[0][r];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) top = fmaxf(top, sh_m[w][r]);
      float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WARPS; ++w) {
        const float f = sh_m[w][r] == -INFINITY ? 0.f : ex2(sh_m[w][r] - top);
        sum = fmaf(sh_l[w][r], f, sum);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(sh_o[w][r][j + e], f, v[e]);
      }
      const int row = tile * R + t * 16 + r, tok = q.first + row / g.group, qh = head * g.group + row % g.group;
      if (whole) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;    // a row that sees nothing: 0, and -inf below
        uint4 pk;
        pk.x = half2_of(v[0] * inv, v[1] * inv); pk.y = half2_of(v[2] * inv, v[3] * inv);
        pk.z = half2_of(v[4] * inv, v[5] * inv); pk.w = half2_of(v[6] * inv, v[7] * inv);
        *reinterpret_cast<uint4*>(g.out + tok * g.ot + qh * g.oh + j) = pk;
        if (g.lse && j == 0) g.lse[(long long)tok * g.q_heads + qh] = sum == 0.f ? -INFINITY : (top - LIFT + log2f(sum)) * 0.6931471805599453f;
      } else {
        float* dst = g.part_o + ((long long)blockIdx.x * R + t * 16 + r) * D + j;
        *reinterpret_cast<float4*>(dst) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(v[4], v[5], v[6], v[7]);
        if (j == 0) g.part_ml[(long long)blockIdx.x * R + t * 16 + r] = make_float2(top, sum);
      }
    }
  }
}

// One warp per row: the ranges' partial results in their order.
template <int D, int MT>
__global__ void __launch_bounds__(256) kv_combine_kernel(const AttArgs g) {
  constexpr int R = 16 * MT, N = D / 32;
  const int lane = threadIdx.x & 31;
  const long long unit = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int r = (int)(unit % R);
  unsigned rest = (unsigned)(unit / R);
  const int tile = (int)(rest % (unsigned)g.tiles); rest /= (unsigned)g.tiles;
  const int head = (int)(rest % (unsigned)g.cache.heads), s = (int)(rest / (unsigned)g.cache.heads);
  if (s >= g.batch.seqs) return;
  const Seq q = load_seq(g.batch, g.cache, s);
  if (!q.ok) return;
  const int rows = min(q.m * g.group - tile * R, R);
  if (r >= rows) return;
  const int lo_tile = view_of(g, q, tile * R).lo, hi_tile = view_of(g, q, tile * R + rows - 1).hi;
  const int ranges = hi_tile > lo_tile ? (hi_tile - 1) / g.range - lo_tile / g.range + 1 : 1;
  if (ranges == 1) return;                                 // written already
  const long long cta0 = (unit / R) * g.splits;
  float top = -INFINITY;
  for (int x = 0; x < ranges; ++x) top = fmaxf(top, g.part_ml[(cta0 + x) * R + r].x);
  float sum = 0.f, v[N];
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = 0.f;
  for (int x = 0; x < ranges; ++x) {
    const float2 ml = g.part_ml[(cta0 + x) * R + r];
    const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
    sum = fmaf(ml.y, f, sum);
    const float* src = g.part_o + ((cta0 + x) * R + r) * D + lane * N;
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = fmaf(src[e], f, v[e]);
  }
  const int row = tile * R + r, tok = q.first + row / g.group, qh = head * g.group + row % g.group;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  __half* dst = g.out + tok * g.ot + qh * g.oh + lane * N;
#pragma unroll
  for (int e = 0; e < N; ++e) dst[e] = __float2half_rn(v[e] * inv);
  if (g.lse && lane == 0) g.lse[(long long)tok * g.q_heads + qh] = sum == 0.f ? -INFINITY : (top - LIFT + log2f(sum)) * 0.6931471805599453f;
}

struct Plan { int mt, tiles, splits, range; long long ctas; };

// How the rows and slots of a call are cut.  Everything follows from what the host knows: the lengths stay on the device,
// the page table's width bounds them.
Plan plan_of(const Cache& c, const Batch& b, int64_t q_heads, int64_t window, int causal, int sms) {
  Plan p;
  const int64_t group = q_heads / c.heads, rows = (int64_t)b.max_new * group;
  p.mt = rows > 16 ? 2 : 1;
  const int64_t tiles = (rows + 16 * p.mt - 1) / (16 * p.mt);
  int64_t bound = (int64_t)b.max_pages << c.page_log2;
  if (window && causal && bound > window + b.max_new) bound = window + b.max_new + 1;
  const int64_t base = (int64_t)b.seqs * c.heads * tiles;
  // Ranges long enough that a CTA's start and its partial result cost little next to its reading (256 slots of d = 128
  // are 64 KB), and no more of them than eight rounds of CTAs: what the bound overstates is CTAs that return at once.
  int64_t range = 256;
  const int64_t most = (int64_t)sms * 3 * 8;
  while (range < bound && base * ((bound + range - 1) / range) > most) range *= 2;
  p.range = (int)(range > (1 << 30) ? (1 << 30) : range);
  p.splits = (int)((bound + p.range - 1) / p.range) + (window ? 1 : 0);
  if (p.splits < 1) p.splits = 1;
  p.tiles = (int)tiles;
  p.ctas = base * p.splits;
  return p;
}

template <int D, int MT>
int launch_decode(const AttArgs& g, long long ctas, cudaStream_t stream) {
  kv_decode_kernel<D, MT><<<(unsigned)ctas, WARPS * 32, 0, stream>>>(g);
  count_launch(false);
  int rc = note_cuda_error(cudaGetLastError(), "cache attention launch");
  if (rc || g.splits == 1) return rc;
  const long long rows = ctas / g.splits * 16 * MT;
  kv_combine_kernel<D, MT><<<(unsigned)((rows + 7) / 8), 256, 0, stream>>>(g);
  count_launch(false);
  return note_cuda_error(cudaGetLastError(), "cache attention join launch");
}
template <int D>
int launch_decode_d(const AttArgs& g, const Plan& p, cudaStream_t stream) {
  return p.mt == 1 ? launch_decode<D, 1>(g, p.ctas, stream) : launch_decode<D, 2>(g, p.ctas, stream);
}

}  // namespace

size_t kv_cache_attention_workspace_bytes(const b200_kv_cache* cache, const b200_kv_batch* batch, int64_t q_heads, int64_t window, int causal) {
  Cache c;
  Batch b;
  if (parse_cache(cache, &c) || parse_batch(batch, &b) || q_heads <= 0 || q_heads % c.heads) return 0;
  if (c.pages == 0) b.max_pages = 0;
  const DeviceState* ds = device_state();
  const Plan p = plan_of(c, b, q_heads, window, causal, ds ? ds->sm_count : 148);
  return p.splits == 1 ? 0 : (size_t)p.ctas * 16 * p.mt * (c.d + 2) * sizeof(float);
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
  if (p.ctas > 0x7fffffff || p.ctas / p.splits * 16 * p.mt > 0x7fffffff) return B200_ERR_LIMIT;
  const size_t need = p.splits == 1 ? 0 : (size_t)p.ctas * 16 * p.mt * (g.cache.d + 2) * sizeof(float);
  if (need && (!workspace || ((uintptr_t)workspace & 15))) return B200_ERR_NULL;
  if (workspace_bytes < need) return B200_ERR_WORKSPACE;
  g.q_heads = (int)q_heads; g.group = (int)(q_heads / g.cache.heads);
  g.tiles = p.tiles; g.splits = p.splits; g.range = p.range;
  g.causal = causal != 0; g.window = (int)window;
  g.scale_log2 = (float)(alpha * 1.4426950408889634);
  g.q = (const __half*)q; g.qt = qs[0]; g.qh = qs[1];
  g.out = (__half*)out; g.ot = os[0]; g.oh = os[1];
  g.lse = lse;
  g.part_o = (float*)workspace;
  g.part_ml = (float2*)((float*)workspace + (size_t)p.ctas * 16 * p.mt * g.cache.d);
  g.status = ds->status;
  switch (g.cache.d) {
    case 32: return launch_decode_d<32>(g, p, stream);
    case 64: return launch_decode_d<64>(g, p, stream);
    case 96: return launch_decode_d<96>(g, p, stream);
    default: return launch_decode_d<128>(g, p, stream);
  }
}

}  // namespace b200
