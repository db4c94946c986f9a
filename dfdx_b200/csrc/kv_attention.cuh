// What the two kernels of the attention over the paged cache share (kv_attention.cu: few rows, kv_attention_tc.cu: many).
#pragma once
#include "kv_common.cuh"

namespace b200 {
namespace kv {

struct AttArgs {
  Cache cache;
  Batch batch;
  int q_heads, group;              // group = q_heads / cache.heads
  int tiles;                       // row tiles of a (sequence, key head)
  int splits, range;               // ranges per row tile (at most), slots per range
  int rows_over, rows_most;        // takes the sequences with more than rows_over rows and at most rows_most
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

constexpr float LIFT = 14.f;       // log2 of the probability at the running maximum, as the second product sees it

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t nan_bytes(uint32_t codes) {    // 0xff where the code is NaN: 0x7f but for its sign
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

// What a CTA works on: a row tile of R rows of one (sequence, key head), and one of its ranges.
struct Work {
  Seq q;
  int s, head, tile, rows;
  int lo_tile, hi_tile;            // slots that some row sees
  int lo_all, hi_all;              // slots that every row sees
  int ranges, begin, end;          // ranges in use; this one's tiles of 16 slots
};
template <int R>
__device__ __forceinline__ bool work_of(const AttArgs& g, unsigned unit, int x, Work& w) {
  w.tile = (int)(unit % (unsigned)g.tiles); unit /= (unsigned)g.tiles;
  w.head = (int)(unit % (unsigned)g.cache.heads);
  w.s = (int)(unit / (unsigned)g.cache.heads);
  if (w.s >= g.batch.seqs) return false;
  w.q = load_seq(g.batch, g.cache, w.s);
  if (!w.q.ok) {
    if (threadIdx.x == 0) flag_index(g.status);
    return false;
  }
  const int rows = w.q.m * g.group;
  w.rows = min(rows - w.tile * R, R);
  if (w.rows <= 0 || rows <= g.rows_over || rows > g.rows_most) return false;
  const View first = view_of(g, w.q, w.tile * R), last = view_of(g, w.q, w.tile * R + w.rows - 1);
  w.lo_tile = first.lo; w.hi_tile = last.hi;
  w.lo_all = last.lo; w.hi_all = first.hi;
  // ranges are counted from the first slot that some row sees (its group of 16)
  const int base = w.lo_tile & ~15;
  w.ranges = w.hi_tile > w.lo_tile ? (w.hi_tile - 1 - base) / g.range + 1 : 1;
  if (x >= w.ranges) return false;
  const long long from = base + (long long)x * g.range, to = from + g.range;
  w.begin = (int)(from >> 4);
  w.end = w.hi_tile > w.lo_tile ? ((int)min((long long)w.hi_tile, to) + 15) >> 4 : w.begin;
  return true;
}

// NaN values in slots that only some rows of a tile see were taken out of the product, `per` groups of 16 slots at a time;
// this puts them where they belong.  Rare enough to read the codes again: eight output elements of one row.
static __device__ __noinline__ void nan_fixup(const AttArgs& g, const Work& w, int per, int row, int j, float (&v)[8]) {
  const View view = view_of(g, w.q, row);
  const int* table = g.batch.table + (long long)w.s * g.batch.table_stride;
  for (int t0 = w.begin; t0 < w.end; t0 += per) {
    if (t0 * 16 >= w.lo_all && (t0 + per) * 16 <= w.hi_all) continue;
    for (int t = t0; t < min(t0 + per, w.end); ++t) {
      const int id = table[(t << 4) >> g.cache.page_log2];
      if (id < 0 || id >= g.cache.pages) continue;
      for (int slot = max(t * 16, view.lo); slot < min(t * 16 + 16, view.hi); ++slot) {
        const uint8_t* p = g.cache.v + (((long long)id * g.cache.heads + w.head) * g.cache.page + (slot & (g.cache.page - 1))) * g.cache.d + j;
        for (int e = 0; e < 8; ++e)
          if ((p[e] & 0x7f) == 0x7f) v[e] = NAN;
      }
    }
  }
}

// kv_attention_tc.cu: the rows of sequences with many.  g.tiles counts tiles of TC_ROWS rows.  sort: the order of the CTAs
// matters.
constexpr int TC_ROWS = 256;
int launch_attention_tc(const AttArgs& g, long long ctas, bool sort, cudaStream_t stream);
int setup_attention_tc();

}  // namespace kv
}  // namespace b200
