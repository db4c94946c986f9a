// Appending keys and values to the paged 8-bit cache (kv_common.cuh), the norm and rotation of the keys on the way, and
// the new tokens' queries normed and rotated by the same launch; and reading blocks of the cache back.
//
//   kv_append_kernel  one CTA per (sequence, page that its new tokens touch, some heads, keys or values), a head's block
//                     after another: it holds all new rows of the block in registers, takes their largest magnitude,
//                     settles the block's scale and writes the codes, so that each input is read once and no other CTA
//                     ever touches the block.  A block whose scale grows under earlier rows has these moved to the new
//                     scale, a power-of-two step.  Further CTAs take the queries, one more looks for sequences that do
//                     not fit.  A page's scale starts anew with its first row.
//                     Bound by instruction issue (two thirds of the cycles issue) and by the latencies of a block's CTA
//                     (bounds, page, rows, the largest of all rows, codes), which three CTAs an SM overlap.  9 prompts of 130
//                     to 1900 tokens, 10117 in all, 32 query and 8 key heads of 128, pages of 64, f16: 58 us, 3.9 TB/s; one
//                     token of 64 sequences: 4.1 us, mostly the launch.
//   kv_read_kernel    codes times scale, 8 codes a thread and step; bound by HBM: 512 pages of 64 slots, 8 heads of 128, to f16:
//                     38 us, 5.3 TB/s.
// Which (sequence, page) a CTA has follows from cu_tokens alone: a sequence that ends at token e can touch at most
// m / page + 2 pages, so the CTAs from cu[s] / page + 2 s on are its own and those behind its last page return.  No
// launch plan is made on the host, which does not know the lengths.
#include "head_transform.cuh"
#include "kv_common.cuh"

namespace b200 {

namespace {

using namespace heads;
using namespace kv;

struct AppendArgs {
  Transform t;
  Cache cache;
  Batch batch;
  int heads_each;                  // heads that a CTA of keys or values takes one after another
  unsigned k_ctas, v_ctas;         // candidates (sequence, page) * groups of heads; the CTAs behind take queries
  int q_heads, per_token;
  int axes;
  const int* pos;                  // axes x tokens, or nullptr: the token's slot on every axis
  const void *q, *k, *v;
  void* q_out;
  long long qt, kt, vt, qot;       // element strides of the token and head axes
  int qh, kh, vh, qoh;
  const void *q_gain, *k_gain;
  int* status;
};

// The last sequence s with key(cu[s], s) <= what, key rising with s, and its bounds: a warp looks at 32 at a time, so that up
// to 31 sequences cost one read's latency (a thread's bisection costs one for every halving).
template <typename Key>
__device__ __forceinline__ Seq find_seq(const AppendArgs& g, long long what, Key key, int& s) {
  const int lane = threadIdx.x & 31, n = g.batch.seqs;
  int lo = 0, span = n;                                    // among [lo, lo + span)
  while (span > 31) {
    const int stride = (span + 31) / 32, at = lo + lane * stride;
    const bool le = at < lo + span && key(__ldg(g.batch.cu + min(at, n)), at) <= what;
    const int count = __popc(__ballot_sync(0xffffffffu, le));
    const int from = lo + max(count - 1, 0) * stride;
    span = min(stride, lo + span - from);
    lo = from;
  }
  const int at = min(lo + lane, n);
  const int cu = __ldg(g.batch.cu + at), len = __ldg(g.batch.lens + min(at, n - 1));
  const bool le = lane < span && key(cu, at) <= what;
  const int pick = max(__popc(__ballot_sync(0xffffffffu, le)) - 1, 0);
  s = lo + pick;
  Seq q;
  q.first = __shfl_sync(0xffffffffu, cu, pick);
  q.m = __shfl_sync(0xffffffffu, cu, pick + 1) - q.first;
  q.len = __shfl_sync(0xffffffffu, len, pick);
  q.ok = fits(g.batch, g.cache, q) && q.m <= q.len;
  return q;
}

template <typename T, int LPR, bool INTER, bool VEC, int NT>
__device__ __forceinline__ void append_queries(const AppendArgs& g, unsigned cta, float2* table) {
  constexpr int GROUPS = NT / LPR, U = !VEC ? 1 : sizeof(T) == 2 ? 4 : 2;      // rows on their way per group
  __shared__ int slots[GROUPS];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR, pairs = g.t.pairs;
  const Lane<T, 4, INTER, VEC> ln(lane, g.cache.d, pairs);
  const int per_cta = GROUPS / g.per_token, first = group % g.per_token, mine = group / g.per_token, step = g.per_token;
  const int t0 = (int)cta * per_cta, tok = t0 + mine, heads = g.q_heads;
  const int tc = min(tok, g.batch.tokens - 1);
  const T* q = reinterpret_cast<const T*>(g.q) + tc * g.qt;
  T* qo = reinterpret_cast<T*>(g.q_out) + tc * g.qot;
  const float inv_d = 1.f / (float)g.cache.d;
  Raw<T, 4, VEC> raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    ln.clear(raw[u]);
    ln.load(q + (long long)min(u * step + first, heads - 1) * g.qh, raw[u]);
  }
  // The tokens' slots in their sequences; -1 for a token of no sequence.  Where sequence i has token i alone, as in a batch
  // without padding, one read finds them.
  bool direct = g.batch.max_new == 1 && g.batch.tokens == g.batch.seqs;
  if (direct) {
    bool mine_is = true;
    if (threadIdx.x < per_cta && t0 + (int)threadIdx.x < g.batch.tokens) {
      const Seq q = load_seq(g.batch, g.cache, t0 + threadIdx.x);
      mine_is = q.m == 1 && q.first == t0 + (int)threadIdx.x;
      slots[threadIdx.x] = q.ok && q.len > 0 ? q.len - 1 : -1;
    } else if (threadIdx.x < per_cta) {
      slots[threadIdx.x] = -1;
    }
    direct = __syncthreads_and(mine_is);
  }
  if (!direct) {
    for (int i = threadIdx.x >> 5; i < per_cta; i += NT / 32) {
      int s;
      const int at = t0 + i;
      const Seq q = find_seq(g, at, [](int cu, int) { return (long long)cu; }, s);
      if ((threadIdx.x & 31) == 0) slots[i] = at < g.batch.tokens && q.ok && at >= q.first && at < q.first + q.m ? q.len - q.m + (at - q.first) : -1;
    }
    __syncthreads();
  }
  const Row<4> gain = ln.gain(g.q_gain);
  fill_table<NT>(g.t, table, per_cta, [&](int i) { return place_of(g.pos, g.axes, g.batch.tokens, min(t0 + i, g.batch.tokens - 1), slots[i]); });
  __syncthreads();
  const bool on = slots[mine] >= 0;                        // a token of no sequence is left alone
  const Coef<4> k = coef(angle_from<4>(table + mine * pairs, ln.j0, on ? pairs : 0), gain);
  for (int r0 = 0;;) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * step + first;
      const Row<4> y = transformed<4, LPR, VEC>(ln.row(raw[u]), k, g.t, ln.j0, inv_d);
      if (on && r < heads) ln.store(qo + (long long)r * g.qoh, y);
    }
    r0 += U * step;
    if (r0 >= heads) break;
#pragma unroll
    for (int u = 0; u < U; ++u) ln.load(q + (long long)min(r0 + u * step + first, heads - 1) * g.qh, raw[u]);
  }
}

// A lane's eight values of a row to their codes: words where the rows may be written in vectors.
template <typename T, bool INTER, bool VEC>
__device__ __forceinline__ void store_codes(const Lane<T, 4, INTER, VEC>& ln, uint8_t* row, const Row<4>& x, float inv) {
  float u[4], v[4];
  ln.values(x, u, v);
  const uint32_t cu = codes4(u, inv), cv = codes4(v, inv);
  if constexpr (!VEC) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (ln.has(e)) {
        row[ln.at(e)] = (uint8_t)(cu >> (8 * e));
        row[ln.at(4 + e)] = (uint8_t)(cv >> (8 * e));
      }
  } else if (ln.live) {
    *reinterpret_cast<uint32_t*>(row + ln.off_u) = cu;
    *reinterpret_cast<uint32_t*>(row + ln.off_v) = cv;
  }
}
template <typename T, bool INTER, bool VEC>
__device__ __forceinline__ float top_of(const Lane<T, 4, INTER, VEC>& ln, const Row<4>& x) {
  float u[4], v[4], top = 0.f;
  ln.values(x, u, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(finite_abs(u[e]), finite_abs(v[e])));
  return top;
}

// NT threads; ROWS: new rows of a block that a group of lanes holds, at most page / (NT / LPR) rounded up.
template <typename T, int LPR, bool INTER, bool VEC, int NT, int ROWS>
__global__ void __launch_bounds__(NT, NT == 256 ? (ROWS * sizeof(T) <= 8 && VEC ? 3 : 2) : 8) kv_append_kernel(const __grid_constant__ AppendArgs g) {
  extern __shared__ float2 table[];                        // cos and sin: new rows of the block (tokens of the CTA) x pairs
  if (blockIdx.x == gridDim.x - 1) {                       // reports every sequence that does not fit, visited below or not
    for (int i = threadIdx.x; i < g.batch.seqs; i += NT) {
      const Seq q = load_seq(g.batch, g.cache, i);
      if (!q.ok || q.m > q.len) flag_index(g.status);
    }
    return;
  }
  if (blockIdx.x >= g.k_ctas + g.v_ctas) {
    append_queries<T, LPR, INTER, VEC, NT>(g, blockIdx.x - g.k_ctas - g.v_ctas, table);
    return;
  }
  constexpr int GROUPS = NT / LPR;
  constexpr bool AHEAD = VEC && ROWS * sizeof(T) <= 16;    // registers for the next head's rows beside this one's
  __shared__ float warp_top[2][NT / 32];
  const bool values = blockIdx.x >= g.k_ctas;
  const int per_unit = (g.cache.heads + g.heads_each - 1) / g.heads_each;
  const unsigned at = blockIdx.x - (values ? g.k_ctas : 0);
  const int unit = (int)(at / (unsigned)per_unit), head0 = (int)(at % (unsigned)per_unit) * g.heads_each;
  const int head1 = min(head0 + g.heads_each, g.cache.heads);
  const int page = g.cache.page, shift = g.cache.page_log2;
  // unit -> (sequence, which of its touched pages)
  int s, nth;
  Seq q;
  if (g.batch.max_new == 1) {
    s = unit;
    nth = 0;
    q = load_seq(g.batch, g.cache, s);
    q.ok = q.ok && q.m <= q.len;
  } else {
    q = find_seq(g, unit, [shift](int cu, int i) { return (long long)(cu >> shift) + 2ll * i; }, s);
    nth = unit - ((q.first >> shift) + 2 * s);
  }
  if (!q.ok || q.m == 0 || nth < 0) return;
  const int start = q.len - q.m, col = (start >> shift) + nth;
  const int slot0 = max(start, col << shift), slot1 = min(q.len, (col + 1) << shift);
  if (slot0 >= slot1) return;                              // behind the sequence's last page
  const int id = __ldg(g.batch.table + (long long)s * g.batch.table_stride + col);
  const int rows = slot1 - slot0, row0 = slot0 & (page - 1), tok0 = q.first + (slot0 - start), pairs = g.t.pairs;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const Lane<T, 4, INTER, VEC> ln(lane, g.cache.d, pairs);
  const float inv_d = 1.f / (float)g.cache.d;
  const T* src = values ? reinterpret_cast<const T*>(g.v) + tok0 * g.vt : reinterpret_cast<const T*>(g.k) + tok0 * g.kt;
  const long long step = values ? g.vt : g.kt;
  const int hs = values ? g.vh : g.kh;
  const bool change = !values && (g.t.normalize || pairs);
  Raw<T, 4, VEC> raw[ROWS];
  auto load = [&](int head) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i)                         // groups without a row take the last one again
      if (i * GROUPS < rows) ln.load(src + (long long)head * hs + min(group + i * GROUPS, rows - 1) * step, raw[i]);
  };
#pragma unroll
  for (int i = 0; i < ROWS; ++i) ln.clear(raw[i]);
  load(head0);                                             // on their way while the page is looked up
  if (id < 0 || id >= g.cache.pages) {
    if (threadIdx.x == 0) flag_index(g.status);
    return;
  }
  Row<4> gain;
  if (change) {
    gain = ln.gain(g.k_gain);
    fill_table<NT>(g.t, table, rows, [&](int i) { return place_of(g.pos, g.axes, g.batch.tokens, tok0 + i, slot0 + i); });
    __syncthreads();
  }
  for (int head = head0; head < head1; ++head) {
    const long long block = (long long)id * g.cache.heads + head;
    float* scale = (values ? g.cache.v_scale : g.cache.k_scale) + block;
    uint8_t* codes = (values ? g.cache.v : g.cache.k) + block * page * g.cache.d;
    const float old = row0 ? *scale : 0.f;
    if (!AHEAD && head > head0) load(head);
    Row<4> x[ROWS];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if (i * GROUPS >= rows) break;                       // the same in every group: the sums inside stay whole
      x[i] = ln.row(raw[i]);
      if (change) {
        const Angle<4> t = angle_from<4>(table + min(group + i * GROUPS, rows - 1) * pairs, ln.j0, pairs);
        x[i] = transformed<4, LPR, VEC>(x[i], coef(t, gain), g.t, ln.j0, inv_d);
      }
      top = fmaxf(top, top_of(ln, x[i]));
    }
    if (AHEAD && head + 1 < head1) load(head + 1);
    top = warp_max(top);
    float* tops = warp_top[head & 1];                      // two sets: the next head's may be written before all have read
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) top = fmaxf(top, tops[w]);
    const float fresh = pow2(scale_exp(top));
    const float now = fmaxf(old, fresh), inv = 1.f / now;  // powers of two: exact
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = group + i * GROUPS;
      if (r < rows) store_codes(ln, codes + (long long)(row0 + r) * g.cache.d, x[i], inv);
    }
    if (now == old) continue;
    if (row0) {                                            // the block's other rows move to the new scale
      const float ratio = old * inv;
      const int words = g.cache.d / 4;
      for (int i = threadIdx.x; i < page * words; i += NT) {
        const int r = i / words;
        if (r >= row0 && r < row0 + rows) continue;
        uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
        const uint2 x4 = values4(*w);
        const float2 f = halves(x4.x), h = halves(x4.y);
        const float v[4] = {f.x, f.y, h.x, h.y};
        *w = codes4(v, ratio);
      }
    }
    if (threadIdx.x == 0) *scale = now;                    // read by all before the barrier
  }
}

// Block i of the output is page pages[i]: (heads, page, d) values.  One CTA per block of one head and keys or values.
template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(const Cache c, const int* __restrict__ pages, T* __restrict__ k_out,
                                                      T* __restrict__ v_out, int* status) {
  const bool values = blockIdx.x & 1;
  const unsigned blk = blockIdx.x >> 1, head = blk % (unsigned)c.heads;
  const int id = pages[blk / (unsigned)c.heads];
  const int chunks = c.page * c.d / 8;                     // of 8 codes
  T* out = (values ? v_out : k_out) + (long long)blk * c.page * c.d;
  const bool ok = id >= 0 && id < c.pages;
  const long long from = (long long)(ok ? id : 0) * c.heads + head;
  const uint2* codes = reinterpret_cast<const uint2*>((values ? c.v : c.k) + from * c.page * c.d);
  const float scale = ok ? (values ? c.v_scale : c.k_scale)[from] : 0.f;
  if (!ok && threadIdx.x == 0) flag_index(status);
#pragma unroll 4
  for (int i = threadIdx.x; i < chunks; i += 256) {
    const uint2 x = ok ? codes[i] : make_uint2(0, 0);
    const uint2 lo = values4(x.x), hi = values4(x.y);
    const float2 a = halves(lo.x), b = halves(lo.y), e = halves(hi.x), f = halves(hi.y);
    if constexpr (sizeof(T) == 2) {
      reinterpret_cast<uint4*>(out)[i] = make_uint4(half2_of(a.x * scale, a.y * scale), half2_of(b.x * scale, b.y * scale),
                                                    half2_of(e.x * scale, e.y * scale), half2_of(f.x * scale, f.y * scale));
    } else {
      reinterpret_cast<float4*>(out)[2 * i] = make_float4(a.x * scale, a.y * scale, b.x * scale, b.y * scale);
      reinterpret_cast<float4*>(out)[2 * i + 1] = make_float4(e.x * scale, e.y * scale, f.x * scale, f.y * scale);
    }
  }
}

// One new token a sequence: two warps have a row and a block to themselves.  Otherwise 256 threads hold a block's rows, up
// to 4 (f16, pages of up to 64) or 8 a group of lanes.
constexpr int NT_ONE = 64, NT_MANY = 256;

template <typename T, int LPR, bool INTER, bool VEC, int NT, int ROWS>
int launch_rows(const AppendArgs& g, unsigned grid, cudaStream_t stream) {
  const int rows = NT == NT_ONE ? 1 : g.cache.page, tokens = NT / LPR;
  const size_t smem = (size_t)(rows > tokens ? rows : tokens) * g.t.pairs * sizeof(float2);
  if (smem > 40 << 10) {                                   // 64 KB at most: pages of 128, heads of 128
    const int rc = note_cuda_error(cudaFuncSetAttribute(kv_append_kernel<T, LPR, INTER, VEC, NT, ROWS>,
                                                        cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "cudaFuncSetAttribute(cache append)");
    if (rc) return rc;
  }
  kv_append_kernel<T, LPR, INTER, VEC, NT, ROWS><<<grid, NT, smem, stream>>>(g);
  count_launch(false);
  return note_cuda_error(cudaGetLastError(), "cache append launch");
}
template <typename T, int LPR, bool INTER, bool VEC>
int launch_page(const AppendArgs& g, unsigned grid, cudaStream_t stream) {
  constexpr int MOST = 128 * LPR / NT_MANY;                // rows of a group with the largest page
  if (g.batch.max_new == 1) return launch_rows<T, LPR, INTER, VEC, NT_ONE, 1>(g, grid, stream);
  if (g.cache.page * LPR / NT_MANY > MOST / 2) return launch_rows<T, LPR, INTER, VEC, NT_MANY, MOST>(g, grid, stream);
  return launch_rows<T, LPR, INTER, VEC, NT_MANY, MOST / 2>(g, grid, stream);
}
template <typename T>
int launch_type(const AppendArgs& g, int lpr, bool inter, bool vec, unsigned grid, cudaStream_t stream) {
  if (!vec)                                                // rows that cannot be moved four elements at a time
    return inter ? launch_page<T, 16, true, false>(g, grid, stream) : launch_page<T, 16, false, false>(g, grid, stream);
  if (lpr == 8) return inter ? launch_page<T, 8, true, true>(g, grid, stream) : launch_page<T, 8, false, true>(g, grid, stream);
  return inter ? launch_page<T, 16, true, true>(g, grid, stream) : launch_page<T, 16, false, true>(g, grid, stream);
}

}  // namespace

// Strides are [token, head] in elements.
int kv_cache_append(int dtype, const b200_kv_cache* cache, const b200_kv_batch* batch, const b200_head_op* op, int64_t q_heads,
                    const void* q, const int64_t qs[2], const void* k, const int64_t ks[2], const void* v, const int64_t vs[2],
                    const int32_t* positions, void* q_out, const int64_t qos[2], cudaStream_t stream) {
  AppendArgs g;
  int rc = parse_cache(cache, &g.cache);
  if (rc) return rc;
  if ((rc = parse_batch(batch, &g.batch))) return rc;
  static const b200_head_op plain = {};
  if (!op) op = &plain;
  if ((rc = parse(op, cache->d, &g.t, &g.axes))) return rc;
  if (g.batch.seqs == 0 || g.batch.tokens == 0 || g.batch.max_new == 0) return B200_OK;
  if (!k || !v) return B200_ERR_NULL;
  const DeviceState* ds = device_state();
  if (!ds) return note_cuda_error(cudaErrorInitializationError, "b200_init not called on this device");
  const int64_t es = dtype == B200_F32 ? 4 : 2;
  g.q_heads = q ? (int)q_heads : 0;
  g.pos = positions;
  g.q = q; g.k = k; g.v = v; g.q_out = q_out;
  if (qs[1] > 0x7fffffff || ks[1] > 0x7fffffff || vs[1] > 0x7fffffff || qos[1] > 0x7fffffff) return B200_ERR_LIMIT;
  g.qt = qs[0]; g.qh = (int)qs[1]; g.kt = ks[0]; g.kh = (int)ks[1];
  g.vt = vs[0]; g.vh = (int)vs[1]; g.qot = qos[0]; g.qoh = (int)qos[1];
  g.q_gain = op->q_gain; g.k_gain = op->k_gain;
  g.status = ds->status;
  const bool inter = op->interleaved != 0;
  bool vec = g.t.pairs % 4 == 0 && vec_ok(4, es, k, 0, ks[0], ks[1]) && vec_ok(4, es, v, 0, vs[0], vs[1]);
  if (g.q_heads) vec = vec && vec_ok(4, es, q, 0, qs[0], qs[1]) && vec_ok(4, es, q_out, 0, qos[0], qos[1]);
  const int lpr = vec && g.cache.d <= 64 ? 8 : 16, groups = (g.batch.max_new == 1 ? NT_ONE : NT_MANY) / lpr;
  // a sequence's m new tokens touch at most (m - 1) / page + 2 pages, one token only one
  const int64_t units = g.batch.max_new == 1 ? g.batch.seqs : (int64_t)(g.batch.tokens >> g.cache.page_log2) + 2 * (int64_t)g.batch.seqs;
  // A CTA takes several heads: its look-ups and the rows' sines serve them all, and the next head's rows load under this one's
  // work.  As long as the keys alone leave a CTA for every SM, beside which the queries' run: 58 us for the 9 prompts, with
  // two for every SM 61, half a one 58; 4.1, 4.5 and 5.0 for one token of 64 sequences; 57, 60 and 73 for 3 prompts of 500
  // to 2000 tokens with 32 key heads.  Without queries two for every SM: 29 us, with one 36, three 31 for the 9 prompts.
  const int64_t least = g.q_heads ? ds->sm_count : 2 * (int64_t)ds->sm_count;
  g.heads_each = 1;
  while (g.heads_each < g.cache.heads && units * ((g.cache.heads + 2 * g.heads_each - 1) / (2 * g.heads_each)) >= least) g.heads_each *= 2;
  const int64_t k_ctas = units * ((g.cache.heads + g.heads_each - 1) / g.heads_each), v_ctas = k_ctas;
  const bool one = g.batch.max_new == 1;
  g.per_token = groups_per_token(g.batch.tokens, g.q_heads, groups, (int64_t)ds->sm_count * (one ? 8 : 3), !vec ? 1 : es == 4 ? 2 : 4, false);
  const int64_t per_cta = groups / g.per_token, q_ctas = g.q_heads ? (g.batch.tokens + per_cta - 1) / per_cta : 0;
  if (units > 0x7fffffff || k_ctas + v_ctas + q_ctas >= 0x7fffffff) return B200_ERR_LIMIT;
  g.k_ctas = (unsigned)k_ctas;
  g.v_ctas = (unsigned)v_ctas;
  const unsigned grid = (unsigned)(k_ctas + v_ctas + q_ctas + 1);
  return dtype == B200_F32 ? launch_type<float>(g, lpr, inter, vec, grid, stream) : launch_type<__half>(g, lpr, inter, vec, grid, stream);
}

int kv_cache_read(int dtype, const b200_kv_cache* cache, int64_t n, const int32_t* pages, void* k_out, void* v_out, cudaStream_t stream) {
  Cache c;
  const int rc = parse_cache(cache, &c);
  if (rc) return rc;
  if (n == 0) return B200_OK;
  const DeviceState* ds = device_state();
  if (!ds) return note_cuda_error(cudaErrorInitializationError, "b200_init not called on this device");
  const int64_t ctas = 2 * n * c.heads;
  if (ctas > 0x7fffffff) return B200_ERR_LIMIT;
  if (dtype == B200_F32) kv_read_kernel<float><<<(unsigned)ctas, 256, 0, stream>>>(c, pages, (float*)k_out, (float*)v_out, ds->status);
  else kv_read_kernel<__half><<<(unsigned)ctas, 256, 0, stream>>>(c, pages, (__half*)k_out, (__half*)v_out, ds->status);
  count_launch(false);
  return note_cuda_error(cudaGetLastError(), "cache read launch");
}

}  // namespace b200
