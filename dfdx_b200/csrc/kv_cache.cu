// Appending keys and values to the paged 8-bit cache (kv_common.cuh), the norm and rotation of the keys on the way, and
// the new tokens' queries normed and rotated by the same launch; and reading blocks of the cache back.
//
//   kv_append_kernel  one CTA per (sequence, page that its new tokens touch, head, keys or values): it holds all new rows
//                     of the block in registers, takes their largest magnitude, settles the block's scale and writes
//                     the codes, so that each input is read once and no other CTA ever touches the block.  A block
//                     whose scale grows under earlier rows has these moved to the new scale, a power-of-two step.
//                     Further CTAs take the queries.  A page's scale starts anew with its first row.
//   kv_read_kernel    codes times scale, 8 codes a thread and step.
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
  unsigned block_ctas;             // (sequence, page) candidates * heads * 2; the CTAs behind them take queries
  int q_heads, per_token;
  int axes;
  const int* pos;                  // axes x tokens, or nullptr: the token's slot on every axis
  const void *q, *k, *v;
  void* q_out;
  long long qt, qh, kt, kh, vt, vh, qot, qoh;      // element strides of the token and head axes
  const void *q_gain, *k_gain;
  int* status;
};

constexpr int THREADS = 256;

// The sequence of a new token, by bisection over cu (the last s with cu[s] <= tok).
__device__ __forceinline__ int owner_of(const int* cu, int n, int tok) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= tok) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T, int LPR, bool INTER, bool VEC>
__device__ __forceinline__ void append_queries(const AppendArgs& g, unsigned cta) {
  constexpr int GROUPS = THREADS / LPR, U = !VEC ? 1 : sizeof(T) == 2 ? 4 : 2;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const Lane<INTER, VEC> ln(lane, g.cache.d, g.t.pairs);
  const int per_cta = GROUPS / g.per_token, first = group % g.per_token;
  const int tok = (int)cta * per_cta + group / g.per_token;
  bool on = tok < g.batch.tokens;
  int slot = 0;
  if (on) {
    const int s = g.batch.max_new == 1 && g.batch.tokens == g.batch.seqs ? tok : owner_of(g.batch.cu, g.batch.seqs, tok);
    const Seq q = load_seq(g.batch, g.cache, s);
    on = q.ok && tok >= q.first && tok < q.first + q.m;    // a token of no sequence is left alone
    slot = q.len - q.m + (tok - q.first);
  }
  const Place at = place_of(on ? g.pos : nullptr, g.axes, g.batch.tokens, tok, slot);
  on = on && ln.live;
  const T* q = reinterpret_cast<const T*>(g.q) + tok * g.qt;
  T* qo = reinterpret_cast<T*>(g.q_out) + tok * g.qot;
  const float inv_d = 1.f / (float)g.cache.d;
  Coef k;
  for (int r0 = 0; r0 < g.q_heads; r0 += U * g.per_token) {
    Raw<T, VEC> raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * g.per_token + first;
      ln.clear(raw[u]);
      if (on && r < g.q_heads) ln.load(q + r * g.qh, raw[u]);
    }
    if (r0 == 0) {
      k = coef(angle_at(g.t, ln.j0, at.p0, at.p1, at.p2), ln.gain(reinterpret_cast<const T*>(g.q_gain)));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * g.per_token + first;
      const Row y = transformed<LPR, VEC>(ln.row(raw[u]), k, g.t, ln.j0, inv_d);
      if (on && r < g.q_heads) ln.store(qo + r * g.qoh, y);
    }
  }
}

// A lane's eight values of a row to their codes: words where the rows may be written in vectors.
template <bool INTER, bool VEC>
__device__ __forceinline__ void store_codes(const Lane<INTER, VEC>& ln, uint8_t* row, const Row& x, float inv) {
  float u[4], v[4];
  ln.values(x, u, v);
  const uint32_t cu = codes4(u, inv), cv = codes4(v, inv);
  if constexpr (VEC && INTER) {
    *reinterpret_cast<uint2*>(row + ln.off_u) = make_uint2(cu, cv);
  } else if constexpr (VEC) {
    *reinterpret_cast<uint32_t*>(row + ln.off_u) = cu;
    *reinterpret_cast<uint32_t*>(row + ln.off_v) = cv;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (ln.has(e)) {
        row[ln.at(e)] = (uint8_t)(cu >> (8 * e));
        row[ln.at(4 + e)] = (uint8_t)(cv >> (8 * e));
      }
  }
}
template <bool INTER, bool VEC>
__device__ __forceinline__ float top_of(const Lane<INTER, VEC>& ln, const Row& x) {
  float u[4], v[4], top = 0.f;
  ln.values(x, u, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(finite_abs(u[e]), finite_abs(v[e])));
  return top;
}

// ROWS: rows that a group of lanes holds, page / (THREADS / LPR) rounded up.
template <typename T, int LPR, bool INTER, bool VEC, int ROWS>
__global__ void __launch_bounds__(THREADS, ROWS == 8 || !VEC ? 2 : 3) kv_append_kernel(const AppendArgs g) {
  if (blockIdx.x >= g.block_ctas) {
    append_queries<T, LPR, INTER, VEC>(g, blockIdx.x - g.block_ctas);
    return;
  }
  constexpr int GROUPS = THREADS / LPR;
  __shared__ float warp_top[THREADS / 32];
  const bool values = blockIdx.x & 1;
  const unsigned rest = blockIdx.x >> 1;
  const int head = (int)(rest % (unsigned)g.cache.heads), unit = (int)(rest / (unsigned)g.cache.heads);
  const int page = g.cache.page, shift = g.cache.page_log2;
  // unit -> (sequence, which of its touched pages)
  int s, nth;
  if (g.batch.max_new == 1) {
    s = unit;
    nth = 0;
  } else {
    int lo = 0, hi = g.batch.seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)(g.batch.cu[mid] >> shift) + 2 * mid <= unit) lo = mid;
      else hi = mid - 1;
    }
    s = lo;
    nth = unit - ((g.batch.cu[s] >> shift) + 2 * s);
  }
  const Seq q = load_seq(g.batch, g.cache, s);
  if (!q.ok || q.m > q.len) {
    if (threadIdx.x == 0) flag_index(g.status);
    return;
  }
  if (q.m == 0 || nth < 0) return;
  const int start = q.len - q.m, col = (start >> shift) + nth;
  const int slot0 = max(start, col << shift), slot1 = min(q.len, (col + 1) << shift);
  if (slot0 >= slot1) return;                              // behind the sequence's last page
  const int id = g.batch.table[(long long)s * g.batch.table_stride + col];
  if (id < 0 || id >= g.cache.pages) {
    if (threadIdx.x == 0) flag_index(g.status);
    return;
  }
  const int rows = slot1 - slot0, row0 = slot0 & (page - 1), tok0 = q.first + (slot0 - start);
  const long long block = (long long)id * g.cache.heads + head;
  float* scale = (values ? g.cache.v_scale : g.cache.k_scale) + block;
  uint8_t* codes = (values ? g.cache.v : g.cache.k) + block * page * g.cache.d;
  const float old = row0 ? *scale : 0.f;

  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const Lane<INTER, VEC> ln(lane, g.cache.d, g.t.pairs);
  const float inv_d = 1.f / (float)g.cache.d;
  const T* base = values ? reinterpret_cast<const T*>(g.v) + head * g.vh : reinterpret_cast<const T*>(g.k) + head * g.kh;
  const long long step = values ? g.vt : g.kt;
  Raw<T, VEC> raw[ROWS];
  Row x[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = group + i * GROUPS;
    ln.clear(raw[i]);
    if (r < rows && ln.live) ln.load(base + (tok0 + r) * step, raw[i]);
  }
  const bool change = !values && (g.t.normalize || g.t.pairs);
  const Row gain = ln.gain(change ? reinterpret_cast<const T*>(g.k_gain) : nullptr);
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    x[i] = ln.row(raw[i]);
    if (i * GROUPS < rows) {                               // the same in every group: the sums inside stay whole
      const int r = min(group + i * GROUPS, rows - 1);
      if (change) {
        const Place at = place_of(g.pos, g.axes, g.batch.tokens, tok0 + r, slot0 + r);
        x[i] = transformed<LPR, VEC>(x[i], coef(angle_at(g.t, ln.j0, at.p0, at.p1, at.p2), gain), g.t, ln.j0, inv_d);
      }
      top = fmaxf(top, top_of(ln, x[i]));                  // rows behind the last are zeros
    }
  }
  top = group_max<32>(top);
  if ((threadIdx.x & 31) == 0) warp_top[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, warp_top[w]);
  const float fresh = pow2(scale_exp(top));
  const float now = fmaxf(old, fresh), inv = 1.f / now;    // powers of two: exact
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = group + i * GROUPS;
    if (r < rows && ln.live) store_codes(ln, codes + (long long)(row0 + r) * g.cache.d, x[i], inv);
  }
  if (now != old) {
    if (row0) {                                            // the block's other rows move to the new scale
      const float ratio = old * inv;
      const int words = g.cache.d / 4;
      for (int i = threadIdx.x; i < page * words; i += THREADS) {
        const int r = i / words;
        if (r >= row0 && r < row0 + rows) continue;
        uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
        const float2 f = halves(values2(*w)), h = halves(values2(*w >> 16));
        const float v[4] = {f.x, f.y, h.x, h.y};
        *w = codes4(v, ratio);
      }
    }
    if (threadIdx.x == 0) *scale = now;
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
    const float2 a = halves(values2(x.x)), b = halves(values2(x.x >> 16)), e = halves(values2(x.y)), f = halves(values2(x.y >> 16));
    if constexpr (sizeof(T) == 2) {
      reinterpret_cast<uint4*>(out)[i] = make_uint4(half2_of(a.x * scale, a.y * scale), half2_of(b.x * scale, b.y * scale),
                                                    half2_of(e.x * scale, e.y * scale), half2_of(f.x * scale, f.y * scale));
    } else {
      reinterpret_cast<float4*>(out)[2 * i] = make_float4(a.x * scale, a.y * scale, b.x * scale, b.y * scale);
      reinterpret_cast<float4*>(out)[2 * i + 1] = make_float4(e.x * scale, e.y * scale, f.x * scale, f.y * scale);
    }
  }
}

template <typename T, int LPR, bool INTER, bool VEC, int ROWS>
int launch_append_rows(const AppendArgs& g, unsigned grid, cudaStream_t stream) {
  kv_append_kernel<T, LPR, INTER, VEC, ROWS><<<grid, THREADS, 0, stream>>>(g);
  count_launch(false);
  return note_cuda_error(cudaGetLastError(), "cache append launch");
}
template <typename T, int LPR, bool INTER>
int launch_append_vec(const AppendArgs& g, bool vec, unsigned grid, cudaStream_t stream) {
  constexpr int MOST = 128 * LPR / THREADS;
  const int rows = g.batch.max_new == 1 ? 1 : g.cache.page * LPR / THREADS;
  if (!vec) return launch_append_rows<T, LPR, INTER, false, MOST>(g, grid, stream);
  if (rows <= 1) return launch_append_rows<T, LPR, INTER, true, 1>(g, grid, stream);
  if (rows <= MOST / 2) return launch_append_rows<T, LPR, INTER, true, MOST / 2>(g, grid, stream);
  return launch_append_rows<T, LPR, INTER, true, MOST>(g, grid, stream);
}

bool vec_ok(int64_t es, const void* p, int64_t t, int64_t h) { return ((uintptr_t)p % (4 * es)) == 0 && t % 4 == 0 && h % 4 == 0; }

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
  g.qt = qs[0]; g.qh = qs[1]; g.kt = ks[0]; g.kh = ks[1]; g.vt = vs[0]; g.vh = vs[1]; g.qot = qos[0]; g.qoh = qos[1];
  g.q_gain = op->q_gain; g.k_gain = op->k_gain;
  g.status = ds->status;
  // a sequence's m new tokens touch at most (m - 1) / page + 2 pages, one token only one
  const int64_t units = g.batch.max_new == 1 ? g.batch.seqs : (int64_t)(g.batch.tokens >> g.cache.page_log2) + 2 * (int64_t)g.batch.seqs;
  const int64_t block_ctas = units * g.cache.heads * 2;
  const bool inter = op->interleaved != 0;
  bool vec = g.t.pairs % 4 == 0 && vec_ok(es, k, ks[0], ks[1]) && vec_ok(es, v, vs[0], vs[1]);
  if (g.q_heads) vec = vec && vec_ok(es, q, qs[0], qs[1]) && vec_ok(es, q_out, qos[0], qos[1]);
  const int lpr = g.cache.d <= 64 ? 8 : 16, groups = THREADS / lpr;
  // groups that share a token's queries, as in the dense norm and rotation
  const int64_t want = (int64_t)ds->sm_count * (2048 / lpr);
  g.per_token = 1;
  while (g.per_token < groups && g.per_token < g.q_heads && (int64_t)g.batch.tokens * g.per_token < want) g.per_token *= 2;
  const int64_t per_cta = groups / g.per_token, q_ctas = g.q_heads ? (g.batch.tokens + per_cta - 1) / per_cta : 0;
  if (units > 0x7fffffff || block_ctas + q_ctas > 0x7fffffff) return B200_ERR_LIMIT;
  g.block_ctas = (unsigned)block_ctas;
  const unsigned grid = (unsigned)(block_ctas + q_ctas);
  if (dtype == B200_F32) {
    if (lpr == 8) return inter ? launch_append_vec<float, 8, true>(g, vec, grid, stream) : launch_append_vec<float, 8, false>(g, vec, grid, stream);
    return inter ? launch_append_vec<float, 16, true>(g, vec, grid, stream) : launch_append_vec<float, 16, false>(g, vec, grid, stream);
  }
  if (lpr == 8) return inter ? launch_append_vec<__half, 8, true>(g, vec, grid, stream) : launch_append_vec<__half, 8, false>(g, vec, grid, stream);
  return inter ? launch_append_vec<__half, 16, true>(g, vec, grid, stream) : launch_append_vec<__half, 16, false>(g, vec, grid, stream);
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
