// Appending keys and values to the paged 8-bit cache (kv_common.cuh), the norm and rotation of the keys on the way, and
// the new tokens' queries normed and rotated by the same launch; and reading blocks of the cache back.
//
//   kv_append_kernel  one CTA per (sequence, page that its new tokens touch, head, keys or values): it holds all new rows
//                     of the block in registers, takes their largest magnitude, settles the block's scale and writes
//                     the codes, so that each input is read once and no other CTA ever touches the block.  A block
//                     whose scale grows under earlier rows has these moved to the new scale, a power-of-two step.
//                     Further CTAs take the queries.  A page's scale starts anew with its first row.
//   kv_read_kernel    codes times scale, 16 codes a thread.
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
  constexpr int GROUPS = THREADS / LPR, U = 2;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const Lane<INTER, VEC> ln(lane, g.cache.d, g.t.pairs);
  const int per_cta = GROUPS / g.per_token, first = group % g.per_token;
  const int tok = (int)cta * per_cta + group / g.per_token;
  Turns turns;
  turns.init(g.t, ln.j0);
  bool on = tok < g.batch.tokens;
  int slot = 0;
  if (on && !(g.pos && g.t.pairs)) {
    const int s = g.batch.max_new == 1 && g.batch.tokens == g.batch.seqs ? tok : owner_of(g.batch.cu, g.batch.seqs, tok);
    const Seq q = load_seq(g.batch, g.cache, s);
    on = q.ok && tok >= q.first && tok < q.first + q.m;    // a token of no sequence is left alone
    slot = q.len - q.m + (tok - q.first);
  } else if (on) {
    const int s = owner_of(g.batch.cu, g.batch.seqs, tok);
    on = tok >= g.batch.cu[s] && tok < g.batch.cu[s + 1];
  }
  const bool own_pos = g.pos && on;
  const int p0 = own_pos ? g.pos[tok] : slot;
  const int p1 = own_pos && g.axes > 1 ? g.pos[g.batch.tokens + tok] : p0;
  const int p2 = own_pos && g.axes > 2 ? g.pos[2 * g.batch.tokens + tok] : p0;
  on = on && ln.live;
  float ga[4], gb[4], c[4], s[4];
  const T* gain = reinterpret_cast<const T*>(g.q_gain);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    ga[e] = gain && ln.has(e) ? to_f(gain[ln.at(e)]) : 1.f;
    gb[e] = gain && ln.has(e) ? to_f(gain[ln.at(4 + e)]) : 1.f;
  }
  const T* q = reinterpret_cast<const T*>(g.q) + tok * g.qt;
  T* qo = reinterpret_cast<T*>(g.q_out) + tok * g.qot;
  const float inv_d = 1.f / (float)g.cache.d;
  bool turned = false;
  for (int r0 = first; r0 - first < g.q_heads; r0 += U * g.per_token) {
    float a[U][4], b[U][4];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * g.per_token;
#pragma unroll
      for (int e = 0; e < 4; ++e) a[u][e] = b[u][e] = 0.f;
      if (on && r < g.q_heads) ln.load(q + r * g.qh, a[u], b[u]);
    }
    if (!turned) {
      turns.at(p0, p1, p2, c, s);
      turned = true;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int r = r0 + u * g.per_token;
      if (g.t.normalize) {
        const float rs = rsqrtf(group_sum<LPR>(sum8(a[u], b[u], a[u], b[u])) * inv_d + g.t.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) { a[u][e] *= rs * ga[e]; b[u][e] *= rs * gb[e]; }
      }
      turn<false>(a[u], b[u], c, s, g.t.pairs - ln.j0);
      if (on && r < g.q_heads) ln.store(qo + r * g.qoh, a[u], b[u]);
    }
  }
}

// Four values of a row to their codes: a word where the rows may be written in vectors.
template <bool INTER, bool VEC>
__device__ __forceinline__ void store_codes(const Lane<INTER, VEC>& ln, uint8_t* row, const float (&a)[4], const float (&b)[4], float inv) {
  if constexpr (VEC) {
    if constexpr (INTER) {
      const float u[4] = {a[0], b[0], a[1], b[1]}, v[4] = {a[2], b[2], a[3], b[3]};
      *reinterpret_cast<uint2*>(row + ln.off_u) = make_uint2(codes4(u, inv), codes4(v, inv));
    } else {
      *reinterpret_cast<uint32_t*>(row + ln.off_u) = codes4(a, inv);
      *reinterpret_cast<uint32_t*>(row + ln.off_v) = codes4(b, inv);
    }
  } else {
    const uint32_t x = codes4(a, inv), y = codes4(b, inv);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (ln.has(e)) {
        row[ln.at(e)] = (uint8_t)(x >> (8 * e));
        row[ln.at(4 + e)] = (uint8_t)(y >> (8 * e));
      }
  }
}

template <typename T, int LPR, bool INTER, bool VEC>
__global__ void __launch_bounds__(THREADS) kv_append_kernel(const AppendArgs g) {
  if (blockIdx.x >= g.block_ctas) {
    append_queries<T, LPR, INTER, VEC>(g, blockIdx.x - g.block_ctas);
    return;
  }
  constexpr int GROUPS = THREADS / LPR;
  constexpr int ROWS = 128 / GROUPS;                       // rows a group can hold: a page has at most 128
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
  float a[ROWS][4], b[ROWS][4];
  float top = 0.f;
  const T* base = values ? reinterpret_cast<const T*>(g.v) + head * g.vh : reinterpret_cast<const T*>(g.k) + head * g.kh;
  const long long step = values ? g.vt : g.kt;
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = group + i * GROUPS;
#pragma unroll
    for (int e = 0; e < 4; ++e) a[i][e] = b[i][e] = 0.f;
    if (r < rows && ln.live) ln.load(base + (tok0 + r) * step, a[i], b[i]);
  }
  if (!values && (g.t.normalize || g.t.pairs)) {
    Turns turns;
    turns.init(g.t, ln.j0);
    float ga[4], gb[4];
    const T* gain = reinterpret_cast<const T*>(g.k_gain);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      ga[e] = gain && ln.has(e) ? to_f(gain[ln.at(e)]) : 1.f;
      gb[e] = gain && ln.has(e) ? to_f(gain[ln.at(4 + e)]) : 1.f;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = group + i * GROUPS;
      if (i * GROUPS >= rows) break;                       // the same in every group: the sums below stay whole
      if (g.t.normalize) {
        const float rs = rsqrtf(group_sum<LPR>(sum8(a[i], b[i], a[i], b[i])) * inv_d + g.t.eps);
#pragma unroll
        for (int e = 0; e < 4; ++e) { a[i][e] *= rs * ga[e]; b[i][e] *= rs * gb[e]; }
      }
      if (g.t.pairs) {
        float c[4], sn[4];
        const int tok = tok0 + min(r, rows - 1);
        const int p0 = g.pos ? g.pos[tok] : slot0 + r;
        const int p1 = g.pos && g.axes > 1 ? g.pos[g.batch.tokens + tok] : p0;
        const int p2 = g.pos && g.axes > 2 ? g.pos[2 * g.batch.tokens + tok] : p0;
        turns.at(p0, p1, p2, c, sn);
        turn<false>(a[i], b[i], c, sn, g.t.pairs - ln.j0);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    if (group + i * GROUPS >= rows || !ln.live) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(finite_abs(a[i][e]), finite_abs(b[i][e])));
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
    if (r < rows && ln.live) store_codes(ln, codes + (long long)(row0 + r) * g.cache.d, a[i], b[i], inv);
  }
  if (now != old) {
    if (row0) {                                            // the block's other rows move to the new scale
      const float ratio = old * inv;
      const int words = g.cache.d / 4;
      for (int i = threadIdx.x; i < page * words; i += THREADS) {
        const int r = i / words;
        if (r >= row0 && r < row0 + rows) continue;
        uint32_t* w = reinterpret_cast<uint32_t*>(codes) + i;
        const uint32_t x = *w, lo = values2(x), hi = values2(x >> 16);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo));
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        const float v[4] = {f.x, f.y, h.x, h.y};
        *w = codes4(v, ratio);
      }
    }
    if (threadIdx.x == 0) *scale = now;
  }
}

// Block i of the output is page pages[i]: (heads, page, d) values.
template <typename T>
__global__ void __launch_bounds__(256) kv_read_kernel(const Cache c, const int* __restrict__ pages, long long blocks, T* k_out,
                                                      T* v_out, int* status) {
  const int per_block = c.page * c.d / 16;                 // chunks of 16 codes
  const long long chunks = blocks * per_block;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < 2 * chunks; i += (long long)gridDim.x * blockDim.x) {
    const bool values = i >= chunks;
    const long long j = values ? i - chunks : i, blk = j / per_block;
    const int at = (int)(j - blk * per_block), head = (int)(blk % c.heads);
    const int id = pages[blk / c.heads];
    uint4 x = make_uint4(0, 0, 0, 0);
    float scale = 0.f;
    if (id >= 0 && id < c.pages) {
      const long long from = (long long)id * c.heads + head;
      x = *reinterpret_cast<const uint4*>((values ? c.v : c.k) + (from * per_block + at) * 16);
      scale = (values ? c.v_scale : c.k_scale)[from];
    } else {
      flag_index(status);
    }
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    T* out = (values ? v_out : k_out) + j * 16;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t lo = values2(w[e]), hi = values2(w[e] >> 16);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo));
      const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
      const float v[4] = {f.x * scale, f.y * scale, h.x * scale, h.y * scale};
      store4(out + 4 * e, v);
    }
  }
}

template <typename T, int LPR>
int launch_append(const AppendArgs& g, bool inter, bool vec, unsigned grid, cudaStream_t stream) {
  if (inter) {
    if (vec) kv_append_kernel<T, LPR, true, true><<<grid, THREADS, 0, stream>>>(g);
    else kv_append_kernel<T, LPR, true, false><<<grid, THREADS, 0, stream>>>(g);
  } else {
    if (vec) kv_append_kernel<T, LPR, false, true><<<grid, THREADS, 0, stream>>>(g);
    else kv_append_kernel<T, LPR, false, false><<<grid, THREADS, 0, stream>>>(g);
  }
  count_launch(false);
  return note_cuda_error(cudaGetLastError(), "cache append launch");
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
  bool vec = (inter || g.t.pairs % 4 == 0) && vec_ok(es, k, ks[0], ks[1]) && vec_ok(es, v, vs[0], vs[1]);
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
  if (dtype == B200_F32)
    return lpr == 8 ? launch_append<float, 8>(g, inter, vec, grid, stream) : launch_append<float, 16>(g, inter, vec, grid, stream);
  return lpr == 8 ? launch_append<__half, 8>(g, inter, vec, grid, stream) : launch_append<__half, 16>(g, inter, vec, grid, stream);
}

int kv_cache_read(int dtype, const b200_kv_cache* cache, int64_t n, const int32_t* pages, void* k_out, void* v_out, cudaStream_t stream) {
  Cache c;
  const int rc = parse_cache(cache, &c);
  if (rc) return rc;
  if (n == 0) return B200_OK;
  const DeviceState* ds = device_state();
  if (!ds) return note_cuda_error(cudaErrorInitializationError, "b200_init not called on this device");
  const int64_t blocks = n * c.heads, work = 2 * blocks * (c.page * c.d / 16);
  int64_t grid = (work + 255) / 256;
  if (grid > (int64_t)ds->sm_count * 32) grid = (int64_t)ds->sm_count * 32;
  if (dtype == B200_F32) kv_read_kernel<float><<<(unsigned)grid, 256, 0, stream>>>(c, pages, blocks, (float*)k_out, (float*)v_out, ds->status);
  else kv_read_kernel<__half><<<(unsigned)grid, 256, 0, stream>>>(c, pages, blocks, (__half*)k_out, (__half*)v_out, ds->status);
  count_launch(false);
  return note_cuda_error(cudaGetLastError(), "cache read launch");
}

}  // namespace b200
