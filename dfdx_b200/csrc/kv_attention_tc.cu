// Attention of many new tokens over the paged 8-bit cache (prompts and long chunks): bound by the products, on tcgen05.
// The formulas, the value scales in the exponent and the lift are those of kv_attention.cu.
//
// A CTA has 256 rows of one (sequence, key head) -- a row is a new token and one of the query heads that share the key
// head, neighbours in that order -- as two tiles of 128, and walks the slots that some row sees, 128 at a time.
//   warps 0-3, 4-7   softmax of tile 0 and 1: a thread owns a row.  Reads its 128 scores from tensor memory, turns them into
//                    probabilities and writes these as f16 over the scores' own columns: the second product takes its
//                    left operand from there, in the type of the values' tile (2^-12 of each probability, of random sign;
//                    the sums take them in f32).  The outputs stay in tensor memory too; they are read, scaled and
//                    written back only when a row's maximum moves by more than 1.
//   warps 8-11       one thread each issues S = Q K^T (8, 9) or O += P V (10, 11) of a tile, half a tile of slots at a time:
//                    while the softmax has one half, the tensor core multiplies the other's probabilities and puts the
//                    next scores in their place.  (With whole tiles the softmax waited 2500 of 5500 cycles for the two.)
//   warps 12-19      bring the codes: whole 16-byte pieces of a row from global memory into registers, one tile ahead, to
//                    f16 (exact), and into the 128B-swizzled layout that both products read; the blocks' scales beside
//                    them.  TMA cannot: the pages are scattered and the tensor core has no product of f16 with e4m3.
// Tensor memory: scores (and probabilities) 2 x 128 columns, outputs 2 x DP.  Shared memory at DP = 128: Q 64 KB, two
// stages of K and V 128 KB.  Every wait is bounded (tc_device.cuh).
// 37 x 256 tokens over 4352 slots, 16 query heads, one key head of 128: 351 us, 933 TFLOP/s, 0.56 of a library product.  What
// is left is the softmax: its chain of a load from tensor memory, maxima, exponentials (half of it) and the store takes
// 3600 of 4350 cycles that 128 slots take, the tensor core 2800.  At heads of 64, with half the products, the cycles are
// the same (490 TFLOP/s).  Letting the two row tiles' warps take turns at the exponentials made it 839 TFLOP/s, other orders
// of the exponentials, sums and packing changed nothing.
#include "attention_common.cuh"
#include "kv_attention.cuh"

namespace b200 {

namespace {

using namespace tcx;
using namespace kv;
using attn::mbar_wait_warp;
using attn::warp_arrive;

constexpr int THREADS = 640;
constexpr int STAGES = 2;
constexpr int SCALE_SETS = 4;

template <int DP> struct Cfg {
  static constexpr int CH = DP / 64;                       // 64-element chunks of a row
  static constexpr int TILE_BYTES = 128 * DP * 2;          // one Q, K or V tile
  static constexpr int OFF_K = 2 * TILE_BYTES;
  static constexpr int OFF_V = OFF_K + STAGES * TILE_BYTES;
  static constexpr int SMEM_BYTES = OFF_V + STAGES * TILE_BYTES + 1024;
  static constexpr uint32_t TM_S = 0, TM_O = 256;
};
// 640 threads x 96 registers at launch: 2 x 128 x 136 + 128 x 40 + 256 x 80 = 60416 of 61440.
constexpr int REGS_LAUNCH = 96, REGS_SOFTMAX = 136, REGS_ISSUE = 40, REGS_CODES = 80;
static_assert(2 * 128 * REGS_SOFTMAX + 128 * REGS_ISSUE + 256 * REGS_CODES <= THREADS * REGS_LAUNCH, "setmaxnreg budget exceeds the CTA's launch allocation");

// D (tensor memory) (+)= A (tensor memory) * B (shared memory), f16 in, f32 out.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t blo, uint32_t bhi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}"
      ::"r"(d), "r"(a), "r"(blo), "r"(bhi), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};"
      ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
  return r;
}
// Two f32 in one register pair: the scores come out of tensor memory in neighbouring registers.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void split(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

struct TcArgs2 {
  AttArgs a;
  uint32_t flip;                   // a negative alpha: the queries' signs are turned instead, so that every scale is positive
  long long wait_limit;
  bool sorted;                     // CTAs take the row tiles of all sequences with the most slots first
};
constexpr int MOST_SORTED = 256;   // row tiles
// The least factor of a block's scores, also where alpha is 0 or alpha * scale vanishes in f32: a masked score is -infinity
// before it is scaled, and 0 would make NaN of it.  Scores are below 65504 * 448 * 128 < 2^32: this one moves no exponent.
constexpr float MIN_FACTOR = 1.1754944e-38f;               // 2^-126

template <int DP>
__global__ void __launch_bounds__(THREADS, 1) kv_prefill_kernel(const __grid_constant__ TcArgs2 ga) {
  using C = Cfg<DP>;
  const AttArgs& g = ga.a;
  extern __shared__ uint8_t smem_dyn[];
  __shared__ __align__(8) uint64_t bar_q[2], bar_k_full[STAGES], bar_k_empty[STAGES], bar_v_full[STAGES], bar_v_empty[STAGES];
  __shared__ __align__(8) uint64_t bar_s_full[2][2], bar_p_full[2][2], bar_pv_done[2][2];   // per row tile and half of the slots
  __shared__ float4 scales[SCALE_SETS][8];                 // per 16 slots: key scale * alpha log2(e), log2 and reciprocal of the value scale
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag, sh_nan, picked;
  __shared__ __align__(16) int slots_of[MOST_SORTED];

  const uint32_t smem_base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2;
  volatile int* abortp = &abort_flag;
  asm volatile("griddepcontrol.launch_dependents;");

  unsigned unit = blockIdx.x / (unsigned)g.splits;
  const int x = (int)(blockIdx.x % (unsigned)g.splits);
  if (ga.sorted) {
    // CTA b has head b % heads of the row tile that is b / heads-th when all sequences' are put in the order of their
    // slots: the last CTAs to start are then the shortest.  Ties go by index.
    const int n = g.batch.seqs * g.tiles, i = threadIdx.x, want = (int)(unit / (unsigned)g.cache.heads);
    if (i < MOST_SORTED) slots_of[i] = -2;                 // behind all others
    if (i < n) {
      const int s = i / g.tiles, row = i % g.tiles * TC_ROWS;
      const Seq q = load_seq(g.batch, g.cache, s);
      const int rows = q.ok ? q.m * g.group - row : 0;
      slots_of[i] = rows > 0 ? max(view_of(g, q, row + min(rows, TC_ROWS) - 1).hi - view_of(g, q, row).lo, 0) : -1;
    }
    __syncthreads();
    if (i < n) {
      const int mine = slots_of[i];
      int before = 0;
#pragma unroll 4
      for (int j = 0; j < n; j += 4) {
        const int4 v = *reinterpret_cast<const int4*>(&slots_of[j]);
        before += (v.x > mine - (j < i)) + (v.y > mine - (j + 1 < i)) + (v.z > mine - (j + 2 < i)) + (v.w > mine - (j + 3 < i));
      }
      if (before == want) picked = i;
    }
    __syncthreads();
    unit = ((unsigned)(picked / g.tiles) * g.cache.heads + unit % (unsigned)g.cache.heads) * g.tiles + picked % g.tiles;
  } else {                                                 // causal rows at the end of a sequence see the most slots
    unit = unit - unit % (unsigned)g.tiles + ((unsigned)g.tiles - 1 - unit % (unsigned)g.tiles);
  }
  Work w;
  if (!work_of<TC_ROWS>(g, unit, x, w)) return;
  const int ntile = w.rows > 128 ? 2 : 1;
  const int base = w.begin << 4;                           // first slot
  const int T = (w.end - w.begin + 7) / 8;                 // tiles of 128 slots
  const int d = g.cache.d;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&bar_q[t]), 4);
      for (int h = 0; h < 2; ++h) {
        mbar_init(smem_u32(&bar_s_full[t][h]), 1);
        mbar_init(smem_u32(&bar_p_full[t][h]), 4);
        mbar_init(smem_u32(&bar_pv_done[t][h]), 1);
      }
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&bar_k_full[s]), 8);
      mbar_init(smem_u32(&bar_k_empty[s]), ntile);
      mbar_init(smem_u32(&bar_v_full[s]), 8);
      mbar_init(smem_u32(&bar_v_empty[s]), ntile);
    }
    abort_flag = 0;
    sh_nan = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(&tmem_slot), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_slot;

  if (wg == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    const int t = warp & 1;
    if (t < ntile && lane == 0) {
      const uint32_t tm_s = tmem_base + C::TM_S + t * 128, tm_o = tmem_base + C::TM_O + t * 128;
      if (warp < 10) {
        // S = Q K^T, half h of tile j: 64 slots, over the probabilities that were multiplied last
        const uint64_t dk = make_smem_desc(smem_base, 16, 1024, 2);           // K-major tiles (Q, K)
        const uint32_t hi_k = (uint32_t)(dk >> 32);
        const uint32_t q_lo = (uint32_t)dk + (uint32_t)(t * C::TILE_BYTES >> 4), k_lo = (uint32_t)dk + (uint32_t)(C::OFF_K >> 4);
        const uint32_t idesc = (1u << 4) | ((uint32_t)(64 >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        const int ksteps = d / 16;
        bool ok = T > 0 && mbar_wait(smem_u32(&bar_q[t]), 0, abortp, ga.wait_limit);
        for (int j = 0; ok && j < T; ++j) {
          if (!mbar_wait(smem_u32(&bar_k_full[j % STAGES]), (uint32_t)(j / STAGES) & 1u, abortp, ga.wait_limit)) break;
          for (int h = 0; h < 2; ++h) {
            if (j > 0 && !(ok = mbar_wait(smem_u32(&bar_pv_done[t][h]), (uint32_t)(j - 1) & 1u, abortp, ga.wait_limit))) break;
            tc_fence_after();
            const uint32_t klo = k_lo + (uint32_t)((j % STAGES * C::TILE_BYTES + h * 8192) >> 4);
            if (ksteps == DP / 16) {
#pragma unroll
              for (int ks = 0; ks < DP / 16; ++ks) {
                const uint32_t off = (uint32_t)(((ks >> 2) * 16384 + (ks & 3) * 32) >> 4);
                umma_lohi<2>(tm_s + h * 64, q_lo + off, hi_k, klo + off, hi_k, idesc, ks > 0 ? 1u : 0u);
              }
            } else {
              for (int ks = 0; ks < ksteps; ++ks) {
                const uint32_t off = (uint32_t)(((ks >> 2) * 16384 + (ks & 3) * 32) >> 4);
                umma_lohi<2>(tm_s + h * 64, q_lo + off, hi_k, klo + off, hi_k, idesc, ks > 0 ? 1u : 0u);
              }
            }
            umma_commit(smem_u32(&bar_s_full[t][h]));
          }
          if (ok) umma_commit(smem_u32(&bar_k_empty[j % STAGES]));            // one arrival per row tile
        }
      } else {
        // O += P V over the half's slots, 16 per product
        const uint64_t dv = make_smem_desc(smem_base, 16384, 1024, 2);        // MN-major tile (V)
        const uint32_t hi_v = (uint32_t)(dv >> 32), v_lo = (uint32_t)dv + (uint32_t)(C::OFF_V >> 4);
        const uint32_t idesc = (1u << 4) | (1u << 16) | ((uint32_t)(DP >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
        bool ok = true;
        for (int j = 0; ok && j < T; ++j) {
          const int s = j % STAGES;
          if (!mbar_wait(smem_u32(&bar_v_full[s]), (uint32_t)(j / STAGES) & 1u, abortp, ga.wait_limit)) break;
          const uint32_t vlo = v_lo + (uint32_t)(s * (C::TILE_BYTES >> 4));
          for (int h = 0; h < 2; ++h) {
            if (!(ok = mbar_wait(smem_u32(&bar_p_full[t][h]), (uint32_t)j & 1u, abortp, ga.wait_limit))) break;
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
              umma_ts(tm_o, tm_s + h * 64 + ks * 8, vlo + (uint32_t)((h * 4 + ks) * 2048 >> 4), hi_v, idesc, (j > 0 || h > 0 || ks > 0) ? 1u : 0u);
            umma_commit(smem_u32(&bar_pv_done[t][h]));
          }
          if (ok) umma_commit(smem_u32(&bar_v_empty[s]));
        }
      }
    }
    __syncwarp();
  } else if (wg >= 3) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 80;");
    // ---------------------------------------------------------------- codes to f16 tiles
    const int cw = warp - 12;
    const int* table = g.batch.table + (long long)w.s * g.batch.table_stride;
    const int in_page = g.cache.page - 1, shift = g.cache.page_log2;
    const int row0 = cw * 8 + (lane >> 2), c4 = lane & 3;  // rows row0 and row0 + 64; 16-code pieces c4 and c4 + 4 of each
    // pieces that do not exist (d < DP) are zeros, written once
    for (int r = row0; r < 128; r += 64)
      for (int p = c4; p < DP / 16; p += 4)
        if (p * 16 >= d)
          for (int s = 0; s < 2 * STAGES; ++s) {
            const uint32_t row = smem_base + C::OFF_K + s * C::TILE_BYTES + (uint32_t)(p >> 2) * 16384 + (uint32_t)r * 128;
            st_shared_v4_u32(row + ((((uint32_t)p & 3u) * 2 ^ ((uint32_t)r & 7u)) << 4), 0, 0, 0, 0);
            st_shared_v4_u32(row + (((((uint32_t)p & 3u) * 2 + 1) ^ ((uint32_t)r & 7u)) << 4), 0, 0, 0, 0);
          }
    constexpr int PC = (DP / 16 + 3) / 4;                  // pieces of a row that a lane holds: 1 or 2
    uint4 kc[2][PC], vc[2][PC];
    uint32_t bad_groups = 0;
    // Page of the 16-slot group that this warp's rows row0 + 64 i lie in, for tile j; -1 where there is none.
    auto page_of = [&](int j, int i) -> int {
      const int grp = w.begin + j * 8 + i * 4 + (cw >> 1);
      if (grp >= w.end) return -1;
      const int id = __ldg(table + ((grp << 4) >> shift));
      if (id < 0 || id >= g.cache.pages) {
        bad_groups |= 1;
        return -1;
      }
      return id;
    };
    auto load = [&](const uint8_t* codes, int j, uint4 (&to)[2][PC], const int (&id)[2]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int slot = base + j * 128 + row0 + 64 * i;
        const uint8_t* row = codes + (((long long)max(id[i], 0) * g.cache.heads + w.head) * g.cache.page + (slot & in_page)) * d;
#pragma unroll
        for (int p = 0; p < PC; ++p) {
          to[i][p] = make_uint4(0, 0, 0, 0);
          if (id[i] >= 0 && (c4 + 4 * p) * 16 < d) to[i][p] = __ldg(reinterpret_cast<const uint4*>(row) + c4 + 4 * p);
        }
      }
    };
    auto store = [&](uint32_t tile, const uint4 (&from)[2][PC]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t r = (uint32_t)(row0 + 64 * i);
#pragma unroll
        for (int p = 0; p < PC; ++p) {
          if ((c4 + 4 * p) * 16 >= d) continue;
          const uint4 q = from[i][p];
          const uint2 a = values4(q.x), b = values4(q.y), e = values4(q.z), f = values4(q.w);
          const uint32_t row = tile + (uint32_t)p * 16384 + r * 128;
          st_shared_v4_u32(row + ((((uint32_t)c4 * 2) ^ (r & 7u)) << 4), a.x, a.y, b.x, b.y);
          st_shared_v4_u32(row + ((((uint32_t)c4 * 2 + 1) ^ (r & 7u)) << 4), e.x, e.y, f.x, f.y);
        }
      }
    };
    // Scales of the group that lane i < 2 answers for (of rows row0 + 64 i), for the tile whose pages are `id`.
    auto scale_of = [&](const int (&id)[2]) -> float4 {
      float4 sc = make_float4(1.f, -INFINITY, 1.f, 0.f);   // no such slots: their scores count for nothing
      const int p = lane == 0 ? id[0] : id[1];
      if ((cw & 1) == 0 && lane < 2 && p >= 0) {
        const long long blk = (long long)p * g.cache.heads + w.head;
        const uint32_t sv = __float_as_uint(__ldg(g.cache.v_scale + blk));
        sc = make_float4(fmaxf(__ldg(g.cache.k_scale + blk) * g.scale_log2, MIN_FACTOR), (float)((int)(sv >> 23) - 127),
                         __uint_as_float((254u << 23) - sv), 0.f);
      }
      return sc;
    };
    // What a tile needs is asked for a tile ahead, the pages two: their latencies would otherwise add up in every round.
    int id[2], id2[2];
    float4 sc = make_float4(0.f, 0.f, 0.f, 0.f);
    if (T > 0) {
#pragma unroll
      for (int i = 0; i < 2; ++i) id[i] = page_of(0, i);
      load(g.cache.k, 0, kc, id);
      load(g.cache.v, 0, vc, id);
      sc = scale_of(id);
#pragma unroll
      for (int i = 0; i < 2; ++i) id2[i] = page_of(1, i);
    }
    for (int j = 0; j < T; ++j) {
      const int s = j % STAGES;
      const uint32_t ph = (uint32_t)(j / STAGES) & 1u;
#pragma unroll
      for (int i = 0; i < 2; ++i) id[i] = id2[i];           // of tile j + 1
      if (!mbar_wait_warp(smem_u32(&bar_k_empty[s]), ph ^ 1u, abortp, ga.wait_limit)) break;
      if ((cw & 1) == 0 && lane < 2) scales[j % SCALE_SETS][lane * 4 + (cw >> 1)] = sc;
      store(smem_base + C::OFF_K + s * C::TILE_BYTES, kc);
      fence_proxy_async_smem();
      warp_arrive(smem_u32(&bar_k_full[s]), lane);
      if (j + 1 < T) {
        load(g.cache.k, j + 1, kc, id);
        sc = scale_of(id);
#pragma unroll
        for (int i = 0; i < 2; ++i) id2[i] = page_of(j + 2, i);
      }
      const int slot0 = base + j * 128;
      if (slot0 < w.lo_all || slot0 + 128 > w.hi_all) {    // NaN values in slots that some rows do not see: see nan_fixup
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int p = 0; p < PC; ++p) {
            const uint4 q = vc[i][p];
            const uint4 n = make_uint4(nan_bytes(q.x), nan_bytes(q.y), nan_bytes(q.z), nan_bytes(q.w));
            any |= n.x | n.y | n.z | n.w;
            vc[i][p] = make_uint4(q.x & ~n.x, q.y & ~n.y, q.z & ~n.z, q.w & ~n.w);
          }
        if (any) sh_nan = 1;
      }
      if (!mbar_wait_warp(smem_u32(&bar_v_empty[s]), ph ^ 1u, abortp, ga.wait_limit)) break;
      store(smem_base + C::OFF_V + s * C::TILE_BYTES, vc);
      fence_proxy_async_smem();
      warp_arrive(smem_u32(&bar_v_full[s]), lane);
      if (j + 1 < T) load(g.cache.v, j + 1, vc, id);
    }
    if (bad_groups && lane == 0) flag_index(g.status);
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    // ---------------------------------------------------------------- softmax and output (warpgroups 0, 1)
    const int t = wg;
    if (t < ntile) {
      const int r = (warp & 3) * 32 + lane;                // row of the tile = lane of tensor memory
      const int rt = t * 128 + r;                          // row of the CTA's 256
      const bool live = rt < w.rows;
      const int row = w.tile * TC_ROWS + min(rt, w.rows - 1), tok = w.q.first + row / g.group, qh = w.head * g.group + row % g.group;
      const uint32_t lane_addr = tmem_base + ((uint32_t)((warp & 3) * 32) << 16);
      const uint32_t tm_s = lane_addr + C::TM_S + t * 128, tm_o = lane_addr + C::TM_O + t * 128;
      {                                                    // the query row into the swizzled tile
        const __half* src = g.q + (long long)tok * g.qt + (long long)qh * g.qh;
        const uint32_t dst = smem_base + t * C::TILE_BYTES + (uint32_t)r * 128;
#pragma unroll
        for (int p = 0; p < DP / 8; ++p) {
          uint4 q = make_uint4(0, 0, 0, 0);
          if (p * 8 < d) q = __ldg(reinterpret_cast<const uint4*>(src) + p);
          q.x ^= ga.flip; q.y ^= ga.flip; q.z ^= ga.flip; q.w ^= ga.flip;
          st_shared_v4_u32(dst + (uint32_t)(p >> 3) * 16384 + ((((uint32_t)p & 7u) ^ ((uint32_t)r & 7u)) << 4), q.x, q.y, q.z, q.w);
        }
        fence_proxy_async_smem();
        warp_arrive(smem_u32(&bar_q[t]), lane);
      }
      const View view = view_of(g, w.q, row);
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int jh = 0; jh < 2 * T; ++jh) {
        const int j = jh >> 1, h = jh & 1;
        if (!mbar_wait_warp(smem_u32(&bar_s_full[t][h]), (uint32_t)j & 1u, abortp, ga.wait_limit)) { ok = false; break; }
        tc_fence_after();
        uint32_t xr[64];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld_32x32(tm_s + h * 64 + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&xr[c * 32]));
        tmem_wait_ld();
        const int slot0 = base + jh * 64;
        if (slot0 < w.lo_all || slot0 + 64 > w.hi_all) {
          const int lo = view.lo - slot0, hi = view.hi - slot0;
#pragma unroll
          for (int q = 0; q < 64; ++q)
            if (q < lo || q >= hi) xr[q] = __float_as_uint(-INFINITY);
        }
        const float4* sc = scales[j % SCALE_SETS] + h * 4;
        float top = -INFINITY;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          float e0 = __uint_as_float(xr[b * 16]), e1 = __uint_as_float(xr[b * 16 + 1]);
#pragma unroll
          for (int q = 2; q < 14; q += 4) {
            e0 = max3(e0, __uint_as_float(xr[b * 16 + q]), __uint_as_float(xr[b * 16 + q + 1]));
            e1 = max3(e1, __uint_as_float(xr[b * 16 + q + 2]), __uint_as_float(xr[b * 16 + q + 3]));
          }
          e0 = max3(e0, __uint_as_float(xr[b * 16 + 14]), __uint_as_float(xr[b * 16 + 15]));
          const float2 s2 = *reinterpret_cast<const float2*>(&sc[b]);
          top = fmaxf(top, fmaf(fmaxf(e0, e1), s2.x, s2.y));   // the scales are positive: see flip
        }
        if (__any_sync(0xffffffffu, top > m + 1.f)) {      // some row's maximum moves: all rows of the warp take theirs
          const float now = fmaxf(m, top);
          const float f = now == -INFINITY ? 1.f : ex2(m - now);
          m = now;
          l *= f;
          if (jh > 0) {                                    // once the half before has been added
            if (!mbar_wait_warp(smem_u32(&bar_pv_done[t][h ^ 1]), (uint32_t)((jh - 1) >> 1) & 1u, abortp, ga.wait_limit)) { ok = false; break; }
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < DP / 16; ++c) {
              uint32_t v[16];
              tmem_ld_32x16(tm_o + c * 16, v);
              tmem_wait_ld();
#pragma unroll
              for (int q = 0; q < 16; ++q) v[q] = __float_as_uint(__uint_as_float(v[q]) * f);
              tmem_st_32x16(tm_o + c * 16, v);
            }
          }
        }
        const float nm = m == -INFINITY ? 0.f : LIFT - m;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int b2 = 0; b2 < 2; ++b2) {
            const int b = c * 2 + b2;
            const float4 s4 = sc[b];
            const float shift = s4.y + nm;
            const uint64_t sx = pair(s4.x, s4.x), sh = pair(shift, shift);
            uint64_t sum = 0;
#pragma unroll
            for (int q = 0; q < 16; q += 2) {
              float p0, p1;
              split(fma_pair(pair(__uint_as_float(xr[b * 16 + q]), __uint_as_float(xr[b * 16 + q + 1])), sx, sh), p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
              sum = add_pair(sum, pair(p0, p1));
              pk[b2 * 8 + q / 2] = half2_of(p0, p1);
            }
            float s0, s1;
            split(sum, s0, s1);
            l = fmaf(s0 + s1, s4.z, l);
          }
          tmem_st_32x16(tm_s + h * 64 + c * 16, pk);
        }
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(smem_u32(&bar_p_full[t][h]), lane);
      }
      if (ok && T > 0) {                                   // the tile's products complete in the order of their issue
        ok = mbar_wait_warp(smem_u32(&bar_pv_done[t][0]), (uint32_t)(T - 1) & 1u, abortp, ga.wait_limit) &&
             mbar_wait_warp(smem_u32(&bar_pv_done[t][1]), (uint32_t)(T - 1) & 1u, abortp, ga.wait_limit);
        tc_fence_after();
      }
      if (ok) {
        const bool whole = w.ranges == 1;
        const float inv = !whole ? 1.f : l == 0.f ? 0.f : 1.f / l;            // a row that sees nothing: 0, and -inf below
        const long long cta = (long long)unit * g.splits + x;
        __half* dst = g.out + (long long)tok * g.ot + (long long)qh * g.oh;
        float* part = g.part_o + (cta * TC_ROWS + rt) * d;
        const bool fix = sh_nan != 0;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t v[32];
          if (T > 0) {
            tmem_ld_32x32(tm_o + c * 32, v);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int q = 0; q < 32; ++q) v[q] = 0;
          }
          if (!live || c * 32 >= d) continue;
#pragma unroll
          for (int q = 0; q < 32; q += 8) {
            float o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = __uint_as_float(v[q + e]) * inv;
            if (fix) nan_fixup(g, w, 8, row, c * 32 + q, o);
            if (whole) {
              *reinterpret_cast<uint4*>(dst + c * 32 + q) =
                  make_uint4(half2_of(o[0], o[1]), half2_of(o[2], o[3]), half2_of(o[4], o[5]), half2_of(o[6], o[7]));
            } else {
              *reinterpret_cast<float4*>(part + c * 32 + q) = make_float4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<float4*>(part + c * 32 + q + 4) = make_float4(o[4], o[5], o[6], o[7]);
            }
          }
        }
        if (live && whole && g.lse)
          g.lse[(long long)tok * g.q_heads + qh] = l == 0.f ? -INFINITY : (m - LIFT + log2f(l)) * 0.6931471805599453f;
        if (live && !whole) g.part_ml[cta * TC_ROWS + rt] = make_float2(m, l);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  teardown(abort_flag, g.status);
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace

namespace kv {

int launch_attention_tc(const AttArgs& g, long long ctas, bool sort, cudaStream_t stream) {
  TcArgs2 a;
  a.a = g;
  a.flip = a.a.scale_log2 < 0.f ? 0x80008000u : 0u;
  a.a.scale_log2 = fabsf(a.a.scale_log2);
  a.sorted = sort && g.splits == 1 && (long long)g.batch.seqs * g.tiles <= MOST_SORTED;
  a.wait_limit = 400000000LL + (long long)(g.range / 128) * 400000LL;
  if (g.cache.d <= 64) kv_prefill_kernel<64><<<(unsigned)ctas, THREADS, Cfg<64>::SMEM_BYTES, stream>>>(a);
  else kv_prefill_kernel<128><<<(unsigned)ctas, THREADS, Cfg<128>::SMEM_BYTES, stream>>>(a);
  count_launch(true);
  return note_cuda_error(cudaGetLastError(), "cache attention launch (many rows)");
}

int setup_attention_tc() {
  int rc = note_cuda_error(cudaFuncSetAttribute(kv_prefill_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<64>::SMEM_BYTES),
                           "cudaFuncSetAttribute(cache attention 64)");
  if (rc) return rc;
  return note_cuda_error(cudaFuncSetAttribute(kv_prefill_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<128>::SMEM_BYTES),
                         "cudaFuncSetAttribute(cache attention 128)");
}

}  // namespace kv

}  // namespace b200
