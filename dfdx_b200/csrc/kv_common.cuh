// The paged 8-bit key/value cache as its kernels see it (kv_cache.cu: append and read back, kv_attention.cu).
//
// Codes are e4m3 (3 mantissa bits, values up to 448); every block of one page's tokens and one head has a scale, a power
// of two: value = code * scale.  A power of two costs e4m3 nothing but at most one of its 15 binades, makes the change
// of a block's scale exact (but for values that fall below 2^-6 * scale), and lets the attention move a value block's
// scale into the softmax's exponent.
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>

namespace b200 {
namespace kv {

constexpr int MAX_SLOTS = 1 << 30; // of a sequence: slot arithmetic stays within 32 bits
constexpr int MIN_EXP = -60;       // the smallest scale is 2^-60: what a block of zeros gets

struct Cache {
  uint8_t *k, *v;                  // pages x heads x page x d
  float *k_scale, *v_scale;        // pages x heads
  int pages, heads, page, page_log2, d;
};

struct Batch {
  int seqs, tokens, max_new;
  const int *cu, *lens, *table;
  int table_stride, max_pages;
};

struct Seq {
  int first, m, len;               // first new token, how many, slots in use with them
  bool ok;
};

// Whether a sequence's bounds fit the buffers; checked before any address is formed from them.
__device__ __forceinline__ bool fits(const Batch& b, const Cache& c, const Seq& q) {
  return q.first >= 0 && q.m >= 0 && q.m <= b.max_new && q.first <= b.tokens - q.m && q.len >= 0 &&
         q.len <= min((long long)b.max_pages << c.page_log2, (long long)MAX_SLOTS);
}
__device__ __forceinline__ Seq load_seq(const Batch& b, const Cache& c, int s) {
  Seq q;
  q.first = b.cu[s];
  q.m = b.cu[s + 1] - q.first;
  q.len = b.lens[s];
  q.ok = fits(b, c, q);
  return q;
}
// A wait that ran out (it exchanges the word) says more, and stays.
__device__ __forceinline__ void flag_index(int* status) { atomicCAS(status, 0, (int)B200_ERR_INDEX); }

// The exponent of the smallest power of two s with absmax <= 448 s; 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exp(float absmax) {
  const uint32_t x = __float_as_uint(absmax);
  const int e = (int)(x >> 23) - 127 - 8 + ((x & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < MIN_EXP ? MIN_EXP : e;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127

// The magnitude that a value asks of its block's scale: infinities and NaN ask nothing.
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}
// Two values to codes, to the nearest with ties to even; infinities to +-448, NaN stays NaN.
__device__ __forceinline__ uint32_t codes2(float x, float y) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(x, y), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t codes4(const float (&x)[4], float inv) {
  return codes2(x[0] * inv, x[1] * inv) | codes2(x[2] * inv, x[3] * inv) << 16;
}
__device__ __forceinline__ uint2 values4(uint32_t codes) {         // four codes as f16, exact
  uint2 r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}"
      : "=r"(r.x), "=r"(r.y) : "r"(codes));
  return r;
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
inline int parse_cache(const b200_kv_cache* c, Cache* out) {
  if (!c) return B200_ERR_NULL;
  if (c->d == 0 || c->d % 32 || c->d > 128) return B200_ERR_UNSUPPORTED;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128) return B200_ERR_UNSUPPORTED;
  if (c->heads == 0) return B200_ERR_SHAPE;
  if (c->pages > 0x7fffffff || c->heads > 65535) return B200_ERR_LIMIT;
  if (c->pages && (!c->k || !c->v || !c->k_scale || !c->v_scale)) return B200_ERR_NULL;
  if (((uintptr_t)c->k | (uintptr_t)c->v) & 15) return B200_ERR_UNSUPPORTED;
  out->k = (uint8_t*)c->k; out->v = (uint8_t*)c->v;
  out->k_scale = c->k_scale; out->v_scale = c->v_scale;
  out->pages = (int)c->pages; out->heads = (int)c->heads; out->page = (int)c->page_size; out->d = (int)c->d;
  out->page_log2 = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  return B200_OK;
}
inline int parse_batch(const b200_kv_batch* b, Batch* out) {
  if (!b) return B200_ERR_NULL;
  if (b->seqs > 0x3fffffff || b->tokens > 0x3fffffff || b->max_pages > 0x3fffffff || b->page_table_stride > 0x7fffffff) return B200_ERR_LIMIT;
  if (b->max_new > b->tokens) return B200_ERR_SHAPE;
  if (b->seqs && b->tokens && (!b->cu_tokens || !b->seq_lens || (b->max_pages && !b->page_table))) return B200_ERR_NULL;
  if (b->seqs > 1 && b->max_pages && b->page_table_stride < b->max_pages) return B200_ERR_STRIDE;
  out->seqs = (int)b->seqs; out->tokens = (int)b->tokens; out->max_new = (int)b->max_new;
  out->cu = b->cu_tokens; out->lens = b->seq_lens; out->table = b->page_table;
  out->table_stride = (int)b->page_table_stride; out->max_pages = (int)b->max_pages;
  return B200_OK;
}

}  // namespace kv
}  // namespace b200
