// The cache in pages as the kernels see it: keys and values [pages][layers][page_tokens][kv_heads][head_dim] in BF16, int8 or
// e4m3, with one FP32 scale per token and head [pages][layers][kv_heads][page_tokens] for the 8-bit formats.
//   A token's scales lie next to those of the page's other tokens, not next to its codes: attention takes the scales of a run of
// keys of one head as one vector, and a page's codes stay a dense box for tiled copies.
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

#include "../../include/pi05_b200.h"

namespace cache {

// Codes of the status words (the word behind holds the sequence).
enum { BAD_PAGE = PI05_CACHE_BAD_PAGE, BAD_POSITION = PI05_CACHE_BAD_POSITION };

__device__ __forceinline__ void report(unsigned int* status, int code, int where) {
  if (atomicCAS(status, 0u, (unsigned)code) == 0u) status[1] = (unsigned)where;
}

// Two codes in the low halves of the two bytes of each 16-bit half of `w` (0x00BB00AA) as a pair of BF16, exactly.
//   int8: a code c = low - 128 * sign with low = c & 127.  0x4300 | low is 128 + low, 0x4300 | (c & 128) is 128 or 256, and the
// difference of the two is exact.
__device__ __forceinline__ uint32_t int8_pair(uint32_t w) {
  const uint32_t a = (w & 0x007f007fu) | 0x43004300u, b = (w & 0x00800080u) | 0x43004300u;
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
//   e4m3: exponent and mantissa moved to where BF16 has them read as the value times 2^-120, subnormals included, and the product with
// 2^120 is exact.  (The two NaN codes read as 480: the kernels never write them.)
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
  const uint32_t a = ((w & 0x007f007fu) << 4) | ((w & 0x00800080u) << 8);
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0x7b807b80u));
  return r;
}
template <int FORMAT>
__device__ __forceinline__ uint32_t pair(uint32_t w) { return FORMAT == PI05_CACHE_INT8 ? int8_pair(w) : e4m3_pair(w); }
// Four codes of a word as two pairs of BF16.
template <int FORMAT>
__device__ __forceinline__ uint2 quad(uint32_t w) {
  return make_uint2(pair<FORMAT>(__byte_perm(w, 0, 0x4140)), pair<FORMAT>(__byte_perm(w, 0, 0x4342)));
}

__device__ __forceinline__ float lo16(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi16(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Host: whether a cache is one that the kernels can work on.
inline bool well_formed(const pi05_cache* c) {
  if (!c || !c->k || !c->v || !c->status) return false;
  if (c->format != PI05_CACHE_BF16 && c->format != PI05_CACHE_INT8 && c->format != PI05_CACHE_E4M3) return false;
  if (c->format != PI05_CACHE_BF16 && (!c->k_scale || !c->v_scale)) return false;
  if (c->pages < 1 || c->layers < 1 || c->kv_heads < 1 || c->kv_heads > 256 || c->page_tokens < 16 || c->page_tokens % 16) return false;
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return false;
  if ((long long)c->pages * c->page_tokens > 0x7fffffffll || c->layers > 4096) return false;
  const uintptr_t bits = (uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale;
  return !(bits & 15) && !((uintptr_t)c->status & 7);
}

}  // namespace cache
