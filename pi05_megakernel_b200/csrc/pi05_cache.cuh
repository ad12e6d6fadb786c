// The cache in pages as the kernels see it: keys and values [pages][layers][page_tokens][kv_heads][head_dim] in BF16, int8 or
// e4m3, with one FP32 scale per token and head [pages][layers][kv_heads][page_tokens] for the 8-bit formats.
//   A token's scales lie next to those of the page's other tokens, not next to its codes: attention takes the scales of a run of
// keys of one head as one vector, and a page's codes stay a dense box for tiled copies.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/pi05_b200.h"

namespace cache {

// Codes of the status words (the word behind holds the sequence).
enum { BAD_PAGE = PI05_CACHE_BAD_PAGE, BAD_POSITION = PI05_CACHE_BAD_POSITION };

__device__ __forceinline__ void report(unsigned int* status, int code, int where) {
  if (atomicCAS(status, 0u, (unsigned)code) == 0u) status[1] = (unsigned)where;
}

// Two codes of a byte as a pair of 16-bit numbers, exactly.  As BF16,
//   int8: a code c is low - 128 sign with low = c & 127.  0x4300 | low is 128 + low, 0x4300 | (c & 128) is 128 or 256, and the difference of the
// two is exact.  `w`: the codes in the low bytes of its halves.
__device__ __forceinline__ uint32_t int8_pair(uint32_t w) {
  const uint32_t a = (w & 0x007f007fu) | 0x43004300u, b = (w & 0x00800080u) | 0x43004300u;
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
//   e4m3: exponent and mantissa moved to where BF16 (FP16) has them read as the value times 2^-120 (2^-8), subnormals included, and the product
// with 2^120 (2^8) is exact.  `w`: the codes in the high bytes of its halves, zeros in the low ones.  (The two NaN codes, which the kernels never write but
// memory may hold at places that do not count, read as +-480.)
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w) {
  const uint32_t a = ((w >> 4) & 0x07f007f0u) | (w & 0x80008000u);
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0x7b807b80u));
  return r;
}
__device__ __forceinline__ uint32_t e4m3_half_pair(uint32_t w) {
  const uint32_t a = ((w >> 1) & 0x3f803f80u) | (w & 0x80008000u);
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0x5c005c00u));
  return r;
}
// Four codes of a word as two pairs of BF16.
template <int FORMAT>
__device__ __forceinline__ uint2 quad(uint32_t w) {
  if (FORMAT == PI05_CACHE_INT8) return make_uint2(int8_pair(__byte_perm(w, 0, 0x4140)), int8_pair(__byte_perm(w, 0, 0x4342)));
  return make_uint2(e4m3_pair(__byte_perm(w, 0, 0x1404)), e4m3_pair(__byte_perm(w, 0, 0x3424)));
}
// The same as FP16.  int8: 0x6400 | (c ^ 128) is 1024 + 128 + c.
template <int FORMAT>
__device__ __forceinline__ uint2 quad_half(uint32_t w) {
  if (FORMAT != PI05_CACHE_INT8) return make_uint2(e4m3_half_pair(__byte_perm(w, 0, 0x1404)), e4m3_half_pair(__byte_perm(w, 0, 0x3424)));
  uint2 r;
  w ^= 0x80808080u;
  const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.x) : "r"(a), "r"(0x64806480u));
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r.y) : "r"(b), "r"(0x64806480u));
  return r;
}

__device__ __forceinline__ float lo16(uint32_t v) { return __uint_as_float(v << 16); }
__device__ __forceinline__ float hi16(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Host: whether rows of `width` elements meet, one at i . stride_a (i_k < size_a[k]) and the other at distance + j . stride_b; with size_b = NULL
// two different rows of the first tensor.  A row's place is a sum of terms stride x index, so this asks for indexes that bring such a sum into (-width, width):
// largest stride first, of whose indexes only those are tried that the smaller strides can still make up for, one to three where strides are nested.
struct MeetTerm { long long stride, lo, hi; };
inline bool meet_search(const MeetTerm* t, int terms, __int128 at, long long width, bool other, bool moved, int* budget) {
  if (--*budget < 0) return true;                                  // cannot be told: as if they met
  if (terms == 0) return at < width && at > -(__int128)width && (other || moved);
  __int128 lo = 0, hi = 0;                                         // what the smaller strides reach
  for (int i = 1; i < terms; ++i) { lo += (__int128)t[i].stride * t[i].lo; hi += (__int128)t[i].stride * t[i].hi; }
  auto down = [&](__int128 v) { return v >= 0 ? v / t->stride : -((-v + t->stride - 1) / t->stride); };
  __int128 first = -down(width - 1 + at + hi), last = down(width - 1 - at - lo);
  if (first < t->lo) first = t->lo;
  if (last > t->hi) last = t->hi;
  for (__int128 x = first; x <= last; ++x)
    if (meet_search(t + 1, terms - 1, at + x * t->stride, width, other, moved || x != 0, budget)) return true;
  return false;
}
inline bool rows_meet(int dims, const long long* size_a, const long long* stride_a, const long long* size_b, const long long* stride_b, long long distance,
                      long long width) {
  MeetTerm t[8];
  int n = 0;
  const bool other = size_b != nullptr;
  for (int k = 0; k < dims; ++k)
    if (size_a[k] <= 0 || (other && size_b[k] <= 0)) return false; // no rows
  for (int side = 0; side < (other ? 2 : 1); ++side)
    for (int k = 0; k < dims; ++k) {
      const long long size = (side ? size_b : size_a)[k], stride = (side ? stride_b : stride_a)[k];
      if (size == 1 || (stride == 0 && other)) continue;
      if (stride == 0) return true;
      const bool up = (side != 0) == (stride > 0);                 // (of the first tensor the index is subtracted)
      MeetTerm term = {stride < 0 ? -stride : stride, other && up ? 0 : -(size - 1), other && !up ? 0 : size - 1};
      int at = 0;
      while (at < n && t[at].stride > term.stride) ++at;
      if (at < n && t[at].stride == term.stride) {
        if (!other) return true;
        t[at].lo += term.lo; t[at].hi += term.hi;
        continue;
      }
      for (int i = n++; i > at; --i) t[i] = t[i - 1];
      t[at] = term;
    }
  if (!other) {                                                    // every stride behind all that the smaller ones reach: as tensors usually lie
    __int128 extent = width;
    int i = n;
    while (i > 0 && t[i - 1].stride >= extent) { --i; extent += (__int128)t[i].stride * t[i].hi; }
    if (i == 0) return false;
  }
  __int128 lo = distance, hi = distance;                           // far apart: as tensors of their own are
  for (int i = 0; i < n; ++i) { lo += (__int128)t[i].stride * t[i].lo; hi += (__int128)t[i].stride * t[i].hi; }
  if (lo >= width || hi <= -width) return false;
  int budget = 10000;
  return meet_search(t, n, distance, width, other, false, &budget);
}

// Host: `dev` as the current device, for as long as this lives.
struct DeviceGuard {
  int prev = -1;
  bool ok;
  explicit DeviceGuard(int dev) { if (cudaGetDevice(&prev) != cudaSuccess) prev = -1; ok = prev == dev || cudaSetDevice(dev) == cudaSuccess; }
  ~DeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};

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
