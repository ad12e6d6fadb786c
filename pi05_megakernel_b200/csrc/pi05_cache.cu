// Rows of keys and values into the pages of a cache, and out of them.
//
// Both are one pass over their data.  A row (head_dim elements of one token, head and layer) is taken by neighbouring lanes, 16 elements each, keys and
// values by the same lanes, which look the page up once.  What bounds them is memory as long as a pair of elements costs no more than some 30
// instructions: hence 16 elements a lane (the page, the row's maximum and its quotient once for them) and arithmetic in pairs.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/pi05_b200.h"
#include "pi05_cache.cuh"
#include "ptx_sm100.cuh"

namespace {

using cache::DeviceGuard;
using cache::hi16;
using cache::lo16;
using cache::pack2;

constexpr int BLOCK = 128;

struct RowArgs {
  pi05_cache c;
  pi05_cache_rows r;
  unsigned rows;                  // tokens x heads, of one sequence and layer
  int wide;                       // rows of 16-bit elements begin on 32 bytes
};

// Where a row of the call is: in the caller's tensors and in the pool (element offsets), and its scale.
struct Place { long long mine, pool, scale; bool has, good; };

__device__ __forceinline__ Place place(const RowArgs& a, unsigned row, int layer, int b) {
  const pi05_cache& c = a.c;
  const pi05_cache_rows& r = a.r;
  Place p;
  const unsigned t = row / (unsigned)c.kv_heads, head = row - t * (unsigned)c.kv_heads;
  p.mine = b * r.batch_stride + layer * r.layer_stride + t * r.token_stride + head * r.head_stride;
  p.has = !r.counts || (int)t < __ldg(r.counts + b);
  const int start = r.starts ? __ldg(r.starts + b) : 0;
  const unsigned pos = (unsigned)start + t, lp = pos / (unsigned)c.page_tokens, at = pos - lp * (unsigned)c.page_tokens;
  p.good = start >= 0 && lp < (unsigned)r.table_pages;
  int page = -1;
  if (p.has) {
    if (p.good) page = __ldg(r.table + (long long)b * r.table_stride + lp);
    if (!p.good) cache::report(c.status, cache::BAD_POSITION, b);
    else if (page < 0 || page >= c.pages) { cache::report(c.status, cache::BAD_PAGE, b); p.good = false; }
  }
  const long long pl = (long long)page * c.layers + r.layer + layer;
  p.pool = ((pl * c.page_tokens + at) * c.kv_heads + head) * c.head_dim;
  p.scale = (pl * c.kv_heads + head) * c.page_tokens + at;
  return p;
}

// A lane's 32 bytes, in one piece where they are aligned (two pieces of 16 leave the gaps of a warp's line to the other one: sixteen prefixes of 968 tokens
// are read back in 60 us in one piece, in 78 in two).
__device__ __forceinline__ void load_32(uint4 (&x)[2], const uint4* from, bool wide) {
  if (wide) {
    asm volatile("ld.global.cs.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(x[0].x), "=r"(x[0].y), "=r"(x[0].z), "=r"(x[0].w), "=r"(x[1].x), "=r"(x[1].y), "=r"(x[1].z), "=r"(x[1].w) : "l"(from));
  } else {
    x[0] = __ldcs(from);
    x[1] = __ldcs(from + 1);
  }
}
__device__ __forceinline__ void store_32(uint4* to, const uint4 (&x)[2], bool wide) {
  if (wide) {
    asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(to), "r"(x[0].x), "r"(x[0].y), "r"(x[0].z), "r"(x[0].w), "r"(x[1].x), "r"(x[1].y), "r"(x[1].z), "r"(x[1].w) : "memory");
  } else {
    __stcs(to, x[0]);
    __stcs(to + 1, x[1]);
  }
}

// Largest magnitude of a pair of BF16, NaN where there is one.
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Sixteen elements of a row as codes, and the row's scale.
//   code = rn(x * peak / a) of the true quotient, a the row's largest magnitude.  With BF16 x and a the quotient is either in the middle of
// two codes exactly (x = a / 2 is 63.5) or at least 2^-16 of itself away from it (int8: mantissas 254 and 255 give 126.502; e4m3: 2^-12.9; over all pairs of
// mantissas), so it only has to be right to that, and exact in the middle: peak / a as the sum of two FP32 numbers (its approximation by the reciprocal,
// corrected once by its residual, as Markstein, IBM J. Res. Dev. 34, 1990, and what the residual of that leaves), and x times it as one FMA on top of the
// small product, which rounds once.  The scale a / peak is corrected by its residual in the same way.
template <int FORMAT, int LANES>
__device__ __forceinline__ uint4 encode(const uint4 (&x)[2], float* scale) {
  constexpr float PEAK = FORMAT == PI05_CACHE_INT8 ? 127.0f : 448.0f, ONE_PEAKTH = 1.0f / PEAK;
  const uint32_t m = 0x7fff7fffu, w[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
  uint32_t top = max_pair(max_pair(max_pair(w[0] & m, w[1] & m), max_pair(w[2] & m, w[3] & m)), max_pair(max_pair(w[4] & m, w[5] & m), max_pair(w[6] & m, w[7] & m)));
  top = max_pair(top, __byte_perm(top, 0, 0x1032));                // both halves
#pragma unroll
  for (int d = LANES / 2; d; d >>= 1) top = max_pair(top, __shfl_xor_sync(0xffffffffu, top, d));
  float a = lo16(top), f = 1.f;
  if (!(a > 0.f && a <= 3.3895314e38f)) {                          // nothing but zeros; an infinity or a NaN: the whole row reads back as NaN
    *scale = a == 0.f ? 0.f : __uint_as_float(0x7fffffffu);
    return make_uint4(0u, 0u, 0u, 0u);
  }
  if (!(a > 1e-30f && a < 1e30f)) {                                // keep quotient and products away from the ends of FP32: both times a power of two
    f = a < 1.f ? 0x1p+90f : 0x1p-90f;
    *scale = __fdiv_rn(a, PEAK);
    a *= f;
  } else {
    const float q = a * ONE_PEAKTH;
    *scale = fmaf(fmaf(-q, PEAK, a), ONE_PEAKTH, q);               // a / peak, rounded once
  }
  const float r = ptx::rcp_approx(a), h = PEAK * r, hi = fmaf(fmaf(-h, a, PEAK), r, h), lo = fmaf(-hi, a, PEAK) * r;
  const float2 hi2 = make_float2(hi, hi), lo2 = make_float2(lo, lo), zero = make_float2(0.f, 0.f), f2 = make_float2(f, f);
  uint32_t code[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float2 y[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float2 v = make_float2(lo16(w[2 * k + i]), hi16(w[2 * k + i]));
      if (f != 1.f) { v.x *= f2.x; v.y *= f2.y; }
      y[i] = ptx::fma2(v, hi2, ptx::fma2(v, lo2, zero));
    }
    if (FORMAT == PI05_CACHE_INT8) {
      // to the nearest whole number, ties to even, by a sum whose last place is 1; its last byte is the code
      const uint32_t a0 = __float_as_uint(y[0].x + 12582912.0f), a1 = __float_as_uint(y[0].y + 12582912.0f), a2 = __float_as_uint(y[1].x + 12582912.0f),
                     a3 = __float_as_uint(y[1].y + 12582912.0f);
      code[k] = __byte_perm(__byte_perm(a0, a1, 0x0040), __byte_perm(a2, a3, 0x0040), 0x5410);
    } else {
      unsigned short p[2];
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p[0]) : "f"(y[0].y), "f"(y[0].x));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p[1]) : "f"(y[1].y), "f"(y[1].x));
      code[k] = p[0] | (uint32_t)p[1] << 16;
    }
  }
  return make_uint4(code[0], code[1], code[2], code[3]);
}

template <int FORMAT, int DIM>
__global__ void __launch_bounds__(BLOCK) write_kernel(const __grid_constant__ RowArgs a) {
  constexpr int LANES = DIM / 16;
  const int lane = threadIdx.x % LANES;
  const unsigned row = blockIdx.x * (BLOCK / LANES) + threadIdx.x / LANES;
  const bool in = row < a.rows;                                    // (every lane takes part in the shuffles)
  const Place p = place(a, in ? row : 0, blockIdx.y, blockIdx.z);
  const bool store = in && p.has && p.good;
  uint4 k[2] = {}, v[2] = {};
  if (store) {
    load_32(k, reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.r.k) + p.mine) + 2 * lane, a.wide);
    load_32(v, reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.r.v) + p.mine) + 2 * lane, a.wide);
  }
  if constexpr (FORMAT == PI05_CACHE_BF16) {
    if (!store) return;
    store_32(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.c.k) + p.pool) + 2 * lane, k, a.wide);
    store_32(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.c.v) + p.pool) + 2 * lane, v, a.wide);
  } else {
    float ks, vs;
    const uint4 kc = encode<FORMAT, LANES>(k, &ks), vc = encode<FORMAT, LANES>(v, &vs);
    if (!store) return;
    reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.c.k) + p.pool)[lane] = kc;
    reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.c.v) + p.pool)[lane] = vc;
    if (lane == 0) { a.c.k_scale[p.scale] = ks; a.c.v_scale[p.scale] = vs; }
  }
}

// Eight of a lane's codes as BF16 values: the code as a 16-bit number, exactly, times the scale in FP32.
template <int FORMAT>
__device__ __forceinline__ uint4 decode(uint32_t lo, uint32_t hi, float scale) {
  const uint2 a = cache::quad<FORMAT>(lo), b = cache::quad<FORMAT>(hi);
  return make_uint4(pack2(lo16(a.x) * scale, hi16(a.x) * scale), pack2(lo16(a.y) * scale, hi16(a.y) * scale),
                    pack2(lo16(b.x) * scale, hi16(b.x) * scale), pack2(lo16(b.y) * scale, hi16(b.y) * scale));
}

template <int FORMAT, int DIM>
__global__ void __launch_bounds__(BLOCK) read_kernel(const __grid_constant__ RowArgs a) {
  constexpr int LANES = DIM / 16;
  const int lane = threadIdx.x % LANES;
  const unsigned row = blockIdx.x * (BLOCK / LANES) + threadIdx.x / LANES;
  if (row >= a.rows) return;
  const Place p = place(a, row, blockIdx.y, blockIdx.z);
  // behind the sequence's tokens zeros; where there is no such page NaN, so that nobody takes it for a key
  const uint32_t none = p.has ? 0x7fff7fffu : 0u;
  uint4 k[2] = {make_uint4(none, none, none, none), make_uint4(none, none, none, none)}, v[2] = {k[0], k[0]};
  if (p.has && p.good) {
    if constexpr (FORMAT == PI05_CACHE_BF16) {
      load_32(k, reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.c.k) + p.pool) + 2 * lane, a.wide);
      load_32(v, reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.c.v) + p.pool) + 2 * lane, a.wide);
    } else {
      const uint4 kc = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.c.k) + p.pool) + lane);
      const uint4 vc = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.c.v) + p.pool) + lane);
      const float ks = __ldg(a.c.k_scale + p.scale), vs = __ldg(a.c.v_scale + p.scale);
      k[0] = decode<FORMAT>(kc.x, kc.y, ks); k[1] = decode<FORMAT>(kc.z, kc.w, ks);
      v[0] = decode<FORMAT>(vc.x, vc.y, vs); v[1] = decode<FORMAT>(vc.z, vc.w, vs);
    }
  }
  store_32(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.r.k) + p.mine) + 2 * lane, k, a.wide);
  store_32(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.r.v) + p.mine) + 2 * lane, v, a.wide);
}

typedef void (*RowKernel)(const RowArgs);
#define BY_DIM(KERNEL, F) {KERNEL<F, 64>, KERNEL<F, 128>, KERNEL<F, 256>}
const RowKernel kWrite[3][3] = {BY_DIM(write_kernel, PI05_CACHE_BF16), BY_DIM(write_kernel, PI05_CACHE_INT8), BY_DIM(write_kernel, PI05_CACHE_E4M3)};
const RowKernel kRead[3][3] = {BY_DIM(read_kernel, PI05_CACHE_BF16), BY_DIM(read_kernel, PI05_CACHE_INT8), BY_DIM(read_kernel, PI05_CACHE_E4M3)};
#undef BY_DIM

int move_rows(const RowKernel (&kernels)[3][3], int device, const pi05_cache* c, const pi05_cache_rows* r, void* stream, bool out) {
  if (device < 0 || !cache::well_formed(c) || !r) return PI05_ERR_ARGUMENT;
  if (r->batch < 0 || r->tokens < 0 || r->layers < 0 || r->layer < 0 || r->layer > c->layers - r->layers || r->table_pages < 0 || r->table_stride < 0)
    return PI05_ERR_ARGUMENT;
  if (r->batch == 0 || r->tokens == 0 || r->layers == 0) return PI05_OK;
  const long long rows = (long long)r->tokens * c->kv_heads;
  if (!r->k || !r->v || !r->table || rows > 0x7fffffffll || r->batch > 65535 || r->layers > 65535) return PI05_ERR_ARGUMENT;
  if ((((uintptr_t)r->k | (uintptr_t)r->v) & 15) || ((r->batch_stride | r->layer_stride | r->token_stride | r->head_stride) & 7) ||
      (((uintptr_t)r->table | (uintptr_t)r->starts | (uintptr_t)r->counts) & 3))
    return PI05_ERR_ARGUMENT;
  if (out) {                                                       // rows on one another would be written by several blocks at once
    const long long size[4] = {r->batch, r->layers, r->tokens, c->kv_heads}, stride[4] = {r->batch_stride, r->layer_stride, r->token_stride, r->head_stride};
    const long long apart = (long long)((intptr_t)r->v - (intptr_t)r->k) / 2;
    if (cache::rows_meet(4, size, stride, nullptr, nullptr, 0, c->head_dim) || cache::rows_meet(4, size, stride, size, stride, apart, c->head_dim))
      return PI05_ERR_ARGUMENT;
  }
  DeviceGuard guard(device);
  if (!guard.ok) { cudaGetLastError(); return PI05_ERR_NO_DEVICE; }
  const int per = BLOCK / (c->head_dim / 16);
  uintptr_t bits = (uintptr_t)r->k | (uintptr_t)r->v | (uintptr_t)(2 * (r->batch_stride | r->layer_stride | r->token_stride | r->head_stride));
  if (c->format == PI05_CACHE_BF16) bits |= (uintptr_t)c->k | (uintptr_t)c->v;
  const RowArgs a = {*c, *r, (unsigned)rows, (bits & 31) == 0};
  const RowKernel kernel = kernels[c->format][c->head_dim == 64 ? 0 : c->head_dim == 128 ? 1 : 2];
  kernel<<<dim3((unsigned)((rows + per - 1) / per), r->layers, r->batch), BLOCK, 0, (cudaStream_t)stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? PI05_OK : PI05_ERR_CUDA;
}

}  // namespace

extern "C" {

int pi05_rows_meet(int dims, const long long* size_a, const long long* stride_a, const long long* size_b, const long long* stride_b, long long distance,
                   int width) {
  if (dims < 0 || dims > 4 || width < 1 || !size_a || !stride_a || (size_b && !stride_b)) return 1;
  return cache::rows_meet(dims, size_a, stride_a, size_b, stride_b, distance, width) ? 1 : 0;
}

int pi05_cache_write(int device, const pi05_cache* cache, const pi05_cache_rows* rows, void* stream) {
  return move_rows(kWrite, device, cache, rows, stream, false);
}

int pi05_cache_read(int device, const pi05_cache* cache, const pi05_cache_rows* rows, void* stream) {
  return move_rows(kRead, device, cache, rows, stream, true);
}

int pi05_cache_status(int device, const pi05_cache* cache, void* stream, int* code, int* where) {
  if (device < 0 || !cache::well_formed(cache) || !code || !where) return PI05_ERR_ARGUMENT;
  DeviceGuard guard(device);
  if (!guard.ok) { cudaGetLastError(); return PI05_ERR_NO_DEVICE; }
  unsigned int st[4] = {0, 0, 0, 0};
  cudaStream_t s = (cudaStream_t)stream;
  cudaError_t e = cudaMemcpyAsync(st, cache->status, sizeof st, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaMemsetAsync(cache->status, 0, sizeof st, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return PI05_ERR_CUDA;
  const unsigned int* first = st[2] ? st + 2 : st;       // a wait that gave up, else what was wrong with the tables
  *code = (int)first[0];
  *where = (int)first[1];
  return st[2] ? PI05_ERR_DEVICE_TIMEOUT : st[0] ? PI05_ERR_PAGE_TABLE : PI05_OK;
}

}  // extern "C"
