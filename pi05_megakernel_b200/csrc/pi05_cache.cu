// Rows of keys and values into the pages of a cache, and out of them.
//
// Both are one pass over their data, bound by memory: a row (head_dim elements of one token, head and layer) is taken by
// head_dim / 8 neighbouring lanes, 16 bytes of BF16 each, keys and values by the same lanes so that a thread has two rows on
// their way and looks the page up once.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/pi05_b200.h"
#include "pi05_cache.cuh"
#include "ptx_sm100.cuh"

namespace {

using cache::hi16;
using cache::lo16;
using cache::pack2;

constexpr int BLOCK = 256;

struct RowArgs {
  pi05_cache c;
  pi05_cache_rows r;
  long long rows;                 // batch x tokens x heads, of one layer
};

// Where a row of the call is: in the caller's tensors and in the pool (element offsets), and its scale.
struct Place { long long mine; long long pool; long long scale; int sequence; bool has, good; };

__device__ __forceinline__ Place place(const RowArgs& a, int row, int layer) {
  const pi05_cache& c = a.c;
  const pi05_cache_rows& r = a.r;
  Place p;
  const int head = row % c.kv_heads, bt = row / c.kv_heads, t = bt % r.tokens, b = bt / r.tokens;
  p.sequence = b;
  p.mine = b * r.batch_stride + layer * r.layer_stride + t * r.token_stride + head * r.head_stride;
  p.has = !r.counts || t < __ldg(r.counts + b);
  const int start = r.starts ? __ldg(r.starts + b) : 0;
  const unsigned pos = (unsigned)start + (unsigned)t, lp = pos / (unsigned)c.page_tokens, at = pos - lp * (unsigned)c.page_tokens;
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

// Largest magnitude of a pair of BF16, NaN where there is one.
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Eight elements of a row as codes, and the row's scale.
//   code = rn(x * peak / a) of the true quotient, a the row's largest magnitude.  With BF16 x and a the quotient is either in the middle of
// two codes exactly (x = a / 2 is 63.5) or at least 2^-10 away from it, so it only has to be right to that, and exact in the middle: peak / a as
// the sum of two FP32 numbers, and x times it as one FMA on top of the small product, which rounds once.
template <int FORMAT, int LANES>
__device__ __forceinline__ uint2 encode(const uint4& x, float* scale) {
  constexpr float PEAK = FORMAT == PI05_CACHE_INT8 ? 127.0f : 448.0f;
  const uint32_t m = 0x7fff7fffu;
  uint32_t top = max_pair(max_pair(x.x & m, x.y & m), max_pair(x.z & m, x.w & m));
#pragma unroll
  for (int d = LANES / 2; d; d >>= 1) top = max_pair(top, __shfl_xor_sync(0xffffffffu, top, d));
  top = max_pair(top, top >> 16);                                  // (the shift brings zeros to the other half)
  float a = lo16(top);
  *scale = __fdiv_rn(a, PEAK);
  float v[8] = {lo16(x.x), hi16(x.x), lo16(x.y), hi16(x.y), lo16(x.z), hi16(x.z), lo16(x.w), hi16(x.w)};
  if (!(a > 0.f && a <= 3.3895314e38f)) {                          // nothing but zeros; an infinity or a NaN: the whole row reads back as NaN
    if (a != 0.f) *scale = __uint_as_float(0x7fffffffu);
    return make_uint2(0u, 0u);
  }
  if (!(a > 1e-30f && a < 1e30f)) {                                // keep peak / a and the products away from the ends of FP32: both times a power of two
    const float f = a < 1.f ? 0x1p+90f : 0x1p-90f;
    a *= f;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= f;
  }
  const float hi = __fdiv_rn(PEAK, a), lo = __fdiv_rn(fmaf(-hi, a, PEAK), a);
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = fmaf(v[4 * h + i], hi, v[4 * h + i] * lo);
    if (FORMAT == PI05_CACHE_INT8) {
      // to the nearest whole number, ties to even, by a sum whose last place is 1; its last byte is the code
      uint32_t n[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) n[i] = __float_as_uint(y[i] + 12582912.0f);
      w[h] = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
    } else {
      unsigned short p[2];
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p[0]) : "f"(y[1]), "f"(y[0]));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(p[1]) : "f"(y[3]), "f"(y[2]));
      w[h] = p[0] | (uint32_t)p[1] << 16;
    }
  }
  return make_uint2(w[0], w[1]);
}

template <int FORMAT, int DIM>
__global__ void __launch_bounds__(BLOCK) write_kernel(const __grid_constant__ RowArgs a) {
  constexpr int LANES = DIM / 8;
  const int lane = threadIdx.x % LANES, layer = blockIdx.y;
  const long long row = (long long)blockIdx.x * (BLOCK / LANES) + threadIdx.x / LANES;
  const bool in = row < a.rows;                                    // (every lane takes part in the shuffles)
  const Place p = place(a, in ? (int)row : 0, layer);
  const bool store = in && p.has && p.good;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  const __nv_bfloat16 *sk = static_cast<const __nv_bfloat16*>(a.r.k) + p.mine, *sv = static_cast<const __nv_bfloat16*>(a.r.v) + p.mine;
  const uint4 k = store ? __ldcs(reinterpret_cast<const uint4*>(sk) + lane) : zero, v = store ? __ldcs(reinterpret_cast<const uint4*>(sv) + lane) : zero;
  if constexpr (FORMAT == PI05_CACHE_BF16) {
    if (!store) return;
    reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.c.k) + p.pool)[lane] = k;
    reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.c.v) + p.pool)[lane] = v;
  } else {
    float ks, vs;
    const uint2 kc = encode<FORMAT, LANES>(k, &ks), vc = encode<FORMAT, LANES>(v, &vs);
    if (!store) return;
    reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.c.k) + p.pool)[lane] = kc;
    reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.c.v) + p.pool)[lane] = vc;
    if (lane == 0) { a.c.k_scale[p.scale] = ks; a.c.v_scale[p.scale] = vs; }
  }
}

template <int FORMAT>
__device__ __forceinline__ uint4 decode(const void* pool, long long at, int lane, float scale) {
  const uint2 w = __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + at) + lane);
  const uint2 a = cache::quad<FORMAT>(w.x), b = cache::quad<FORMAT>(w.y);
  return make_uint4(pack2(lo16(a.x) * scale, hi16(a.x) * scale), pack2(lo16(a.y) * scale, hi16(a.y) * scale),
                    pack2(lo16(b.x) * scale, hi16(b.x) * scale), pack2(lo16(b.y) * scale, hi16(b.y) * scale));
}

template <int FORMAT, int DIM>
__global__ void __launch_bounds__(BLOCK) read_kernel(const __grid_constant__ RowArgs a) {
  constexpr int LANES = DIM / 8;
  const int lane = threadIdx.x % LANES, layer = blockIdx.y;
  const long long row = (long long)blockIdx.x * (BLOCK / LANES) + threadIdx.x / LANES;
  if (row >= a.rows) return;
  const Place p = place(a, (int)row, layer);
  uint4 k = make_uint4(0u, 0u, 0u, 0u), v = k;
  if (p.has && p.good) {
    if constexpr (FORMAT == PI05_CACHE_BF16) {
      k = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.c.k) + p.pool) + lane);
      v = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.c.v) + p.pool) + lane);
    } else {
      k = decode<FORMAT>(a.c.k, p.pool, lane, __ldg(a.c.k_scale + p.scale));
      v = decode<FORMAT>(a.c.v, p.pool, lane, __ldg(a.c.v_scale + p.scale));
    }
  } else if (p.has) {
    k = v = make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu);      // no such page: NaN, so that nobody takes it for a key
  }
  __stcs(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.r.k) + p.mine) + lane, k);
  __stcs(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.r.v) + p.mine) + lane, v);
}

typedef void (*RowKernel)(const RowArgs);
#define BY_DIM(KERNEL, F) {KERNEL<F, 64>, KERNEL<F, 128>, KERNEL<F, 256>}
const RowKernel kWrite[3][3] = {BY_DIM(write_kernel, PI05_CACHE_BF16), BY_DIM(write_kernel, PI05_CACHE_INT8), BY_DIM(write_kernel, PI05_CACHE_E4M3)};
const RowKernel kRead[3][3] = {BY_DIM(read_kernel, PI05_CACHE_BF16), BY_DIM(read_kernel, PI05_CACHE_INT8), BY_DIM(read_kernel, PI05_CACHE_E4M3)};
#undef BY_DIM

struct DeviceGuard {
  int prev = -1;
  bool ok;
  explicit DeviceGuard(int dev) { if (cudaGetDevice(&prev) != cudaSuccess) prev = -1; ok = prev == dev || cudaSetDevice(dev) == cudaSuccess; }
  ~DeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};

int move_rows(const RowKernel (&kernels)[3][3], int device, const pi05_cache* c, const pi05_cache_rows* r, void* stream) {
  if (device < 0 || !cache::well_formed(c) || !r) return PI05_ERR_ARGUMENT;
  if (r->batch < 0 || r->tokens < 0 || r->layers < 0 || r->layer < 0 || r->layer > c->layers - r->layers || r->table_pages < 0 || r->table_stride < 0)
    return PI05_ERR_ARGUMENT;
  if (r->batch == 0 || r->tokens == 0 || r->layers == 0) return PI05_OK;
  const long long rows = (long long)r->batch * r->tokens * c->kv_heads;
  if (!r->k || !r->v || !r->table || rows > 0x7fffffffll || (long long)r->batch * r->tokens > 0x7fffffffll) return PI05_ERR_ARGUMENT;
  if ((((uintptr_t)r->k | (uintptr_t)r->v) & 15) || ((r->batch_stride | r->layer_stride | r->token_stride | r->head_stride) & 7) ||
      (((uintptr_t)r->table | (uintptr_t)r->starts | (uintptr_t)r->counts) & 3))
    return PI05_ERR_ARGUMENT;
  DeviceGuard guard(device);
  if (!guard.ok) { cudaGetLastError(); return PI05_ERR_NO_DEVICE; }
  const int per = BLOCK / (c->head_dim / 8);
  const RowArgs a = {*c, *r, rows};
  const RowKernel kernel = kernels[c->format][c->head_dim == 64 ? 0 : c->head_dim == 128 ? 1 : 2];
  kernel<<<dim3((unsigned)((rows + per - 1) / per), r->layers), BLOCK, 0, (cudaStream_t)stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? PI05_OK : PI05_ERR_CUDA;
}

}  // namespace

extern "C" {

int pi05_cache_write(int device, const pi05_cache* cache, const pi05_cache_rows* rows, void* stream) {
  return move_rows(kWrite, device, cache, rows, stream);
}

int pi05_cache_read(int device, const pi05_cache* cache, const pi05_cache_rows* rows, void* stream) {
  return move_rows(kRead, device, cache, rows, stream);
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
