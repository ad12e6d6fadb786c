// Attention of several sequences over one shared prefix and their own tokens, out of the pages of a cache.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/pi05_b200.h"
#include "pi05_cache.cuh"
#include "ptx_sm100.cuh"

namespace {

constexpr int WARPS = 8;

struct SharedArgs {
  pi05_cache c;
  pi05_shared_call s;
};

// One block per query row: its warps take every eighth key each, a lane DIM / 32 dims, and the parts are merged at the end.
template <int FORMAT, int DIM>
__global__ void __launch_bounds__(32 * WARPS) rows_kernel(const __grid_constant__ SharedArgs a) {
  constexpr int E = DIM / 32;
  const pi05_cache& c = a.c;
  const pi05_shared_call& s = a.s;
  __shared__ float s_m[WARPS], s_l[WARPS], s_o[WARPS][DIM];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x % s.q_heads, bt = blockIdx.x / s.q_heads, t = bt % s.tokens, b = bt / s.tokens;
  const int kh = h / (s.q_heads / c.kv_heads);
  int length = s.table ? __ldg(s.lengths + b) : 0;
  const long long most = (long long)s.table_pages * c.page_tokens;
  if (length < 0 || length > most) {
    if (threadIdx.x == 0) cache::report(c.status, cache::BAD_POSITION, b);
    length = length < 0 ? 0 : (int)most;
  }
  int sees = s.causal ? length - s.tokens + t + 1 : length;
  if (sees < 0) sees = 0;
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(s.q) + b * s.q_batch_stride + t * s.q_token_stride + h * s.q_head_stride;
  float qv[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) { qv[e] = __bfloat162float(q[lane * E + e]); o[e] = 0.f; }
  auto value = [&](const void* pool, long long at, float scale, int e) {
    if (FORMAT == PI05_CACHE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(pool)[at + e]);
    const uint32_t w = static_cast<const uint8_t*>(pool)[at + e];
    return cache::lo16(cache::pair<FORMAT == PI05_CACHE_BF16 ? PI05_CACHE_INT8 : FORMAT>(w)) * scale;
  };
  for (int j = warp; j < s.prefix_tokens + sees; j += WARPS) {
    const bool own = j >= s.prefix_tokens;
    if (!own && s.prefix_valid && !s.prefix_valid[j]) continue;
    const int pos = own ? j - s.prefix_tokens : j, lp = pos / c.page_tokens, in = pos - lp * c.page_tokens;
    const int page = own ? __ldg(s.table + (long long)b * s.table_stride + lp) : __ldg(s.prefix_table + lp);
    if (page < 0 || page >= c.pages) {
      if (lane == 0) cache::report(c.status, cache::BAD_PAGE, own ? b : -1);
      m = l = NAN;
      continue;
    }
    const long long pl = (long long)page * c.layers + s.layer;
    const long long at = ((pl * c.page_tokens + in) * c.kv_heads + kh) * DIM + lane * E, sc = (pl * c.kv_heads + kh) * c.page_tokens + in;
    const float ks = FORMAT == PI05_CACHE_BF16 ? 1.f : c.k_scale[sc], vs = FORMAT == PI05_CACHE_BF16 ? 1.f : c.v_scale[sc];
    float x = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) x += qv[e] * value(c.k, at, ks, e);
#pragma unroll
    for (int d = 16; d; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    x *= s.scale;
    const float top = fmaxf(m, x), f = expf(m - top), p = expf(x - top);
    m = top;
    l = l * f + p;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * f + p * value(c.v, at, vs, e);
  }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = o[e];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < WARPS; ++w) M = fmaxf(M, s_m[w]);
  for (int w = 0; w < WARPS; ++w) L += s_m[w] == -INFINITY ? 0.f : s_l[w] * expf(s_m[w] - M);
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(s.out) + b * s.out_batch_stride + t * s.out_token_stride + h * s.out_head_stride;
  for (int d = threadIdx.x; d < DIM; d += 32 * WARPS) {
    float v = 0.f;
    for (int w = 0; w < WARPS; ++w) v += s_m[w] == -INFINITY ? 0.f : s_o[w][d] * expf(s_m[w] - M);
    out[d] = __float2bfloat16_rn(M == -INFINITY ? 0.f : v / L);
  }
  if (threadIdx.x == 0 && s.lse) s.lse[blockIdx.x] = M == -INFINITY ? -INFINITY : M + logf(L);
}

typedef void (*RowsKernel)(const SharedArgs);
#define BY_DIM(F) {rows_kernel<F, 64>, rows_kernel<F, 128>, rows_kernel<F, 256>}
const RowsKernel kRows[3][3] = {BY_DIM(PI05_CACHE_BF16), BY_DIM(PI05_CACHE_INT8), BY_DIM(PI05_CACHE_E4M3)};
#undef BY_DIM

struct DeviceGuard {
  int prev = -1;
  bool ok;
  explicit DeviceGuard(int dev) { if (cudaGetDevice(&prev) != cudaSuccess) prev = -1; ok = prev == dev || cudaSetDevice(dev) == cudaSuccess; }
  ~DeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};

}  // namespace

extern "C" {

int pi05_shared_workspace(int sms, const pi05_cache* cache, int q_heads, int max_batch, int max_tokens, size_t* bytes) {
  if (sms < 1 || sms > 1024 || !cache::well_formed(cache) || q_heads < 1 || q_heads % cache->kv_heads || max_batch < 1 || max_tokens < 1 || !bytes)
    return PI05_ERR_ARGUMENT;
  *bytes = 256;
  return PI05_OK;
}

int pi05_shared_attention(int device, const pi05_cache* cache, const pi05_shared_call* call, void* workspace, size_t workspace_bytes, void* stream) {
  if (device < 0 || !cache::well_formed(cache) || !call) return PI05_ERR_ARGUMENT;
  const pi05_shared_call& s = *call;
  if (s.batch < 0 || s.tokens < 0 || s.q_heads < 1 || s.q_heads % cache->kv_heads || s.layer < 0 || s.layer >= cache->layers || s.prefix_tokens < 0)
    return PI05_ERR_ARGUMENT;
  if (s.batch == 0 || s.tokens == 0) return PI05_OK;
  if (!s.q || !s.out || (s.prefix_tokens && !s.prefix_table) || (s.table && (!s.lengths || s.table_pages < 0 || s.table_stride < 0))) return PI05_ERR_ARGUMENT;
  if ((((uintptr_t)s.q | (uintptr_t)s.out) & 15) ||
      ((s.q_batch_stride | s.q_token_stride | s.q_head_stride | s.out_batch_stride | s.out_token_stride | s.out_head_stride) & 7) ||
      (((uintptr_t)s.lse | (uintptr_t)s.prefix_table | (uintptr_t)s.table | (uintptr_t)s.lengths) & 3))
    return PI05_ERR_ARGUMENT;
  DeviceGuard guard(device);
  if (!guard.ok) { cudaGetLastError(); return PI05_ERR_NO_DEVICE; }
  const SharedArgs a = {*cache, s};
  const RowsKernel kernel = kRows[cache->format][cache->head_dim == 64 ? 0 : cache->head_dim == 128 ? 1 : 2];
  kernel<<<s.batch * s.tokens * s.q_heads, 32 * WARPS, 0, (cudaStream_t)stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? PI05_OK : PI05_ERR_CUDA;
}

}  // extern "C"
