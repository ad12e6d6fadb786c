// Host side of the attention over a shared prefix: how a call is cut, tensor maps, launches.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>

#include "../../include/pi05_b200.h"
#include "pi05_ops.h"
#include "pi05_shared.cuh"

namespace {

using cache::DeviceGuard;
using shared::Args;

typedef void (*AttentionKernel)(const Args);
typedef void (*CombineKernel)(const Args, int);
#define BY_DIM(F) {shared::attention_kernel<F, 64>, shared::attention_kernel<F, 128>, shared::attention_kernel<F, 256>}
const AttentionKernel kAttention[3][3] = {BY_DIM(PI05_CACHE_BF16), BY_DIM(PI05_CACHE_INT8), BY_DIM(PI05_CACHE_E4M3)};
#undef BY_DIM
const CombineKernel kCombine[3] = {shared::combine_kernel<64>, shared::combine_kernel<128>, shared::combine_kernel<256>};

int dim_index(int dim) { return dim == 64 ? 0 : dim == 128 ? 1 : 2; }
long long up256(long long v) { return (v + 255) / 256 * 256; }

// Tiles of query rows, and what unfinished items may leave behind: a slot per CTA and per item (a CTA's run ends at most one item early).
struct Cut { long long a_tiles, b_tiles, b_rows, b_slot, a_bytes, b_bytes, plan_bytes; };
Cut cut_rows(int sms, const pi05_cache& c, int q_heads, long long batch, long long tokens) {
  const long long rows = tokens * (q_heads / c.kv_heads);
  Cut k;
  k.a_tiles = (batch * rows + shared::ROWS - 1) / shared::ROWS;
  k.b_tiles = (rows + shared::ROWS - 1) / shared::ROWS;
  k.b_rows = (rows + k.b_tiles - 1) / k.b_tiles;
  k.b_slot = (k.b_rows + 3) / 4 * 4;
  k.plan_bytes = up256((k.a_tiles + batch * k.b_tiles) * c.kv_heads * 8);
  k.a_bytes = up256((sms + k.a_tiles * c.kv_heads) * shared::ROWS * (c.head_dim + 2) * 4);
  k.b_bytes = up256((sms + k.b_tiles * batch * c.kv_heads) * k.b_slot * (c.head_dim + 2) * 4);
  return k;
}

}  // namespace

extern "C" {

int pi05_shared_workspace(int sms, const pi05_cache* cache, int q_heads, int max_batch, int max_tokens, size_t* bytes) {
  if (sms < 1 || sms > 1024 || !cache::well_formed(cache) || q_heads < 1 || q_heads % cache->kv_heads || max_batch < 1 || max_tokens < 1 || !bytes)
    return PI05_ERR_ARGUMENT;
  if (max_batch > shared::MAX_BATCH || (long long)max_batch * max_tokens * q_heads > 1ll << 27) return PI05_ERR_UNSUPPORTED;
  const Cut k = cut_rows(sms, *cache, q_heads, max_batch, max_tokens);
  // fewer tokens may make the tiles of a sequence taller, up to all rows
  const long long rows = std::min<long long>(shared::ROWS, ((long long)max_tokens * (q_heads / cache->kv_heads) + 3) / 4 * 4);
  *bytes = (size_t)(k.plan_bytes + k.a_bytes + up256((sms + k.b_tiles * max_batch * cache->kv_heads) * rows * (cache->head_dim + 2) * 4));
  return PI05_OK;
}

int pi05_shared_attention(int device, const pi05_cache* cache, const pi05_shared_call* call, void* workspace, size_t workspace_bytes, void* stream_) {
  if (device < 0 || device >= 64 || !cache::well_formed(cache) || !call) return PI05_ERR_ARGUMENT;
  const pi05_cache& c = *cache;
  const pi05_shared_call& s = *call;
  if (s.batch < 0 || s.tokens < 0 || s.q_heads < 1 || s.q_heads % c.kv_heads || s.layer < 0 || s.layer >= c.layers || s.prefix_tokens < 0)
    return PI05_ERR_ARGUMENT;
  if (s.batch == 0 || s.tokens == 0) return PI05_OK;
  if (!s.q || !s.out || !workspace || (s.prefix_tokens && !s.prefix_table) || (s.table && (!s.lengths || s.table_pages < 0 || s.table_stride < 0)))
    return PI05_ERR_ARGUMENT;
  if ((((uintptr_t)s.q | (uintptr_t)s.out) & 15) || ((uintptr_t)workspace & 255) ||
      ((s.q_batch_stride | s.q_token_stride | s.q_head_stride | s.out_batch_stride | s.out_token_stride | s.out_head_stride) & 7) ||
      (((uintptr_t)s.lse | (uintptr_t)s.prefix_table | (uintptr_t)s.table | (uintptr_t)s.lengths) & 3) || !(s.scale > 0.f && s.scale < INFINITY))
    return PI05_ERR_ARGUMENT;
  if (s.batch > shared::MAX_BATCH || (long long)s.batch * s.tokens * s.q_heads > 1ll << 27) return PI05_ERR_UNSUPPORTED;
  // places of keys are counted in 32 bits, in whole tiles: far enough from their end that rounding up does not pass it
  if (s.prefix_tokens > 1 << 30 || (s.table && (long long)s.table_pages * c.page_tokens > 1ll << 30)) return PI05_ERR_UNSUPPORTED;
  {                                             // outputs on one another, or over queries that another CTA has yet to read
    const long long size[3] = {s.batch, s.tokens, s.q_heads}, os[3] = {s.out_batch_stride, s.out_token_stride, s.out_head_stride},
                    qs[3] = {s.q_batch_stride, s.q_token_stride, s.q_head_stride};
    const long long apart = (long long)((intptr_t)s.out - (intptr_t)s.q) / 2;
    if (cache::rows_meet(3, size, os, nullptr, nullptr, 0, c.head_dim) || cache::rows_meet(3, size, qs, size, os, apart, c.head_dim)) return PI05_ERR_ARGUMENT;
  }
  DeviceGuard guard(device);
  int sms = 0;
  if (!guard.ok || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) { cudaGetLastError(); return PI05_ERR_NO_DEVICE; }
  const Cut k = cut_rows(sms, c, s.q_heads, s.batch, s.tokens);
  if ((long long)workspace_bytes < k.plan_bytes + k.a_bytes + k.b_bytes) return PI05_ERR_ARGUMENT;

  Args a;
  memset(&a, 0, sizeof a);
  a.c = c; a.s = s;
  a.group = s.q_heads / c.kv_heads;
  a.piece = c.page_tokens % 64 == 0 ? 64 : c.page_tokens % 32 == 0 ? 32 : 16;
  a.a_tiles = (int)k.a_tiles; a.b_tiles = (int)k.b_tiles; a.b_rows = (int)k.b_rows; a.b_slot = (int)k.b_slot;
  a.overhead = shared::overhead(c.format);
  a.p_tiles = (s.prefix_tokens + shared::TILE - 1) / shared::TILE;
  // Prefix and own tokens as one list of keys where packing the batch's rows would not save a quarter of the tiles.  8 heads of 256, one list / packed, in us
  // (BF16; int8): 16 x 50 over 200 31.8 / 37.5; 34.9 / 36.4, over 968 40.3 / 42.8; 45.2 / 47.9, over 4000 60.9 / 67.7; 77.1 / 73.2.  8 x 50 over 968 26.3 / 26.7;
  // 31.0 / 31.5, over 4000 39.8 / 40.5; 47.2 / 45.3.  Where packing saves more it still is up to 17% slower for a few sequences (8 x 20 over 968 23.1 / 24.4;
  // 26.2 / 27.7, 2 x 8 over 200 13.2 / 15.5; 15.2 / 17.6), but it is what makes the prefix one pass for many of a token each
  a.joined = a.p_tiles == 0 || 3ll * s.batch * k.b_tiles <= 4 * k.a_tiles;
  const long long own = s.table ? ((long long)s.table_pages * c.page_tokens + shared::TILE - 1) / shared::TILE : 0;
  const long long most = c.kv_heads * ((a.joined ? 0 : k.a_tiles * (a.overhead + a.p_tiles)) +
                                       s.batch * k.b_tiles * (a.overhead + own + (a.joined ? a.p_tiles : 0)));
  if (most > 0x3fffffffll) return PI05_ERR_UNSUPPORTED;
  a.grid = (int)std::min<long long>(sms, most);
  a.c_log2 = s.scale * 1.4426950408889634f;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.parts = reinterpret_cast<int2*>(ws);
  a.a_parts = reinterpret_cast<float*>(ws + k.plan_bytes);
  a.b_parts = reinterpret_cast<float*>(ws + k.plan_bytes + k.a_bytes);
  a.limit = 2000000000u;                        // about a second
  if (!pi05::map_pages(&a.k, c.k, c.format != PI05_CACHE_BF16, c.head_dim, c.page_tokens, c.kv_heads, c.layers, c.pages, s.layer, a.piece) ||
      !pi05::map_pages(&a.v, c.v, c.format != PI05_CACHE_BF16, c.head_dim, c.page_tokens, c.kv_heads, c.layers, c.pages, s.layer, a.piece))
    return PI05_ERR_CUDA;

  const int d = dim_index(c.head_dim);
  const AttentionKernel attention = kAttention[c.format][d];
  const CombineKernel combine = kCombine[d];
  const int smem = shared::smem_bytes(c.format, c.head_dim);
  static std::atomic<uint64_t> done[3][3];
  cudaError_t e = pi05::once_per_device(&done[c.format][d], device, [&] {
    const cudaError_t first = pi05::chain_opt_in((const void*)attention, smem);
    return first == cudaSuccess ? pi05::chain_opt_in((const void*)combine, 0) : first;
  });
  cudaStream_t stream = (cudaStream_t)stream_;
  if (e == cudaSuccess) e = pi05::launch_kernel(attention, a.grid, shared::threads(c.format), smem, stream, 1, true, a);
  // A row's parts are added by one warp, or by up to sixteen of a block where there are many: as many as leave each no more than it loads at once
  const long long items = c.kv_heads * (a.joined ? s.batch * k.b_tiles : k.a_tiles), tiles = a.p_tiles + own;
  const long long parts = std::min(a.grid / items + 2, tiles);
  int split = 1;
  while (split < shared::COMBINE_THREADS / 32 && parts > split * shared::AT_ONCE) split *= 2;
  const long long work = (long long)c.kv_heads * (((long long)s.batch * s.tokens * a.group + 7) / 8) * (c.head_dim / 16);
  const int per = shared::COMBINE_THREADS / 32 / split;
  if (e == cudaSuccess) e = pi05::launch_kernel(combine, dim3((unsigned)((work + per - 1) / per)), shared::COMBINE_THREADS, 0, stream, 1, true, a, split);
  if (e != cudaSuccess) { cudaGetLastError(); return PI05_ERR_CUDA; }
  return PI05_OK;
}

}  // extern "C"
