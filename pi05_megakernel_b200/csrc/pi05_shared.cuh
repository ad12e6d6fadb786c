// Attention of several sequences over one shared prefix and their own tokens, out of the pages of a cache, on the tcgen05 tensor cores.
//
//   S = Q K^T (128 query rows x 64 keys), P = exp2(S c - m), O += P V (128 x head_dim), rows = lanes of tensor memory.
//
//   * Query rows of one KV head are packed into tiles of 128: of the whole batch against the prefix, so that its keys and values are read
//     once for 128 / (tokens x group) sequences, of one sequence against its own tokens.  Where a sequence fills its tiles by itself (`joined`)
//     prefix and own tokens are one list of keys and nothing has to be put together afterwards.
//   * Q, P, S and O all live in tensor memory (D = 256: 128 + 2 x 64 + 256 columns, P in place of S): both products take their A operand from
//     there, an MMA only reads its 64 keys or head_dim values from shared memory, and all of it is a ring of keys and values: what this
//     kernel mostly is bound by are the bytes of the cache.
//   * The list (item, tile of 64 keys) of a launch is one sequence, cut into equal ranges, one per CTA, whatever the lengths are
//     ("stream-K"): every CTA reads as many keys as any other.  A range that is not a whole item leaves unnormalised sums with their
//     reference and weight, which combine_kernel adds in a fixed order: results do not depend on who is first.
//   * Warp 0 copies (TMA), warp 1 issues the MMAs, warps 2 and 3 look pages and masks up ahead of both, warps 4-7 are the softmax, a
//     thread per query row, and of an 8-bit cache warps 8-15 turn codes into BF16, exactly (pi05_cache.cuh).  A key's scale multiplies its score, a
//     value's scale its probability, both in FP32.
//   * The reference m of a row only moves when a score is more than 2^RESCALE above it; then the row's sums in tensor memory are rescaled.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "pi05_cache.cuh"
#include "ptx_sm100.cuh"

namespace shared {

constexpr int TILE = 64;                    // keys of a tile
constexpr int ROWS = 128;                   // query rows of a tile
constexpr int INFO = 8;                     // tiles that pages and masks are looked up ahead
constexpr int OVERHEAD = 1;                 // what an item costs beside its tiles: loading Q, storing O
constexpr int MAX_BATCH = 1024;
constexpr float RESCALE = 8.0f;             // of exponents to the base 2: probabilities up to 256, their sums far from the ends of FP32

__host__ __device__ constexpr int unit_bytes(int dim) { return TILE * dim * 2; }
// Units (64 keys or values) of the BF16 ring and of the ring of codes in front of it.
__host__ __device__ constexpr int units(int format, int dim) { return format == PI05_CACHE_BF16 ? (dim == 256 ? 6 : 12) : 4; }
__host__ __device__ constexpr int raw_units(int format, int dim) { return format == PI05_CACHE_BF16 ? 0 : dim == 256 ? 5 : 10; }
__host__ __device__ constexpr int scale_bytes(int format) { return format == PI05_CACHE_BF16 ? 0 : INFO * 2 * TILE * 4; }
__host__ __device__ constexpr int smem_bytes(int format, int dim) {
  return units(format, dim) * unit_bytes(dim) + raw_units(format, dim) * TILE * dim + scale_bytes(format) + (MAX_BATCH + 1) * 8 + 1024;
}
__host__ __device__ constexpr int threads(int format) { return format == PI05_CACHE_BF16 ? 256 : 512; }

struct Args {
  CUtensorMap k, v;                         // BF16: {64 dims, page tokens, D / 64, heads, pages}; codes: {D, page tokens, heads, pages}
  pi05_cache c;
  pi05_shared_call s;
  int piece;                                // tokens of a copy: 64, 32 or 16, which divides the page
  int whole;                                // BF16: a copy brings all head_dim elements (pieces of 64 tokens), else 64 of them
  int group;                                // query heads per KV head
  int joined;
  int a_tiles;                              // row tiles of the batch against the prefix (not joined)
  int b_tiles, b_rows, b_slot;              // row tiles of one sequence, their rows, and those of a slot (a multiple of 4: it begins on 16 bytes)
  int p_tiles;                              // tiles of the prefix
  int grid;
  float c_log2;                             // scale x log2 e
  long long* plan;                          // what the combine kernel has to know: {units, CTAs, prefix sums of the sequences' units}
  float *a_parts, *b_parts;                 // slots of unfinished items: [D / 4][rows][4], then (reference, weight) per row
  long long limit;
};

enum { WAIT_INFO = 1, WAIT_INFO_EMPTY, WAIT_RAW_EMPTY, WAIT_RAW_FULL, WAIT_KV_EMPTY, WAIT_KV_FULL, WAIT_Q, WAIT_S, WAIT_S_FREE, WAIT_P, WAIT_PV, WAIT_SCALES };

// A run of tiles of one item.
struct Segment {
  bool batch;                               // rows of the whole batch against the prefix
  int h, b, r;                              // KV head, sequence, row tile
  int item;                                 // its number among those of its kind
  int first, n, tiles;                      // tiles first .. first + n of `tiles`
};

struct Walk {
  const long long* sums;                    // of the sequences' units, batch + 1
  long long a_cost, a_units, b_units, units;
  long long at, end;
  int ctas;

  __device__ __forceinline__ void set(const Args& p, const long long* s, int cta) {
    sums = s;
    a_cost = OVERHEAD + p.p_tiles;
    a_units = p.joined ? 0 : a_cost * p.a_tiles * p.c.kv_heads;
    b_units = s[p.s.batch];
    units = a_units + b_units * p.c.kv_heads;
    ctas = units < p.grid ? (int)units : p.grid;
    at = end = 0;
    if (cta < ctas) { at = units * cta / ctas; end = units * (cta + 1) / ctas; }
  }
  __device__ __forceinline__ int cta_of(long long unit) const { return (int)(((unit + 1) * ctas - 1) / units); }
  // The next run of this CTA that has tiles.
  __device__ __forceinline__ bool next(const Args& p, Segment& g) {
    while (at < end) {
      long long off, cost;
      if (at < a_units) {
        g.batch = true;
        g.item = (int)(at / a_cost);
        off = at - g.item * a_cost;
        cost = a_cost;
        g.h = g.item / p.a_tiles;
        g.r = g.item - g.h * p.a_tiles;
        g.b = 0;
        g.tiles = p.p_tiles;
      } else {
        g.batch = false;
        const long long u = at - a_units;
        g.h = (int)(u / b_units);
        const long long w = u - g.h * b_units;
        int lo = 0, hi = p.s.batch;         // the last sequence that begins at or before w (and has units)
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (sums[mid] <= w) lo = mid; else hi = mid;
        }
        g.b = lo;
        cost = (sums[lo + 1] - sums[lo]) / p.b_tiles;
        g.r = (int)((w - sums[lo]) / cost);
        off = w - sums[lo] - g.r * cost;
        g.item = (g.h * p.s.batch + g.b) * p.b_tiles + g.r;
        g.tiles = (int)cost - OVERHEAD;
      }
      const long long last = off + (end - at) < cost ? off + (end - at) : cost;      // units of the item before `end`
      g.first = off > OVERHEAD ? (int)off - OVERHEAD : 0;
      g.n = (int)last - OVERHEAD - g.first;
      at += last - off;
      if (g.n > 0) return true;
    }
    return false;
  }
};

// Which sequence, token and query head row `row` of a tile is; false: none.
__device__ __forceinline__ bool row_of(const Args& p, const Segment& g, int row, int& b, int& t, int& head) {
  int f;
  if (g.batch) {
    f = g.r * ROWS + row;
    if (f >= p.s.batch * p.s.tokens * p.group) return false;
  } else {
    f = g.r * p.b_rows + row;
    if (row >= p.b_rows || f >= p.s.tokens * p.group) return false;
  }
  const int bt = f / p.group;
  head = g.h * p.group + f - bt * p.group;
  b = g.batch ? bt / p.s.tokens : g.b;
  t = g.batch ? bt - b * p.s.tokens : bt;
  return true;
}

__device__ __forceinline__ int own_length(const Args& p, int b) {
  if (!p.s.table) return 0;
  const int n = __ldcg(p.s.lengths + b);
  const long long most = (long long)p.s.table_pages * p.c.page_tokens;
  return n < 0 ? 0 : n > most ? (int)most : n;
}

// A operand from tensor memory, B from shared memory: one MMA of K = 16.
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t blo, uint32_t idesc, uint32_t accumulate, uint32_t on) {
  asm volatile("{\n.reg .pred p, q;\n.reg .b64 db;\nsetp.ne.b32 p, %4, 0;\nsetp.ne.b32 q, %5, 0;\nmov.b64 db, {%2, %6};\n"
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}"
               ::"r"(d), "r"(a), "r"(blo), "r"(idesc), "r"(accumulate), "r"(on), "n"(ptx::UMMA_DESC_HI) : "memory");
}
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]) : "memory");
}
// Untiled copy of a multiple of 16 bytes between 16-byte boundaries.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// What warps 2 and 3 say about a tile.
struct Info {
  uint32_t mask[2];                         // keys that count
  uint32_t bad[2];                          // keys of pages that do not exist
  int page[4];                              // of the tile's pieces; -1: nothing to copy
};

template <int FORMAT, int DIM>
__global__ void __launch_bounds__(threads(FORMAT), 1) attention_kernel(const __grid_constant__ Args p) {
  constexpr bool CODES = FORMAT != PI05_CACHE_BF16;
  constexpr int UNITS = units(FORMAT, DIM), UNIT = unit_bytes(DIM), RAW = raw_units(FORMAT, DIM), RAW_UNIT = TILE * DIM, BLOCKS = DIM / 64;
  constexpr bool OVER = DIM == 256;         // P in place of S
  constexpr int TM_O = 0, TM_Q = DIM, TM_S = DIM + DIM / 2, TM_P = OVER ? TM_S : TM_S + 2 * TILE, P_STEP = OVER ? TILE : TILE / 2;
  constexpr int TM_COLS = 512;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * INFO + INFO + 2 * UNITS + 2 * (RAW ? RAW : 1) + 1 + 8];
  __shared__ Info s_info[INFO];
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t ring = ptx::smem_u32(smem), raw = ring + UNITS * UNIT, scales = raw + RAW * RAW_UNIT;
  long long* sums = reinterpret_cast<long long*>(smem + UNITS * UNIT + RAW * RAW_UNIT + scale_bytes(FORMAT));
  const float* s_scales = reinterpret_cast<const float*>(smem + UNITS * UNIT + RAW * RAW_UNIT);
  uint32_t bar = ptx::smem_u32(bars);
  auto take = [&](int n) { const uint32_t b = bar; bar += 8 * n; return b; };
  const uint32_t info_full = take(INFO), info_empty = take(INFO), scale_full = take(INFO), kv_full = take(UNITS), kv_empty = take(UNITS),
                 raw_full = take(RAW ? RAW : 1), raw_empty = take(RAW ? RAW : 1), q_full = take(1), s_full = take(2), s_free = take(2), p_full = take(2), pv_done = take(2);
  const bool leader = ptx::elect_one();

  if (warp == 0) {
    auto init = [&](uint32_t b, int n, int count) { for (int i = lane; i < n; i += 32) ptx::mbar_init(b + 8 * i, count); };
    init(info_full, INFO, 1); init(info_empty, INFO, 5); init(scale_full, INFO, 1);
    init(kv_full, UNITS, CODES ? 8 : 1); init(kv_empty, UNITS, 1); init(raw_full, RAW ? RAW : 1, 1); init(raw_empty, RAW ? RAW : 1, 8);
    init(q_full, 1, 4); init(s_full, 2, 1); init(s_free, 2, 4); init(p_full, 2, 4); init(pv_done, 2, 1);
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_shared();
    if (leader) { ptx::prefetch_tensormap(&p.k); ptx::prefetch_tensormap(&p.v); }
  } else if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), TM_COLS);
    ptx::tmem_relinquish();
  } else if (warp == 2) {
    // units of the sequences, added up
    ptx::grid_dep_wait();
    long long before = 0;
    if (lane == 0) sums[0] = 0;
    for (int b0 = 0; b0 < p.s.batch; b0 += 32) {
      const int b = b0 + lane;
      long long cost = 0;
      if (b < p.s.batch) {
        const int n = own_length(p, b);
        if (blockIdx.x == 0 && p.s.table && __ldcg(p.s.lengths + b) != n) cache::report(p.c.status, cache::BAD_POSITION, b);
        const int tiles = (p.joined ? p.p_tiles : 0) + (n + TILE - 1) / TILE;
        cost = tiles ? (long long)(OVERHEAD + tiles) * p.b_tiles : 0;
      }
      for (int d = 1; d < 32; d <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, cost, d);
        if (lane >= d) cost += up;
      }
      if (b < p.s.batch) sums[b + 1] = before + cost;
      before += __shfl_sync(0xffffffffu, cost, 31);
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::grid_dep_launch();
  const uint32_t tmem = s_tmem;
  Walk walk;
  walk.set(p, sums, blockIdx.x);
  if (blockIdx.x == 0) {
    for (int b = tid; b <= p.s.batch; b += blockDim.x) p.plan[2 + b] = sums[b];
    if (tid == 0) { p.plan[0] = walk.units; p.plan[1] = walk.ctas; }
  }
  // Where the keys and values of a segment's tile i of n stand among the segment's units: K0, K1, V0, K2, V1, .., K(n-1), V(n-2), V(n-1).
  auto k_unit = [](int i) { return i ? 2 * i - 1 : 0; };
  auto v_unit = [](int i, int n) { return i < n - 1 ? 2 * i + 2 : 2 * n - 1; };
  bool ok = true;
  Segment g;

  if (warp == 0) {
    // ---- copies
    uint32_t unit = 0, tile = 0;            // of all segments
    ptx::grid_dep_wait();
    while (ok && walk.next(p, g)) {
      auto copy = [&](int i, bool is_v) {
        const uint32_t n = tile + i, slot = n % INFO;
        if (!is_v) ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, info_full + 8 * slot, (n / INFO) & 1, WAIT_INFO);
        if (!ok) return;
        const Info& info = s_info[slot];
        const int pieces = TILE / p.piece;
        int page[4], there = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { page[j] = j < pieces ? info.page[j] : -1; there += page[j] >= 0; }
        constexpr int RING = CODES ? (RAW ? RAW : 1) : UNITS;
        const uint32_t full = CODES ? raw_full : kv_full, empty = CODES ? raw_empty : kv_empty, base = CODES ? raw : ring;
        const uint32_t at = unit % RING, round = unit / RING;
        ++unit;
        if (round) ok = ptx::wait_bar(p.c.status + 2, p.limit, empty + 8 * at, (round - 1) & 1, CODES ? WAIT_RAW_EMPTY : WAIT_KV_EMPTY);
        if (!ok) return;
        const uint32_t key = (uint32_t)(!g.batch && g.first + i >= (p.joined ? p.p_tiles : 0) ? g.first + i - (p.joined ? p.p_tiles : 0) : g.first + i) * TILE;
        if (leader) {
          const uint32_t bar = full + 8 * at, dst = base + at * (CODES ? RAW_UNIT : UNIT);
          const CUtensorMap* map = is_v ? &p.v : &p.k;
          ptx::mbar_expect_tx(bar, there * p.piece * DIM * (CODES ? 1 : 2));
          if (CODES && !is_v) ptx::mbar_expect_tx(scale_full + 8 * slot, there * p.piece * 8);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (page[j] < 0) continue;
            const int in = (int)((key + j * p.piece) % (unsigned)p.c.page_tokens);
            if constexpr (CODES) {
              ptx::tma_load_4d(dst + j * p.piece * DIM, map, bar, 0, in, g.h, page[j]);
              if (!is_v) {
                const long long sc = (((long long)page[j] * p.c.layers + p.s.layer) * p.c.kv_heads + g.h) * p.c.page_tokens + in;
                const uint32_t sd = scales + (slot * 2 * TILE + j * p.piece) * 4;
                bulk_load(sd, p.c.k_scale + sc, p.piece * 4, scale_full + 8 * slot);
                bulk_load(sd + TILE * 4, p.c.v_scale + sc, p.piece * 4, scale_full + 8 * slot);
              }
            } else if (p.whole) {
              ptx::tma_load_5d(dst, map, bar, 0, in, 0, g.h, page[j]);
            } else {
#pragma unroll 1
              for (int blk = 0; blk < BLOCKS; ++blk) ptx::tma_load_5d(dst + blk * TILE * 128 + j * p.piece * 128, map, bar, 0, in, blk, g.h, page[j]);
            }
          }
          if (is_v) ptx::mbar_arrive(info_empty + 8 * slot);
        }
        __syncwarp();
      };
      copy(0, false);
      for (int i = 1; i < g.n && ok; ++i) { copy(i, false); copy(i - 1, true); }
      copy(g.n - 1, true);
      tile += g.n;
    }
  } else if (warp == 1) {
    // ---- MMAs
    const uint32_t on = leader ? 1u : 0u;
    const uint32_t idesc_s = ptx::umma_idesc_bf16(ROWS, TILE), idesc_o = ptx::umma_idesc_bf16(ROWS, DIM) | ptx::UMMA_B_MN_MAJOR;
    const uint32_t kdesc = (uint32_t)ptx::umma_smem_desc(ring), vdesc = (uint32_t)ptx::umma_smem_desc_mn(ring, TILE * 128);
    uint32_t unit = 0, tile = 0, seg = 0;
    while (ok && walk.next(p, g)) {
      ok = ptx::wait_bar(p.c.status + 2, p.limit, q_full, seg & 1, WAIT_Q);
      ptx::tc_fence_after();
      ++seg;
      auto scores = [&](int i) {
        const uint32_t n = tile + i, buf = n & 1, u = unit + k_unit(i), at = u % UNITS;
        if (n > 1) ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, (OVER ? pv_done : s_free) + 8 * buf, ((n >> 1) - 1) & 1, OVER ? WAIT_PV : WAIT_S_FREE);
        ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, kv_full + 8 * at, (u / UNITS) & 1, WAIT_KV_FULL);
        if (!ok) return;
        ptx::tc_fence_after();
        const uint32_t kd = kdesc + at * (UNIT >> 4);
#pragma unroll
        for (int j = 0; j < DIM / 16; ++j)
          umma_ts(tmem + TM_S + buf * TILE, tmem + TM_Q + 8 * j, kd + (j >> 2) * (TILE * 128 >> 4) + (j & 3) * 2, idesc_s, j ? 1u : 0u, on);
        if (leader) { ptx::umma_commit(kv_empty + 8 * at); ptx::umma_commit(s_full + 8 * buf); }
        __syncwarp();
      };
      auto products = [&](int i) {
        const uint32_t n = tile + i, buf = n & 1, u = unit + v_unit(i, g.n), at = u % UNITS;
        ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, kv_full + 8 * at, (u / UNITS) & 1, WAIT_KV_FULL);
        ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, p_full + 8 * buf, (n >> 1) & 1, WAIT_P);
        if (!ok) return;
        ptx::tc_fence_after();
        const uint32_t vd = vdesc + at * (UNIT >> 4);
#pragma unroll
        for (int j = 0; j < TILE / 16; ++j)
          umma_ts(tmem + TM_O, tmem + TM_P + buf * P_STEP + 8 * j, vd + j * (16 * 128 >> 4), idesc_o, i || j ? 1u : 0u, on);
        if (leader) { ptx::umma_commit(kv_empty + 8 * at); ptx::umma_commit(pv_done + 8 * buf); }
        __syncwarp();
      };
      if (ok) scores(0);
      for (int i = 1; i < g.n && ok; ++i) { scores(i); products(i - 1); }
      if (ok) products(g.n - 1);
      unit += 2 * g.n;
      tile += g.n;
    }
  } else if (warp < 4) {
    // ---- pages and masks, every second tile each
    uint32_t tile = 0;
    while (ok && walk.next(p, g)) {
      const int p_tiles = g.batch || p.joined ? p.p_tiles : 0, length = g.batch ? 0 : own_length(p, g.b);
      for (int i = 0; i < g.n && ok; ++i) {
        const uint32_t n = tile + i, slot = n % INFO;
        if ((n & 1) != (uint32_t)(warp & 1)) continue;
        const bool own = g.first + i >= p_tiles;
        const uint32_t key = (uint32_t)(own ? g.first + i - p_tiles : g.first + i) * TILE;
        const uint32_t end = own ? length : p.s.prefix_tokens;
        const int* table = own ? p.s.table + (long long)g.b * p.s.table_stride : p.s.prefix_table;
        const uint32_t first = key + lane * p.piece;
        int page = -1;
        bool bad = false;
        if (lane < TILE / p.piece && first < end) {
          page = __ldcg(table + first / (unsigned)p.c.page_tokens);
          bad = page < 0 || page >= p.c.pages;
          if (bad) { page = -1; cache::report(p.c.status, cache::BAD_PAGE, own ? g.b : -1); }
        }
        bool c0 = key + lane < end, c1 = key + 32 + lane < end;
        if (!own && p.s.prefix_valid) {
          c0 = c0 && __ldcg(p.s.prefix_valid + key + lane);
          c1 = c1 && __ldcg(p.s.prefix_valid + key + 32 + lane);
        }
        const unsigned lost = __ballot_sync(0xffffffffu, bad);
        const bool b0 = lost >> (lane / p.piece) & 1, b1 = lost >> ((lane + 32) / p.piece) & 1;
        const unsigned m0 = __ballot_sync(0xffffffffu, c0), m1 = __ballot_sync(0xffffffffu, c1), l0 = __ballot_sync(0xffffffffu, b0 && c0),
                       l1 = __ballot_sync(0xffffffffu, b1 && c1);
        if (n >= INFO) ok = ptx::wait_bar(p.c.status + 2, p.limit, info_empty + 8 * slot, (n / INFO - 1) & 1, WAIT_INFO_EMPTY);
        if (!ok) break;
        Info& info = s_info[slot];
        if (lane < 4) info.page[lane] = page;
        if (lane == 0) { info.mask[0] = m0; info.mask[1] = m1; info.bad[0] = l0; info.bad[1] = l1; }
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(info_full + 8 * slot);
        __syncwarp();
      }
      tile += g.n;
    }
  } else if (warp < 8) {
    // ---- softmax: thread = query row.  A wait that gave up lets the rest run through, with NaN as the result
    const int quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    uint32_t unit = 0, tile = 0;
    const uint4* q = nullptr;
    int sees = 0;                           // own tokens that the row sees
    bool mine = false;
    int b = 0, t = 0, head = 0;
    ptx::grid_dep_wait();
    while (walk.next(p, g)) {
      mine = row_of(p, g, row, b, t, head);
      q = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.s.q) + b * p.s.q_batch_stride + t * p.s.q_token_stride + head * p.s.q_head_stride);
#pragma unroll 1
      for (int c = 0; c < DIM / 64; ++c) {
        uint32_t w[32];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint4 x = mine ? __ldcg(q + c * 8 + j) : make_uint4(0u, 0u, 0u, 0u);
          w[4 * j] = x.x; w[4 * j + 1] = x.y; w[4 * j + 2] = x.z; w[4 * j + 3] = x.w;
        }
        tmem_st_32x32(lanes + TM_Q + 32 * c, w);
      }
      ptx::tmem_wait_st();
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(q_full);
      __syncwarp();
      const int p_tiles = g.batch || p.joined ? p.p_tiles : 0, length = g.batch ? 0 : own_length(p, g.b);
      sees = p.s.causal ? length - p.s.tokens + t + 1 : length;
      float m = -INFINITY, l = 0.f;         // reference (of exponents to the base 2) and sum
#pragma unroll 1
      for (int i = 0; i < g.n; ++i) {
        const uint32_t n = tile + i, buf = n & 1, slot = n % INFO;
        ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, info_full + 8 * slot, (n / INFO) & 1, WAIT_INFO);
        if (CODES) ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, scale_full + 8 * slot, (n / INFO) & 1, WAIT_SCALES);
        const uint32_t mask0 = s_info[slot].mask[0], mask1 = s_info[slot].mask[1], bad0 = s_info[slot].bad[0], bad1 = s_info[slot].bad[1];
        uint32_t k0 = mask0, k1 = mask1;    // keys that count for this row
        if (g.first + i >= p_tiles) {
          const long long left = sees - (long long)(g.first + i - p_tiles) * TILE;
          k0 &= left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
          k1 &= left >= 64 ? 0xffffffffu : left > 32 ? (1u << (left - 32)) - 1u : 0u;
        }
        const bool special = __any_sync(0xffffffffu, (k0 & k1) != 0xffffffffu || (bad0 | bad1));
        ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, s_full + 8 * buf, (n >> 1) & 1, WAIT_S);
        ptx::tc_fence_after();
        float x[64];
        ptx::tmem_ld_32x32(lanes + TM_S + buf * TILE, *reinterpret_cast<uint32_t(*)[32]>(&x[0]));
        ptx::tmem_ld_32x32(lanes + TM_S + buf * TILE + 32, *reinterpret_cast<uint32_t(*)[32]>(&x[32]));
        ptx::tmem_wait_ld();
        if (!OVER) {
          ptx::tc_fence_before();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(s_free + 8 * buf);
          __syncwarp();
        }
        const float4* ks = reinterpret_cast<const float4*>(s_scales + slot * 2 * TILE);
        if (CODES) {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float4 f = ks[j];
            x[4 * j] *= f.x; x[4 * j + 1] *= f.y; x[4 * j + 2] *= f.z; x[4 * j + 3] *= f.w;
          }
        }
        if (special) {
#pragma unroll
          for (int j = 0; j < 64; ++j) {
            if (!((j < 32 ? k0 : k1) >> (j & 31) & 1)) x[j] = -INFINITY;
            else if ((j < 32 ? bad0 : bad1) >> (j & 31) & 1) x[j] = __uint_as_float(0x7fffffffu);
          }
        }
        float top[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int j = 4; j < 64; ++j) top[j & 3] = fmaxf(top[j & 3], x[j]);
        const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.c_log2;
        if (i == 0) {
          m = high;
        } else {
          const bool move = high > m + RESCALE;
          if (__any_sync(0xffffffffu, move)) {
            const float f = move ? ptx::ex2_approx(m - high) : 1.f;
            if (move) m = high;
            l *= f;
            ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, pv_done + 8 * (buf ^ 1), ((n - 1) >> 1) & 1, WAIT_PV);
            ptx::tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < DIM; c += 32) {
              uint32_t o[32];
              ptx::tmem_ld_32x32(lanes + TM_O + c, o);
              ptx::tmem_wait_ld();
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st_32x32(lanes + TM_O + c, o);
            }
            ptx::tmem_wait_st();
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[32];
#pragma unroll
        for (int j = 0; j < 64; j += 4) {
          float e[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) { e[k] = ptx::ex2_approx(fmaf(x[j + k], p.c_log2, -ref)); sum[k] += e[k]; }
          if (CODES) {
            const float4 f = ks[16 + j / 4];
            e[0] *= f.x; e[1] *= f.y; e[2] *= f.z; e[3] *= f.w;
            if (special)
#pragma unroll
              for (int k = 0; k < 4; ++k) e[k] = (j < 32 ? k0 : k1) >> ((j + k) & 31) & 1 ? e[k] : 0.f;
          }
          pk[j / 2] = cache::pack2(e[0], e[1]);
          pk[j / 2 + 1] = cache::pack2(e[2], e[3]);
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if (!OVER && n > 1) {               // the buffer of P is free once the product before the last has read it
          ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, pv_done + 8 * buf, ((n >> 1) - 1) & 1, WAIT_PV);
          ptx::tc_fence_after();
        }
        tmem_st_32x32(lanes + TM_P + buf * P_STEP, pk);
        ptx::tmem_wait_st();
        if (!CODES && (mask0 & mask1 & ~(bad0 | bad1)) != 0xffffffffu) {
          // values at places that do not count are whatever memory holds, and 0 x NaN is NaN: zeros in their place
          const uint32_t u = unit + v_unit(i, g.n), at = u % UNITS;
          ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, kv_full + 8 * at, (u / UNITS) & 1, WAIT_KV_FULL);
          const uint32_t z0 = ~mask0 | bad0, z1 = ~mask1 | bad1;
          for (int c = row; c < TILE * DIM / 8; c += 128) {
            const int key = c & 63, chunk = c >> 6;
            if ((key < 32 ? z0 : z1) >> (key & 31) & 1) ptx::st_shared_v4(ring + at * UNIT + (chunk >> 3) * (TILE * 128) + key * 128 + (chunk & 7) * 16, 0u, 0u, 0u, 0u);
          }
          ptx::fence_proxy_async_shared();
        }
        __syncwarp();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) { ptx::mbar_arrive(p_full + 8 * buf); ptx::mbar_arrive(info_empty + 8 * slot); }
        __syncwarp();
      }
      unit += 2 * g.n;
      tile += g.n;
      // ---- the segment's sums
      ok = ok && ptx::wait_bar(p.c.status + 2, p.limit, pv_done + 8 * ((tile - 1) & 1), ((tile - 1) >> 1) & 1, WAIT_PV);
      ptx::tc_fence_after();
      if (!ok) l = __uint_as_float(0x7fffffffu);
      if (!g.batch && p.joined && g.n == g.tiles) {
        const float il = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;        // (no key: zeros; NaN stays)
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.s.out) + b * p.s.out_batch_stride + t * p.s.out_token_stride + head * p.s.out_head_stride;
#pragma unroll 1
        for (int c = 0; c < DIM; c += 32) {
          uint32_t o[32];
          ptx::tmem_ld_32x32(lanes + TM_O + c, o);
          ptx::tmem_wait_ld();
          if (mine)
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              *reinterpret_cast<uint4*>(out + c + j) = make_uint4(
                  cache::pack2(__uint_as_float(o[j]) * il, __uint_as_float(o[j + 1]) * il), cache::pack2(__uint_as_float(o[j + 2]) * il, __uint_as_float(o[j + 3]) * il),
                  cache::pack2(__uint_as_float(o[j + 4]) * il, __uint_as_float(o[j + 5]) * il), cache::pack2(__uint_as_float(o[j + 6]) * il, __uint_as_float(o[j + 7]) * il));
          __syncwarp();
        }
        if (mine && p.s.lse) p.s.lse[((long long)b * p.s.tokens + t) * p.s.q_heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      } else {
        const int rows = g.batch ? ROWS : p.b_slot;
        float* part = (g.batch ? p.a_parts : p.b_parts) + (long long)(blockIdx.x + g.item) * rows * (DIM + 2);
#pragma unroll 1
        for (int c = 0; c < DIM; c += 32) {
          uint32_t o[32];
          ptx::tmem_ld_32x32(lanes + TM_O + c, o);
          ptx::tmem_wait_ld();
          if (mine)
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              __stcg(reinterpret_cast<uint4*>(part) + ((c + j) / 4) * rows + row, make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]));
          __syncwarp();
        }
        if (mine) __stcg(reinterpret_cast<float2*>(part + DIM * rows) + row, make_float2(m, l));
      }
      ptx::tc_fence_before();
      __syncwarp();
    }
  } else if constexpr (CODES) {
    // ---- codes to BF16: 16 codes per thread and turn, to two 16-byte chunks of the swizzled unit.  Eight neighbouring lanes take 64 bytes
    // of an even row and the other 64 of the odd one, so that neither the loads nor the stores share banks
    const int w = warp - 8, odd = lane >> 2 & 1, chunk = lane & 3, high = lane >> 3;
    const int blk = BLOCKS == 4 ? high ^ odd : BLOCKS == 2 ? (high & 1) ^ odd : 0;
    constexpr int AT_ONCE = 8 / BLOCKS;     // rows of a warp's turn
    const int first = odd + (BLOCKS == 4 ? 0 : BLOCKS == 2 ? (high >> 1) * 2 : high * 2);
    uint32_t unit = 0;
    while (ok && walk.next(p, g)) {
      for (int i = 0; i < 2 * g.n && ok; ++i, ++unit) {
        const uint32_t from = unit % RAW, to = unit % UNITS;
        ok = ptx::wait_bar(p.c.status + 2, p.limit, raw_full + 8 * from, (unit / RAW) & 1, WAIT_RAW_FULL);
        if (ok && unit >= UNITS) ok = ptx::wait_bar(p.c.status + 2, p.limit, kv_empty + 8 * to, (unit / UNITS - 1) & 1, WAIT_KV_EMPTY);
        if (!ok) break;
        constexpr int TURNS = TILE / AT_ONCE / 8;
        uint4 x[TURNS];
#pragma unroll
        for (int j = 0; j < TURNS; ++j) x[j] = ptx::ld_shared_v4(raw + from * RAW_UNIT + ((j * 8 + w) * AT_ONCE + first) * DIM + blk * 64 + chunk * 16);
#pragma unroll
        for (int j = 0; j < TURNS; ++j) {
          const int r = (j * 8 + w) * AT_ONCE + first;
          const uint2 a = cache::quad<FORMAT>(x[j].x), c = cache::quad<FORMAT>(x[j].y), d = cache::quad<FORMAT>(x[j].z), e = cache::quad<FORMAT>(x[j].w);
          const uint32_t line = ring + to * UNIT + blk * (TILE * 128) + r * 128;
          ptx::st_shared_v4(line + (((2 * chunk) ^ (r & 7)) << 4), a.x, a.y, c.x, c.y);
          ptx::st_shared_v4(line + (((2 * chunk + 1) ^ (r & 7)) << 4), d.x, d.y, e.x, e.y);
        }
        ptx::fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) { ptx::mbar_arrive(kv_full + 8 * to); ptx::mbar_arrive(raw_empty + 8 * from); }
        __syncwarp();
      }
    }
  }
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, TM_COLS);
  }
}

// The unfinished items of a launch put together: a warp has eight query rows x 16 dims, of which `split` warps of a block take every split-th
// part each.
template <int DIM>
__global__ void __launch_bounds__(256) combine_kernel(const __grid_constant__ Args p, int split) {
  __shared__ float s_m[8][8], s_l[8][8];
  __shared__ float4 s_o[8][32];
  ptx::grid_dep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, share = warp % split;
  const int flat = p.s.batch * p.s.tokens * p.group, groups = (flat + 7) / 8;
  const long long work = (long long)blockIdx.x * (8 / split) + warp / split;
  const int column = (int)(work % (DIM / 16)) * 4 + (lane & 3);          // of four dims
  const long long hg = work / (DIM / 16);
  const int h = (int)(hg / groups), f = (int)(hg % groups) * 8 + row;
  const bool in = h < p.c.kv_heads && f < flat;
  const int bt = f / p.group, gi = f - bt * p.group, b = bt / p.s.tokens, t = bt - b * p.s.tokens;
  Walk walk;
  walk.a_cost = OVERHEAD + p.p_tiles;
  walk.a_units = p.joined ? 0 : walk.a_cost * p.a_tiles * p.c.kv_heads;
  walk.units = __ldcg(p.plan);
  walk.ctas = (int)__ldcg(p.plan + 1);
  // parts a0 .. a0 + na - 1 of the prefix, b0 .. b0 + nb - 1 of the sequence's own item
  int a0 = 0, na = 0, b0 = 0, nb = 0, b_row = 0;
  bool done = false;                        // one CTA had it all
  if (in) {
    if (!p.joined && p.p_tiles) {
      const int item = h * p.a_tiles + f / ROWS;
      const long long u = item * walk.a_cost + OVERHEAD;
      const int c0 = walk.cta_of(u);
      na = walk.cta_of(u + p.p_tiles - 1) - c0 + 1;
      a0 = c0 + item;
    }
    const long long s0 = __ldcg(p.plan + 2 + b), s1 = __ldcg(p.plan + 3 + b);
    if (s1 > s0) {
      const int fs = f - b * p.s.tokens * p.group, r = fs / p.b_rows, item = (h * p.s.batch + b) * p.b_tiles + r;
      b_row = fs - r * p.b_rows;
      const long long cost = (s1 - s0) / p.b_tiles, u = walk.a_units + h * __ldcg(p.plan + 2 + p.s.batch) + s0 + r * cost + OVERHEAD;
      const int c0 = walk.cta_of(u);
      nb = walk.cta_of(u + cost - OVERHEAD - 1) - c0 + 1;
      b0 = c0 + item;
      done = p.joined && nb == 1;
    }
  }
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float2 ml, float4 v) {
    const float top = fmaxf(m, ml.x), w0 = m == top ? 1.f : ptx::ex2_approx(m - top), w1 = ml.x == top ? 1.f : ptx::ex2_approx(ml.x - top);
    l = l * w0 + ml.y * w1;
    o.x = o.x * w0 + v.x * w1; o.y = o.y * w0 + v.y * w1; o.z = o.z * w0 + v.z * w1; o.w = o.w * w0 + v.w * w1;
    m = top;
  };
  if (!done) {
#pragma unroll 4
    for (int k = share; k < na + nb; k += split) {
      const bool own = k >= na;
      const int rows = own ? p.b_slot : ROWS, r = own ? b_row : f % ROWS;
      const float* part = (own ? p.b_parts : p.a_parts) + (long long)(own ? b0 + k - na : a0 + k) * rows * (DIM + 2);
      const float4 v = __ldcg(reinterpret_cast<const float4*>(part) + column * rows + r);
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(part + DIM * rows) + r);
      add(ml, v);
    }
  }
  if (split > 1) {
    if ((lane & 3) == 0) { s_m[warp][row] = m; s_l[warp][row] = l; }
    s_o[warp][lane] = o;
    __syncthreads();
    if (share) return;
    for (int k = 1; k < split; ++k) add(make_float2(s_m[warp + k][row], s_l[warp + k][row]), s_o[warp + k][lane]);
  }
  if (!in || done) return;
  const float il = l == 0.f ? 0.f : 1.0f / l;
  const int head = h * p.group + gi;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.s.out) + b * p.s.out_batch_stride + t * p.s.out_token_stride + head * p.s.out_head_stride;
  *reinterpret_cast<uint2*>(out + column * 4) = make_uint2(cache::pack2(o.x * il, o.y * il), cache::pack2(o.z * il, o.w * il));
  if (column == 0 && p.s.lse) p.s.lse[((long long)b * p.s.tokens + t) * p.s.q_heads + head] = l == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m) + log2f(l)) * 0.6931471805599453f;
}

}  // namespace shared
