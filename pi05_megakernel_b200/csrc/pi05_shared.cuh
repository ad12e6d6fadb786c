// Attention of several sequences over one shared prefix and their own tokens, out of the pages of a cache, on the tcgen05 tensor cores.
//
//   S = Q K^T (128 query rows x 64 keys), P = exp2(S c - m), O += P V (128 x head_dim), rows = lanes of tensor memory.
//
//   * Query rows of one KV head are packed into tiles of 128: of the whole batch against the prefix, so that its keys and values are read
//     once for 128 / (tokens x group) sequences, of one sequence against its own tokens.  Where a sequence fills its tiles by itself (`joined`)
//     prefix and own tokens are one list of keys.
//   * Q, P, S and O all live in tensor memory (D = 256: 128 + 2 x 64 + 256 columns, P in place of S): both products take their A operand from
//     there, an MMA only reads its 64 keys or head_dim values from shared memory, and all of it is a ring of keys and values: what this
//     kernel mostly is bound by are the bytes of the cache.
//   * The list (item, tile of 64 keys) of a launch is one sequence, cut into equal ranges, one per CTA, whatever the lengths are
//     ("stream-K"): every CTA reads as many keys as any other.  A range that is not a whole item leaves unnormalised sums with their
//     reference and weight, which combine_kernel adds in a fixed order: results do not depend on who is first.
//   * Warp 0 copies (TMA), warp 1 issues the MMAs, warp 2 looks pages and masks up ahead of both.  Two groups of four warps are the softmax, a
//     thread per query row, and take the tiles in turn: what a tile costs a group is mostly latency (tensor memory, barriers, the special
//     functions of one warp per scheduler), which the other group's tile hides.  They share the reference m of a row, which goes from tile to
//     tile in order; it only moves when an exponent to the base 2 is more than RESCALE above it, and then the row's sums in tensor memory are rescaled.
//   * Of an 8-bit cache two more groups turn codes into 16 bits, exactly: keys into BF16, as the queries are, values into FP16.  A key's scale
//     multiplies its score and a value's scale its probability, both in FP32.  The product, rounded to FP16, keeps three bits more than
//     BF16 would; so that it stays in FP16's range whatever the scales are, the reference of a row is the largest exponent of such a product, of a key that
//     the row sees: max_j (y_j + log2 s_j), with the logarithms of the values' scales by warp 3, once a tile.  A shift that the division by the row's sum
//     takes out again.  What is below 2^-21 of the row's largest product loses bits to FP16's subnormals.  (In BF16 the outputs were 0.0025 off the definition,
//     relative to 0.0017 of their own rounding; now 0.0017.)
//
// What bounds it (one B200, both kernels): 64 sequences over 16384 tokens in BF16 78 us beside 31 of HBM, 224 MB read at 2.9 TB/s, tensor pipe 24%: the chain of a tile
// through one group (2800 cycles for 64 keys) and the latency of 512 short items; drafts in e4m3 122 us beside 21 of tensor pipe: instructions of softmax and
// converters; steps of a few sequences 12 to 18 us: launch, lengths, page lookup, first bytes, one tile, its parts and the second kernel, one after the other.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <stdint.h>

#include "pi05_cache.cuh"
#include "ptx_sm100.cuh"

namespace shared {

constexpr int TILE = 64;                    // keys of a tile
constexpr int ROWS = 128;                   // query rows of a tile
constexpr int INFO = 16;                    // tiles that pages and masks are looked up ahead, in
constexpr int BATCH = 8;                    // rounds of
// What an item costs beside its tiles (loading Q, filling the pipeline, storing O), in tiles.  Times in us with 2 / 3 / 4 / 5 / 6:
//                                                         BF16                        int8 (e4m3 within 1 us of it)
//   drafts, 32 x 8 over 8192, heads of 128    109 / 99 / 92 / 88 / 90                 142 / 128 / 118 / 121 / 118
//   the same, 4 heads of 256                   78 / 70 / 69 / 69 / 68                  91 / 86 / 86 / 86 / 87
//   the same, heads of 64                      85 / 78 / 75 / 77 / 79                 118 / 108 / 100 / 106 / 105
//   64 x 1 over 16384, heads of 128            80 / 79 / 82 / 84 / 88                 119 / 115 / 111 / 112 / 122
//   64 x 1 over 8192, 2 heads of 256           46 / 44 / 44 / 44 / 45                  54 / 53 / 53 / 53 / 54
//   13 x 1 over 30001, one head of 256         27 / 27 / 25 / 25 / 25                  32 / 32 / 30 / 30 / 30
// 3 and 5 are within 12% of the best of every row.
__host__ __device__ constexpr int overhead(int format) { return format == PI05_CACHE_BF16 ? 3 : 5; }
constexpr int MAX_BATCH = 1024;
constexpr float RESCALE = 8.0f;             // of exponents to the base 2: probabilities up to 256, their sums far from the ends of FP32
// Of 8 bits: what is added to the logarithm of a value's scale, so that its products with probabilities are up to 2^7, 2^15 before the reference moves; and
// the smallest such logarithm, which keeps 2^30 probabilities of up to 2^(80 + 7 + 8) in FP32 (of values below 1e-22 bits are lost instead).
constexpr float LOG_SHIFT = -7.0f, LOG_LEAST = -80.0f;

__host__ __device__ constexpr int unit_bytes(int dim) { return TILE * dim * 2; }
// Units (64 keys or values) of the BF16 ring and of the ring of codes in front of it.
__host__ __device__ constexpr int units(int format, int dim) { return format == PI05_CACHE_BF16 ? (dim == 256 ? 6 : 12) : dim == 256 ? 4 : 8; }
__host__ __device__ constexpr int raw_units(int format, int dim) { return format == PI05_CACHE_BF16 ? 0 : dim == 256 ? 4 : 8; }
// Of a tile: its keys' scales, its values', and the logarithms of the latter.
__host__ __device__ constexpr int scale_bytes(int format) { return format == PI05_CACHE_BF16 ? 0 : INFO * 3 * TILE * 4; }
__host__ __device__ constexpr int smem_bytes(int format, int dim) {
  return units(format, dim) * unit_bytes(dim) + raw_units(format, dim) * TILE * dim + scale_bytes(format) + (2 * MAX_BATCH + 1) * 4 + 1024;
}
__host__ __device__ constexpr int threads(int format) { return format == PI05_CACHE_BF16 ? 384 : 640; }

struct Args {
  CUtensorMap k, v;                         // BF16: {64 dims, page tokens, D / 64, heads, pages}; codes: {D, page tokens, heads, pages}
  pi05_cache c;
  pi05_shared_call s;
  int piece;                                // tokens of a copy: 64, 32 or 16, which divides the page
  int group;                                // query heads per KV head
  int joined;
  int a_tiles;                              // row tiles of the batch against the prefix (not joined)
  int b_tiles, b_rows, b_slot;              // row tiles of one sequence, their rows, and those of a slot (a multiple of 4: it begins on 16 bytes)
  int p_tiles;                              // tiles of the prefix
  int grid;
  float c_log2;                             // scale x log2 e
  int2* parts;                              // of every item, the batch's before the sequences': its first slot, and how many there are (0 or 1 that was finished: none to add)
  float *a_parts, *b_parts;                 // slots of unfinished items: [D / 4][rows][4], then (reference, weight) per row
  int overhead;                             // units of an item beside its tiles
  uint32_t limit;                           // of a wait, in cycles
};

enum { WAIT_INFO = 1, WAIT_INFO_EMPTY, WAIT_RAW_EMPTY, WAIT_RAW_FULL, WAIT_KV_EMPTY, WAIT_KV_FULL, WAIT_Q, WAIT_S, WAIT_S_FREE, WAIT_P, WAIT_PV, WAIT_SCALES, WAIT_O_FREE };

// A run of tiles of one item.
struct Segment {
  bool batch;                               // rows of the whole batch against the prefix
  int h, b, r;                              // KV head, sequence, row tile
  int item;                                 // its number among those of its kind
  int first, n, tiles;                      // tiles first .. first + n of `tiles`
};

// The launch's sequence of units: how it is cut, and where it comes from.
struct Walk {
  const int* sums;                          // of the sequences' units, batch + 1
  int a_cost, a_units, b_units, units, ctas;
  int each, more;                           // units of a CTA; the first `more` have one more

  __device__ __forceinline__ void cut(int u, int c) {
    units = u; ctas = c;
    each = c ? u / c : 0;
    more = u - each * c;
  }
  __device__ __forceinline__ int begin(int cta) const { return cta < ctas ? cta * each + (cta < more ? cta : more) : units; }
  __device__ __forceinline__ int cta_of(int unit) const {
    const int big = more * (each + 1);
    return unit < big ? unit / (each + 1) : more + (unit - big) / each;
  }
  __device__ __forceinline__ void set(const Args& p, const int* s) {
    sums = s;
    a_cost = p.overhead + p.p_tiles;
    a_units = p.joined ? 0 : a_cost * p.a_tiles * p.c.kv_heads;
    b_units = s[p.s.batch];
    const int u = a_units + b_units * p.c.kv_heads;
    cut(u, u < p.grid ? u : p.grid);
  }
};

// The next run of this CTA that has tiles, from unit `at` on, to *out, by a whole warp; returns the unit behind it, or -1: there is none.  (One function
// for all warps: what they execute does not fit the instruction cache many times.)
static __device__ __noinline__ int next_segment(const Args& p, const Walk& w, int at, Segment* out) {
  const int end = w.begin(blockIdx.x + 1);
  Segment g;
  g.n = 0;
  while (at < end && g.n <= 0) {
    int off, cost;
    if (at < w.a_units) {
      g.batch = true;
      g.item = at / w.a_cost;
      off = at - g.item * w.a_cost;
      cost = w.a_cost;
      g.h = g.item / p.a_tiles;
      g.r = g.item - g.h * p.a_tiles;
      g.b = 0;
      g.tiles = p.p_tiles;
    } else {
      g.batch = false;
      const int u = at - w.a_units;
      g.h = u / w.b_units;
      const int x = u - g.h * w.b_units;
      int lo = 0, hi = p.s.batch;           // the last sequence that begins at or before x (and has units)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (w.sums[mid] <= x) lo = mid; else hi = mid;
      }
      g.b = lo;
      off = x - w.sums[lo];
      cost = w.sums[lo + 1] - w.sums[lo];
      g.r = 0;
      if (p.b_tiles > 1) { cost /= p.b_tiles; g.r = off / cost; off -= g.r * cost; }
      g.item = (g.h * p.s.batch + g.b) * p.b_tiles + g.r;
      g.tiles = cost - p.overhead;
    }
    const int last = off + (end - at) < cost ? off + (end - at) : cost;      // units of the item before `end`
    g.first = off > p.overhead ? off - p.overhead : 0;
    g.n = last - p.overhead - g.first;
    at += last - off;
  }
  __syncwarp();
  if (g.n > 0 && (threadIdx.x & 31) == 0) *out = g;
  __syncwarp();
  return g.n > 0 ? at : -1;
}

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

// Four MMAs of K = 16, the A operand from tensor memory, B from shared memory: 8 columns and STEP descriptor units further each.
template <int STEP>
__device__ __forceinline__ void umma_ts4(uint32_t d, uint32_t a, uint32_t blo, uint32_t idesc, uint32_t accumulate) {
#define PI05_UMMA1(P0) "mov.b64 db, {bl, %5};\ntcgen05.mma.cta_group::1.kind::f16 [%0], [aa], db, %3, " P0 ";\n"
#define PI05_UMMA_STEP "add.u32 bl, bl, %6;\n add.u32 aa, aa, 8;\n"
  asm volatile("{\n.reg .pred p, t;\n.reg .b32 aa, bl;\n.reg .b64 db;\nsetp.ne.b32 p, %4, 0;\nsetp.eq.b32 t, 0, 0;\n"
               "mov.b32 aa, %1;\nmov.b32 bl, %2;\n" PI05_UMMA1("p") PI05_UMMA_STEP PI05_UMMA1("t") PI05_UMMA_STEP PI05_UMMA1("t") PI05_UMMA_STEP PI05_UMMA1("t") "}"
               ::"r"(d), "r"(a), "r"(blo), "r"(idesc), "r"(accumulate), "n"(ptx::UMMA_DESC_HI), "n"(STEP) : "memory");
#undef PI05_UMMA1
#undef PI05_UMMA_STEP
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

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long ra, rb, rd;
  asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(rd));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long ra, rb, rd;
  asm("mov.b64 %0, {%1, %2};" : "=l"(ra) : "f"(a.x), "f"(a.y));
  asm("mov.b64 %0, {%1, %2};" : "=l"(rb) : "f"(b.x), "f"(b.y));
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(rd) : "l"(ra), "l"(rb));
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(rd));
  return d;
}

// Bounded wait of a converged warp on a barrier; one that gives up is reported and returns when what the CTA may still have in flight has finished.
static __device__ __noinline__ bool wait_slow(const Args& p, uint32_t bar, uint32_t parity, int kind) {
  const uint32_t t0 = (uint32_t)clock();
#pragma unroll 1
  do {
    if (__all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity))) return true;
  } while (!__any_sync(0xffffffffu, (uint32_t)clock() - t0 > p.limit));
  if ((threadIdx.x & 31) == 0 && atomicCAS(p.c.status + 2, 0u, (unsigned)kind) == 0u) p.c.status[3] = blockIdx.x << 16;
  const uint32_t t1 = (uint32_t)clock();
  while ((uint32_t)clock() - t1 < 200000u) __nanosleep(1000);
  __syncwarp();
  return false;
}
__device__ __forceinline__ bool wait(const Args& p, uint32_t bar, uint32_t parity, int kind) {
  return __all_sync(0xffffffffu, ptx::mbar_try_wait(bar, parity)) || wait_slow(p, bar, parity, kind);
}

// The same for one thread of a warp.
static __device__ __noinline__ bool wait_one_slow(const Args& p, uint32_t bar, uint32_t parity, int kind) {
  const uint32_t t0 = (uint32_t)clock();
#pragma unroll 1
  do {
    if (ptx::mbar_try_wait(bar, parity)) return true;
  } while ((uint32_t)clock() - t0 <= p.limit);
  if (atomicCAS(p.c.status + 2, 0u, (unsigned)kind) == 0u) p.c.status[3] = blockIdx.x << 16;
  const uint32_t t1 = (uint32_t)clock();
  while ((uint32_t)clock() - t1 < 200000u) __nanosleep(1000);
  return false;
}
__device__ __forceinline__ bool wait_one(const Args& p, uint32_t bar, uint32_t parity, int kind) {
  return ptx::mbar_try_wait(bar, parity) || wait_one_slow(p, bar, parity, kind);
}

// The queries of a softmax warp's 32 rows, as they lie, into tensor memory.
template <int DIM>
__device__ __noinline__ void load_queries(const Args& p, const Segment& s, int row, uint32_t columns) {
  int b = 0, t = 0, head = 0;
  const bool mine = row_of(p, s, row, b, t, head);
  const uint4* q = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p.s.q) + b * p.s.q_batch_stride + t * p.s.q_token_stride + head * p.s.q_head_stride);
  constexpr int WORDS = DIM >= 128 ? 64 : 32;                      // on their way at once
#pragma unroll 1
  for (int c = 0; c < DIM / 2; c += WORDS) {
    uint32_t w[WORDS];
#pragma unroll
    for (int j = 0; j < WORDS / 4; ++j) {
      const uint4 x = mine ? __ldcg(q + c / 4 + j) : make_uint4(0u, 0u, 0u, 0u);
      w[4 * j] = x.x; w[4 * j + 1] = x.y; w[4 * j + 2] = x.z; w[4 * j + 3] = x.w;
    }
#pragma unroll
    for (int j = 0; j < WORDS; j += 32) tmem_st_32x32(columns + c + j, reinterpret_cast<uint32_t(&)[32]>(w[j]));
  }
  ptx::tmem_wait_st();
  ptx::tc_fence_before();
  __syncwarp();
}

// What warp 2 says about a tile.
struct Info {
  uint32_t mask[2];                         // keys that count
  uint32_t bad[2];                          // keys of pages that do not exist
  int page[4], in[4];                       // page and place of the tile's pieces; page -1: nothing to copy
  long long scale[4];                       // of their first scales
  int there;                                // pieces to copy
};

template <int FORMAT, int DIM>
__global__ void __launch_bounds__(threads(FORMAT), 1) attention_kernel(const __grid_constant__ Args p) {
  constexpr bool CODES = FORMAT != PI05_CACHE_BF16;
  constexpr int UNITS = units(FORMAT, DIM), UNIT = unit_bytes(DIM), RAW = CODES ? raw_units(FORMAT, DIM) : 1, RAW_UNIT = TILE * DIM, BLOCKS = DIM / 64;
  constexpr bool OVER = DIM == 256;         // P in place of S
  // S is ahead of P V by LOOK tiles; where there is room in tensor memory the next segment's queries have columns of their own
  constexpr int LOOK = OVER ? 1 : 2, S_BUFS = LOOK + 1, Q_BUFS = OVER ? 1 : 2;
  constexpr int TM_O = 0, TM_Q = DIM, TM_S = TM_Q + Q_BUFS * DIM / 2, TM_P = OVER ? TM_S : TM_S + S_BUFS * TILE, P_STEP = OVER ? TILE : TILE / 2;
  static_assert(TM_P + 2 * P_STEP <= 512, "tensor memory");
  constexpr int TM_COLS = 512;
  constexpr int CHUNK = CODES ? 16 : 32;    // scores that a softmax thread takes at a time: the code of an 8-bit cache's warps is the longer one
  constexpr int TOKEN = 1, END = 9, LOST = 13;      // named barriers: of a pair of softmax warps, reference handed on (by group), end of a segment; of a group
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[4 * INFO + 2 * UNITS + 2 * RAW + Q_BUFS + 2 * S_BUFS + 5];
  __shared__ Info s_info[INFO];
  __shared__ uint32_t s_bad[INFO][2];       // Info::bad and the keys whose value's scale is not a number
  __shared__ float s_ref[2][ROWS];          // the rows' references, by segment
  __shared__ float2 s_ml[2][2][ROWS];       // at its end: the groups' references and sums
  __shared__ Segment s_seg[threads(FORMAT) / 32], s_ahead[8];      // a warp's segment; a softmax warp's next one
  __shared__ Walk s_walk;
  __shared__ uint32_t s_lost[2][2][2];      // by group, and by turn of its ragged tiles: keys of one whose values are not all numbers
  __shared__ __align__(16) float s_ones[CODES ? TILE : 1];
  __shared__ uint32_t s_tmem;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int AT_SCALES = UNITS * UNIT + (CODES ? RAW * RAW_UNIT : 0), AT_SUMS = AT_SCALES + scale_bytes(FORMAT);
  const uint32_t ring = ptx::smem_u32(smem), raw = ring + UNITS * UNIT, scales = ring + AT_SCALES;
  int* sums = reinterpret_cast<int*>(smem + AT_SUMS);
  int* lengths = sums + MAX_BATCH + 1;
  const float* s_scales = reinterpret_cast<const float*>(smem + AT_SCALES);
  uint32_t bar = ptx::smem_u32(bars);
  auto take = [&](int n) { const uint32_t b = bar; bar += 8 * n; return b; };
  const uint32_t info_full = take(INFO), info_empty = take(INFO), scale_full = take(INFO), vlog_full = take(INFO), kv_full = take(UNITS),
                 kv_empty = take(UNITS), raw_full = take(RAW), raw_empty = take(RAW), q_full = take(Q_BUFS), o_free = take(1),
                 s_full = take(S_BUFS), s_free = take(S_BUFS), p_full = take(2), pv_done = take(2);
  const bool leader = ptx::elect_one();
#define WAIT(BAR, PARITY, KIND) wait(p, BAR, PARITY, KIND)
#define WAIT_ONE(BAR, PARITY, KIND) wait_one(p, BAR, PARITY, KIND)

  if (CODES && tid < TILE) s_ones[tid] = 1.f;
  if (!CODES && tid < 8) (&s_lost[0][0][0])[tid] = 0u;
  if (warp == 0) {
    auto init = [&](uint32_t b, int n, int count) { for (int i = lane; i < n; i += 32) ptx::mbar_init(b + 8 * i, count); };
    init(info_full, INFO, 1); init(info_empty, INFO, CODES ? 6 : 5); init(scale_full, INFO, 1); init(vlog_full, INFO, 1);
    init(kv_full, UNITS, CODES ? 4 : 1); init(kv_empty, UNITS, 1); init(raw_full, RAW, 1); init(raw_empty, RAW, 4);
    init(q_full, Q_BUFS, 4); init(o_free, 1, 8); init(s_full, S_BUFS, 1); init(s_free, S_BUFS, 4); init(p_full, 2, 4); init(pv_done, 2, 1);
    ptx::fence_mbar_init();
    ptx::fence_proxy_async_shared();
    if (leader) { ptx::prefetch_tensormap(&p.k); ptx::prefetch_tensormap(&p.v); }
  } else if (warp == 1) {
    ptx::tmem_alloc(ptx::smem_u32(&s_tmem), TM_COLS);
    ptx::tmem_relinquish();
  } else if (warp == 2) {
    // units of the sequences, added up
    ptx::grid_dep_wait();
    int before = 0;
    if (lane == 0) sums[0] = 0;
    for (int b0 = 0; b0 < p.s.batch; b0 += 32) {
      const int b = b0 + lane;
      int cost = 0;
      if (b < p.s.batch) {
        const int n = own_length(p, b);
        if (blockIdx.x == 0 && p.s.table && __ldcg(p.s.lengths + b) != n) cache::report(p.c.status, cache::BAD_POSITION, b);
        lengths[b] = n;
        const int tiles = (p.joined ? p.p_tiles : 0) + (n + TILE - 1) / TILE;
        cost = tiles ? (p.overhead + tiles) * p.b_tiles : 0;
      }
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, cost, d);
        if (lane >= d) cost += up;
      }
      if (b < p.s.batch) sums[b + 1] = before + cost;
      before += __shfl_sync(0xffffffffu, cost, 31);
    }
    __syncwarp();
    if (lane == 0) s_walk.set(p, sums);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  ptx::grid_dep_launch();
  const uint32_t tmem = s_tmem;
  const Walk& walk = s_walk;
  // Where the keys and values of a segment's tile i of n stand among the segment's units, which is the order of their use: LOOK = 1: K0, K1, V0,
  // K2, V1, .., V(n-1); 2: K0, K1, K2, V0, K3, V1, .., V(n-2), V(n-1).  And what unit u is.
  auto k_unit = [](int i) { return i < LOOK ? i : 2 * i - LOOK; };
  auto v_unit = [](int i, int n) { return i < n - LOOK ? 2 * i + 1 + LOOK : n + i; };
  auto what = [](int u, int n, bool& is_v) {
    if (u < LOOK && u < n) { is_v = false; return u; }
    if (u >= 2 * n - LOOK) { is_v = true; return u - n; }
    is_v = (u + LOOK) & 1;
    return is_v ? (u - 1 - LOOK) >> 1 : (u + LOOK) >> 1;
  };
  bool ok = true;
  const Segment& g = s_seg[warp];
  int at_unit = walk.begin(blockIdx.x);
#define NEXT ((at_unit = next_segment(p, walk, at_unit, &s_seg[warp])) >= 0)

  if (warp < 4) {
    if (warp == 0) {
      // ---- copies, by one thread
      uint32_t unit = 0, tile = 0;            // of all segments
      const int pieces = TILE / p.piece;
      ptx::grid_dep_wait();
      while (ok && NEXT) {
        if (leader) {
          const int units_here = 2 * g.n, h = g.h;
#pragma unroll 1
          for (int u = 0; u < units_here; ++u, ++unit) {
            bool is_v;
            const uint32_t n = tile + what(u, g.n, is_v), slot = n % INFO;
            constexpr int RING = CODES ? RAW : UNITS;
            const uint32_t at = unit % RING, round = unit / RING, full = (CODES ? raw_full : kv_full) + 8 * at;
            if (!is_v) ok = WAIT_ONE(info_full + 8 * slot, (n / INFO) & 1, WAIT_INFO);
            if (ok && round) ok = WAIT_ONE((CODES ? raw_empty : kv_empty) + 8 * at, (round - 1) & 1, CODES ? WAIT_RAW_EMPTY : WAIT_KV_EMPTY);
            if (!ok) break;
            const Info& info = s_info[slot];
            const int there = info.there * p.piece;
            const CUtensorMap* map = is_v ? &p.v : &p.k;
            const uint32_t dst = CODES ? raw + at * RAW_UNIT : ring + at * UNIT;
            ptx::mbar_expect_tx(full, there * DIM * (CODES ? 1 : 2));
            if (CODES && !is_v) ptx::mbar_expect_tx(scale_full + 8 * slot, there * 8);
#pragma unroll 1
            for (int j = 0; j < pieces; ++j) {
              const int page = info.page[j], in = info.in[j];
              if (page < 0) continue;
              if constexpr (CODES) {
                ptx::tma_load_4d(dst + j * p.piece * DIM, map, full, 0, in, h, page);
                if (!is_v) {
                  const uint32_t to = scales + (slot * 3 * TILE + j * p.piece) * 4;
                  bulk_load(to, p.c.k_scale + info.scale[j], p.piece * 4, scale_full + 8 * slot);
                  bulk_load(to + TILE * 4, p.c.v_scale + info.scale[j], p.piece * 4, scale_full + 8 * slot);
                }
              } else if (pieces == 1) {
                ptx::tma_load_5d(dst, map, full, 0, in, 0, h, page);
              } else {
#pragma unroll 1
                for (int blk = 0; blk < BLOCKS; ++blk) ptx::tma_load_5d(dst + blk * TILE * 128 + j * p.piece * 128, map, full, 0, in, blk, h, page);
              }
            }
            if (is_v) ptx::mbar_arrive(info_empty + 8 * slot);
          }
        }
        __syncwarp();
        ok = __any_sync(0xffffffffu, leader && ok);
        tile += g.n;
      }
    } else if (warp == 1) {
      // ---- MMAs, by one thread
      const uint32_t idesc_s = ptx::umma_idesc_bf16(ROWS, TILE);
      const uint32_t idesc_o = (ptx::umma_idesc_bf16(ROWS, DIM) & (CODES ? ~((1u << 7) | (1u << 10)) : ~0u)) | ptx::UMMA_B_MN_MAJOR;     // (FP16 is type 0)
      const uint32_t kdesc = (uint32_t)ptx::umma_smem_desc(ring), vdesc = (uint32_t)ptx::umma_smem_desc_mn(ring, TILE * 128);
      uint32_t unit = 0, tile = 0, seg = 0;
      while (ok && NEXT) {
        if (leader) {
          ok = WAIT_ONE(q_full + 8 * (seg % Q_BUFS), (seg / Q_BUFS) & 1, WAIT_Q);
          ptx::tc_fence_after();
          const uint32_t q = tmem + TM_Q + seg % Q_BUFS * (DIM / 2);
          const int count = g.n;
#pragma unroll 1
          for (int i = 0; i < count + LOOK && ok; ++i) {
            if (i < count) {
              const uint32_t n = tile + i, buf = n % S_BUFS, u = unit + k_unit(i), at = u % UNITS;
              if (OVER && n > 1) ok = WAIT_ONE(pv_done + 8 * buf, ((n >> 1) - 1) & 1, WAIT_PV);
              if (!OVER && n >= S_BUFS) ok = WAIT_ONE(s_free + 8 * buf, (n / S_BUFS - 1) & 1, WAIT_S_FREE);
              if (ok) ok = WAIT_ONE(kv_full + 8 * at, (u / UNITS) & 1, WAIT_KV_FULL);
              if (!ok) break;
              ptx::tc_fence_after();
              const uint32_t kd = kdesc + at * (UNIT >> 4);
#pragma unroll
              for (int j = 0; j < BLOCKS; ++j) umma_ts4<2>(tmem + TM_S + buf * TILE, q + 32 * j, kd + j * (TILE * 128 >> 4), idesc_s, j ? 1u : 0u);
              ptx::umma_commit(kv_empty + 8 * at);
              ptx::umma_commit(s_full + 8 * buf);
            }
            if (i >= LOOK) {
              const uint32_t n = tile + i - LOOK, buf = n & 1, u = unit + v_unit(i - LOOK, count), at = u % UNITS;
              if (i == LOOK && seg) ok = WAIT_ONE(o_free, (seg - 1) & 1, WAIT_O_FREE);
              if (ok) ok = WAIT_ONE(kv_full + 8 * at, (u / UNITS) & 1, WAIT_KV_FULL);
              if (ok) ok = WAIT_ONE(p_full + 8 * buf, (n >> 1) & 1, WAIT_P);
              if (!ok) break;
              ptx::tc_fence_after();
              umma_ts4<(16 * 128 >> 4)>(tmem + TM_O, tmem + TM_P + buf * P_STEP, vdesc + at * (UNIT >> 4), idesc_o, i > LOOK ? 1u : 0u);
              ptx::umma_commit(kv_empty + 8 * at);
              ptx::umma_commit(pv_done + 8 * buf);
            }
          }
        }
        __syncwarp();
        ok = __any_sync(0xffffffffu, leader && ok);
        unit += 2 * g.n;
        tile += g.n;
        ++seg;
      }
    } else if (warp == 2) {
      // ---- pages and masks, eight tiles at a time: a lane looks up a piece
      uint32_t tile = 0;
      const int pieces = TILE / p.piece;
      while (ok && NEXT) {
        const int p_tiles = g.batch || p.joined ? p.p_tiles : 0;
        const uint32_t length = g.batch ? 0 : lengths[g.b];
#pragma unroll 1
        for (int i0 = 0; i0 < g.n && ok; i0 += BATCH) {
          // this lane's piece of tile i0 + lane / pieces
          int page = -1, in = 0;
          int looked = 0;                     // 1: in the prefix's table, 2: in the sequence's
          {
            const int i = g.first + i0 + lane / pieces;
            const bool own = i >= p_tiles;
            const uint32_t first = (uint32_t)(own ? i - p_tiles : i) * TILE + lane % pieces * p.piece, end = own ? length : (uint32_t)p.s.prefix_tokens;
            if (lane < BATCH * pieces && i < g.first + g.n && first < end) {
              const uint32_t lp = first / (uint32_t)p.c.page_tokens;
              in = (int)(first - lp * (uint32_t)p.c.page_tokens);
              page = __ldcg((own ? p.s.table + (long long)g.b * p.s.table_stride : p.s.prefix_table) + lp);
              looked = own ? 2 : 1;
            }
          }
          uint32_t bits = 0;                  // sixteen keys of the prefix a lane, on their way together with the pages
          const bool masked = p.s.prefix_valid && g.first + i0 < p_tiles;
          if (masked) {
            const uint32_t key = (uint32_t)(g.first + i0) * TILE + 16 * lane, end = p.s.prefix_tokens;
#pragma unroll
            for (int k = 0; k < 16; ++k) bits |= (key + k >= end || __ldcg(p.s.prefix_valid + key + k) ? 1u : 0u) << k;
          }
          const bool bad = looked && (page < 0 || page >= p.c.pages);
          if (bad) { page = -1; cache::report(p.c.status, cache::BAD_PAGE, looked == 2 ? g.b : -1); }
          const unsigned gone = __ballot_sync(0xffffffffu, bad);
          const long long scale = (((long long)page * p.c.layers + p.s.layer) * p.c.kv_heads + g.h) * p.c.page_tokens + in;
          // lane k: keys of tile i0 + k that count
          uint32_t m0, m1;
          {
            const int i = g.first + i0 + lane;
            const bool own = i >= p_tiles;
            const uint32_t key = (uint32_t)(own ? i - p_tiles : i) * TILE, end = own ? length : (uint32_t)p.s.prefix_tokens;
            const uint32_t left = end > key ? end - key : 0u;
            m0 = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
            m1 = left >= 64 ? 0xffffffffu : left > 32 ? (1u << (left - 32)) - 1u : 0u;
          }
          if (masked) {
            const int from = 4 * (lane & 7);
            const uint32_t a = __shfl_sync(0xffffffffu, bits, from), b = __shfl_sync(0xffffffffu, bits, from + 1), c = __shfl_sync(0xffffffffu, bits, from + 2),
                           d = __shfl_sync(0xffffffffu, bits, from + 3);
            if (g.first + i0 + lane < p_tiles) { m0 &= a | b << 16; m1 &= c | d << 16; }
          }
#pragma unroll 1
          for (int k = 0; k < BATCH && i0 + k < g.n && ok; ++k) {
            const uint32_t n = tile + i0 + k, slot = n % INFO;
            if (n >= INFO) ok = WAIT(info_empty + 8 * slot, (n / INFO - 1) & 1, WAIT_INFO_EMPTY);
            if (!ok) break;
            Info& info = s_info[slot];
            const int j = lane - k * pieces;
            if (j >= 0 && j < pieces) { info.page[j] = page; info.in[j] = in; info.scale[j] = scale; }
            const int there = __popc(__ballot_sync(0xffffffffu, j >= 0 && j < pieces && page >= 0));
            if (lane == k) {
              unsigned long long lost = 0;
              if (gone)
#pragma unroll 1
                for (int q = 0; q < pieces; ++q)
                  if (gone >> (k * pieces + q) & 1) lost |= (p.piece == 64 ? ~0ull : (1ull << p.piece) - 1) << (q * p.piece);
              const uint32_t b0 = (uint32_t)lost, b1 = (uint32_t)(lost >> 32);
              info.there = there;
              info.mask[0] = m0; info.mask[1] = m1; info.bad[0] = b0 & m0; info.bad[1] = b1 & m1;
            }
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(info_full + 8 * slot);
            __syncwarp();
          }
        }
        tile += g.n;
      }
    } else if (warp == 3) {
      // What the combine kernel has to know of the items: the slots of their parts
      {
        const int a_items = p.joined ? 0 : p.a_tiles * p.c.kv_heads, items = a_items + p.s.batch * p.c.kv_heads * p.b_tiles;
        for (int item = lane * gridDim.x + blockIdx.x; item < items; item += gridDim.x * 32) {
          int at = 0, tiles = 0;                // first unit behind the item's overhead
          const int own = item - a_items;
          if (own < 0) {
            at = item * walk.a_cost;
            tiles = p.p_tiles;
          } else {
            const int hb = own / p.b_tiles, h = hb / p.s.batch, b = hb - h * p.s.batch, units = sums[b + 1] - sums[b];
            if (units) {
              const int cost = units / p.b_tiles;
              at = walk.a_units + h * walk.b_units + sums[b] + (own - hb * p.b_tiles) * cost;
              tiles = cost - p.overhead;
            }
          }
          int2 part = make_int2(0, 0);
          if (tiles) {
            const int first = walk.cta_of(at + p.overhead), n = walk.cta_of(at + p.overhead + tiles - 1) - first + 1;
            part = make_int2(first + (own < 0 ? item : own), own >= 0 && p.joined && n == 1 ? -1 : n);
          }
          p.parts[item] = part;
        }
      }
      // ---- a tile's scales: of the keys times the softmax's constant, of the values at places that count, and the logarithms of those
      if constexpr (CODES) {
        uint32_t tile = 0;
        while (ok && NEXT) {
#pragma unroll 1
          for (int i = 0; i < g.n && ok; ++i) {
            const uint32_t n = tile + i, slot = n % INFO;
            ok = WAIT(info_full + 8 * slot, (n / INFO) & 1, WAIT_INFO);
            if (ok) ok = WAIT(scale_full + 8 * slot, (n / INFO) & 1, WAIT_SCALES);
            if (!ok) break;
            float* ks = const_cast<float*>(s_scales) + slot * 3 * TILE;
            const Info& info = s_info[slot];
            unsigned none[2];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              float *k = ks + 32 * half + lane, *v = k + TILE;
              const bool counts = (info.mask[half] & ~info.bad[half]) >> lane & 1;
              const float s = counts ? *v : 0.f;
              // a scale that does not count is whatever memory holds, and 0 x NaN is NaN: zero in its place, also where it counts and is not a number
              const bool finite = fabsf(s) < INFINITY;
              none[half] = __ballot_sync(0xffffffffu, !finite);
              if (!counts || !finite) *v = 0.f;
              *k *= p.c_log2;               // (a score then is an exponent to the base 2 by one product)
              v[TILE] = fmaxf(__log2f(finite ? fabsf(s) : 0.f), LOG_LEAST) + LOG_SHIFT;
            }
            ptx::fence_proxy_async_shared();  // a later copy writes where these zeros went
            __syncwarp();                     // (and lane 0 reports for all)
            if (lane == 0) {
              s_bad[slot][0] = info.bad[0] | none[0];
              s_bad[slot][1] = info.bad[1] | none[1];
              ptx::mbar_arrive(vlog_full + 8 * slot);
              ptx::mbar_arrive(info_empty + 8 * slot);
            }
            __syncwarp();
          }
          tile += g.n;
        }
      }
    }
  } else if (warp < 12) {
    // ---- softmax: thread = query row, group = every second tile.  A wait that gave up lets the rest run through, with NaN as the result
    const int group = (warp - 4) >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t lanes = tmem + ((uint32_t)(quad * 32) << 16);
    uint32_t unit = 0, tile = 0, seg = 0, turn = 0;
    auto load_q = [&](const Segment& s, uint32_t seg) {
      load_queries<DIM>(p, s, row, lanes + TM_Q + seg % Q_BUFS * (DIM / 2));
      if (lane == 0) ptx::mbar_arrive(q_full + 8 * (seg % Q_BUFS));
      __syncwarp();
    };
    const int sw = warp - 4;
    ptx::grid_dep_wait();
    int at = next_segment(p, walk, walk.begin(blockIdx.x), &s_seg[warp]);
    bool more = at >= 0;
    if (more && group == 1) load_q(s_seg[warp], 0);        // (the first tile is the other group's)
    while (more) {
      const int par = seg & 1;
      const Segment& d = par ? s_ahead[sw] : s_seg[warp];
      Segment& ahead = par ? s_seg[warp] : s_ahead[sw];      // the one after it
      const int count = d.n;
      int own;                              // of the segment's first tile: its place among the tiles of own tokens
      int sees;                             // own tokens that the row sees
      int all_see;                          // and those that all rows of the item do
      bool mine, idle;
      {
        int b = 0, t = 0, head = 0;
        mine = row_of(p, d, row, b, t, head);
        idle = !__any_sync(0xffffffffu, mine);
        own = d.first - (d.batch || p.joined ? p.p_tiles : 0);
        const int length = d.batch ? 0 : lengths[d.b];
        sees = p.s.causal ? length - p.s.tokens + t + 1 : length;
        all_see = p.s.causal && p.s.tokens > 1 ? length - p.s.tokens + 1 : 0x7fffffff;
      }
      float m = -INFINITY, l = 0.f;         // reference (of exponents to the base 2) and sum
      at = next_segment(p, walk, at, &ahead);
      more = at >= 0;
      if (Q_BUFS == 2 && more && ((tile & 1) ^ group)) load_q(ahead, seg + 1);
#pragma unroll 1
      for (int i = (tile & 1) ^ group; i < count; i += 2) {
        const uint32_t n = tile + i, buf = group, sbuf = n % S_BUFS, slot = n % INFO;
        // (warp 3 has waited for the tile's masks and scales before it reports)
        ok = ok && WAIT((CODES ? vlog_full : info_full) + 8 * slot, (n / INFO) & 1, CODES ? WAIT_SCALES : WAIT_INFO);
        const uint32_t mask0 = s_info[slot].mask[0], mask1 = s_info[slot].mask[1];
        const uint32_t bad0 = CODES ? s_bad[slot][0] : s_info[slot].bad[0], bad1 = CODES ? s_bad[slot][1] : s_info[slot].bad[1];
        uint32_t k0 = mask0, k1 = mask1;    // keys that count for this row
        if (own + i >= 0) {
          const int left = sees - (own + i) * TILE;
          if (left < TILE) {
            k0 &= left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
            k1 &= left > 32 ? (1u << (left - 32)) - 1u : 0u;
          }
        }
        const bool poison = (k0 & bad0) | (k1 & bad1);     // the row sees a key that does not exist, or a value that is not a number
        k0 &= ~bad0;
        k1 &= ~bad1;
        const bool special = __any_sync(0xffffffffu, (k0 & k1) != 0xffffffffu);
        ok = ok && WAIT(s_full + 8 * sbuf, (n / S_BUFS) & 1, WAIT_S);
        ptx::tc_fence_after();
        const float4* ks = reinterpret_cast<const float4*>(s_scales + slot * 3 * TILE);
        // Of 8 bits: what turns a score into an exponent, the first time and, where keys that do not count are marked, the second
        const float4* scale = special ? reinterpret_cast<const float4*>(s_ones) : ks;
        const uint32_t s_at = lanes + TM_S + sbuf * TILE, p_at = lanes + TM_P + buf * P_STEP;
        // A tile is read twice, CHUNK scores at a time: for the row's maximum, then for the probabilities.  (What the warps of a CTA execute per tile has to fit the
        // instruction cache.  With all 64 scores in registers 26% of the fetches missed it and drafts, 32 x 8 over 8192 in e4m3, took 245 us; read
        // twice in 32s 14%, 142; in 16s and with the converters' loop rolled 121, now 122 with a reference that goes by the keys that a row sees)
        auto load_chunk = [](uint32_t from, float (&x)[CHUNK]) {
          if constexpr (CHUNK == 32) ptx::tmem_ld_32x32(from, reinterpret_cast<uint32_t(&)[32]>(x));
          else ptx::tmem_ld_32x16(from, reinterpret_cast<uint32_t(&)[16]>(x));
          ptx::tmem_wait_ld();
        };
        float high = -INFINITY;
        if (!idle) {
#pragma unroll 1
          for (int h = 0; h < TILE; h += CHUNK) {
            float x[CHUNK];
            load_chunk(s_at + h, x);
            if (special) {                  // keys that do not count: -infinity, there (of 8 bits exponents) for the second time too
              if (CODES) {
#pragma unroll
                for (int j = 0; j < CHUNK; j += 4) {
                  const float4 f = ks[(h + j) / 4];
                  const float2 y = mul2(make_float2(x[j], x[j + 1]), make_float2(f.x, f.y)), z = mul2(make_float2(x[j + 2], x[j + 3]), make_float2(f.z, f.w));
                  x[j] = y.x; x[j + 1] = y.y; x[j + 2] = z.x; x[j + 3] = z.y;
                }
              }
              const uint32_t k = (h < 32 ? k0 : k1) >> (h & 31);
#pragma unroll
              for (int j = 0; j < CHUNK; ++j) x[j] = k >> j & 1 ? x[j] : -INFINITY;
#pragma unroll
              for (int j = 0; j < CHUNK; j += 8) ptx::tmem_st_32x8(s_at + h + j, reinterpret_cast<uint32_t(&)[8]>(x[j]));
            }
            if (CODES) {                    // exponents of the products of probability and value's scale
#pragma unroll
              for (int j = 0; j < CHUNK; j += 4) {
                const float4 f = scale[(h + j) / 4], v = ks[(2 * TILE + h + j) / 4];
                const float2 y = ptx::fma2(make_float2(x[j], x[j + 1]), make_float2(f.x, f.y), make_float2(v.x, v.y)),
                             z = ptx::fma2(make_float2(x[j + 2], x[j + 3]), make_float2(f.z, f.w), make_float2(v.z, v.w));
                x[j] = y.x; x[j + 1] = y.y; x[j + 2] = z.x; x[j + 3] = z.y;
              }
            }
            float a = high, b = -INFINITY;
#pragma unroll
            for (int j = 0; j < CHUNK; j += 4) {
              a = fmaxf(fmaxf(a, x[j]), x[j + 1]);
              b = fmaxf(fmaxf(b, x[j + 2]), x[j + 3]);
            }
            high = fmaxf(a, b);
          }
          if (special) ptx::tmem_wait_st();
          if (!CODES) high *= p.c_log2;
          bool write = true;
          if (i == 0) {
            m = high;
          } else {
            ptx::named_bar_sync(TOKEN + 4 * group + quad, 64);
            const float r = s_ref[par][row];
            if (r != m) { l *= ptx::ex2_approx(m - r); m = r; }
            const bool move = high > m + RESCALE;
            write = __any_sync(0xffffffffu, move);
            if (write) {
              const float f = move ? ptx::ex2_approx(m - high) : 1.f;
              if (move) m = high;
              l *= f;
              ok = ok && WAIT(pv_done + 8 * (buf ^ 1), ((n - 1) >> 1) & 1, WAIT_PV);
              ptx::tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < DIM; c += 16) {
                uint32_t o[16];
                ptx::tmem_ld_32x16(lanes + TM_O + c, o);
                ptx::tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                ptx::tmem_st_32x8(lanes + TM_O + c, reinterpret_cast<uint32_t(&)[8]>(o[0]));
                ptx::tmem_st_32x8(lanes + TM_O + c + 8, reinterpret_cast<uint32_t(&)[8]>(o[8]));
              }
              ptx::tmem_wait_st();
            }
          }
          if (write) s_ref[par][row] = m;
          __syncwarp();
          if (i + 1 < count) ptx::bar_arrive(TOKEN + 4 * (group ^ 1) + quad, 64);
        }
        // The buffer of P is free once the product before the last has read it.  (A warp without rows waits as well: it must not report its part of
        // this tile before the others have reported theirs of that one)
        if (!OVER && n > 1) {
          ok = ok && WAIT(pv_done + 8 * buf, ((n >> 1) - 1) & 1, WAIT_PV);
          ptx::tc_fence_after();
        }
        if (!idle) {
          const float ref = m == -INFINITY ? 0.f : m;
          const float2 c2 = make_float2(p.c_log2, p.c_log2), r2 = make_float2(-ref, -ref);
          float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll 1
          for (int h = 0; h < TILE; h += CHUNK) {
            float x[CHUNK];
            load_chunk(s_at + h, x);
            uint32_t pk[CHUNK / 2];
#pragma unroll
            for (int j = 0; j < CHUNK; j += 4) {
              float2 e = make_float2(x[j], x[j + 1]), f = make_float2(x[j + 2], x[j + 3]);
              float2 ce = c2, cf = c2;
              if (CODES) {
                const float4 s = scale[(h + j) / 4];
                ce = make_float2(s.x, s.y); cf = make_float2(s.z, s.w);
              }
              e = ptx::fma2(e, ce, r2);
              f = ptx::fma2(f, cf, r2);
              e.x = ptx::ex2_approx(e.x); e.y = ptx::ex2_approx(e.y); f.x = ptx::ex2_approx(f.x); f.y = ptx::ex2_approx(f.y);
              sum[0] = add2(sum[0], e);
              sum[1] = add2(sum[1], f);
              if (CODES) {
                const float4 s = ks[(TILE + h + j) / 4];
                e = mul2(e, make_float2(s.x, s.y));
                f = mul2(f, make_float2(s.z, s.w));
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pk[j / 2]) : "f"(e.y), "f"(e.x));
                asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(pk[j / 2 + 1]) : "f"(f.y), "f"(f.x));
              } else {
                pk[j / 2] = cache::pack2(e.x, e.y);
                pk[j / 2 + 1] = cache::pack2(f.x, f.y);
              }
            }
#pragma unroll
            for (int j = 0; j < CHUNK / 2; j += 8) ptx::tmem_st_32x8(p_at + h / 2 + j, reinterpret_cast<uint32_t(&)[8]>(pk[j]));
          }
          const float2 both = add2(sum[0], sum[1]);
          l += both.x + both.y;
          if (poison) l = __uint_as_float(0x7fffffffu);
          ptx::tmem_wait_st();
        }
        // Values at places that do not count are whatever memory holds, and 0 x NaN is NaN: zeros in their place.  Where only some of the tile's rows see a token
        // (`ragged`) the same for an infinity or a NaN among its values, and the rows that do see it get NaN
        const bool ragged = !CODES && own + i >= 0 && (own + i + 1) * TILE > all_see;
        if (!CODES && (ragged || (mask0 & mask1 & ~(bad0 | bad1)) != 0xffffffffu)) {
          const uint32_t u = unit + v_unit(i, count), at = u % UNITS;
          ok = ok && WAIT(kv_full + 8 * at, (u / UNITS) & 1, WAIT_KV_FULL);
          const uint32_t z0 = ~mask0 | bad0, z1 = ~mask1 | bad1, line = ring + at * UNIT;
          // a key's row by D / 8 lanes, sixteen keys a warp
          const uint32_t mine_clear = (quad & 2 ? z1 : z0) >> (16 * (quad & 1));
#pragma unroll 4
          for (int c = lane / (DIM / 8); c < 16; c += 32 / (DIM / 8))
            if (mine_clear >> c & 1)
              ptx::st_shared_v4(line + (lane % (DIM / 8) >> 3) * (TILE * 128) + (16 * quad + c) * 128 + (lane & 7) * 16, 0u, 0u, 0u, 0u);
          if (ragged) {
            // The next ragged tile's, whatever tiles and items lie between: the last one that used it is an earlier tile of the group, whose product
            // needed all four warps to be through with it and has been waited for above
            if (row < 2) s_lost[group][turn ^ 1][row] = 0u;
#pragma unroll 1
            for (int c = row; c < TILE * DIM / 8; c += 128) {
              const int key = c & 63, chunk = c >> 6;
              const uint32_t to = line + (chunk >> 3) * (TILE * 128) + key * 128 + (chunk & 7) * 16;
              if ((key < 32 ? z0 : z1) >> (key & 31) & 1) continue;
              const uint4 x = ptx::ld_shared_v4(to);
              const uint32_t w[4] = {x.x, x.y, x.z, x.w};
              bool found = false;
#pragma unroll
              for (int k = 0; k < 4; ++k) found |= (w[k] & 0x7f80u) == 0x7f80u || (w[k] & 0x7f800000u) == 0x7f800000u;
              if (found) {
                atomicOr(&s_lost[group][turn][key >> 5], 1u << (key & 31));
                ptx::st_shared_v4(to, 0u, 0u, 0u, 0u);
              }
            }
            __syncwarp();
          }
          ptx::fence_proxy_async_shared();
          if (ragged) {
            ptx::named_bar_sync(LOST + group, 128);
            if ((k0 & s_lost[group][turn][0]) | (k1 & s_lost[group][turn][1])) l = __uint_as_float(0x7fffffffu);
            turn ^= 1;
          }
        }
        __syncwarp();
        ptx::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (!OVER) ptx::mbar_arrive(s_free + 8 * sbuf);
          ptx::mbar_arrive(p_full + 8 * buf);
          ptx::mbar_arrive(info_empty + 8 * slot);
        }
        __syncwarp();
      }
      const uint32_t last = tile + count - 1;
      unit += 2 * count;
      tile += count;
      // ---- the next segment's queries, by the group that does not have the last tile, once the last scores are there
      if (Q_BUFS == 1 && more && (last & 1) != (uint32_t)group) {
        ok = ok && WAIT(s_full + 8 * (last % S_BUFS), (last / S_BUFS) & 1, WAIT_S);
        ptx::tc_fence_after();
        load_q(ahead, seg + 1);
      }
      // ---- the segment's sums, half of the columns each
      if (!idle) {
        s_ml[par][group][row] = make_float2(m, l);
        ptx::named_bar_sync(END + quad, 64);
        const float2 other = s_ml[par][group ^ 1][row];
        const float r = s_ref[par][row];
        l = (m == r ? l : l * ptx::ex2_approx(m - r)) + (other.x == r ? other.y : other.y * ptx::ex2_approx(other.x - r));
        m = r;
      }
      ok = ok && WAIT(pv_done + 8 * (last & 1), (last >> 1) & 1, WAIT_PV);
      ptx::tc_fence_after();
      if (!ok) l = __uint_as_float(0x7fffffffu);
      if (!idle) {
        int b = 0, t = 0, head = 0;
        row_of(p, d, row, b, t, head);
        const bool direct = !d.batch && p.joined && d.n == d.tiles;
        const float il = !direct ? 1.f : l == 0.f ? 0.f : 1.0f / l;        // (no key: zeros)
        __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.s.out) + b * p.s.out_batch_stride + t * p.s.out_token_stride + head * p.s.out_head_stride;
        const int rows = d.batch ? ROWS : p.b_slot;
        float* part = (d.batch ? p.a_parts : p.b_parts) + (long long)(blockIdx.x + d.item) * rows * (DIM + 2);
#pragma unroll 1
        for (int c = group * (DIM / 2); c < (group + 1) * (DIM / 2); c += 32) {
          uint32_t o[32];
          ptx::tmem_ld_32x32(lanes + TM_O + c, o);
          ptx::tmem_wait_ld();
          if (mine && direct) {
#pragma unroll
            for (int j = 0; j < 32; j += 8)
              *reinterpret_cast<uint4*>(out + c + j) = make_uint4(
                  cache::pack2(__uint_as_float(o[j]) * il, __uint_as_float(o[j + 1]) * il), cache::pack2(__uint_as_float(o[j + 2]) * il, __uint_as_float(o[j + 3]) * il),
                  cache::pack2(__uint_as_float(o[j + 4]) * il, __uint_as_float(o[j + 5]) * il), cache::pack2(__uint_as_float(o[j + 6]) * il, __uint_as_float(o[j + 7]) * il));
          } else if (mine) {
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              __stcg(reinterpret_cast<uint4*>(part) + ((c + j) / 4) * rows + row, make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]));
          }
          __syncwarp();
        }
        if (mine && group == 0) {
          if (!direct) __stcg(reinterpret_cast<float2*>(part + DIM * rows) + row, make_float2(m, l));
          else if (p.s.lse) p.s.lse[((long long)b * p.s.tokens + t) * p.s.q_heads + head] = l == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m) + log2f(l)) * 0.6931471805599453f;
        }
      }
      ++seg;
      ptx::tc_fence_before();
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(o_free);
      __syncwarp();
    }
  } else if constexpr (CODES) {
    // ---- codes to 16 bits, the two groups in turn: 16 codes per thread and turn, to two 16-byte chunks of the swizzled unit.  Eight
    // neighbouring lanes take 64 bytes of an even row and the other 64 of the odd one, so that neither the loads nor the stores share banks
    const int group = (warp - 12) >> 2, w = warp & 3, odd = lane >> 2 & 1, chunk = lane & 3, high = lane >> 3;
    const int blk = BLOCKS == 4 ? high ^ odd : BLOCKS == 2 ? (high & 1) ^ odd : 0;
    constexpr int ROWS_AT_ONCE = 8 / BLOCKS;         // rows of a warp's turn
    const int first = odd + (BLOCKS == 4 ? 0 : BLOCKS == 2 ? (high >> 1) * 2 : high * 2);
    uint32_t unit = 0;
    while (ok && NEXT) {
#pragma unroll 1
      for (int u = (unit & 1) ^ group; u < 2 * g.n && ok; u += 2) {
        bool is_v;
        what(u, g.n, is_v);
        const uint32_t n = unit + u, from = n % RAW, to = n % UNITS;
        ok = WAIT(raw_full + 8 * from, (n / RAW) & 1, WAIT_RAW_FULL);
        if (ok && n >= UNITS) ok = WAIT(kv_empty + 8 * to, (n / UNITS - 1) & 1, WAIT_KV_EMPTY);
        if (!ok) break;
        constexpr int TURNS = TILE / ROWS_AT_ONCE / 4;
        auto turns = [&](auto value) {
#pragma unroll 1                        // (unrolled twice, drafts of 121 us took 142: the instruction cache)
          for (int j = 0; j < TURNS; ++j) {
            const int r = (j * 4 + w) * ROWS_AT_ONCE + first;
            const uint4 x = ptx::ld_shared_v4(raw + from * RAW_UNIT + r * DIM + blk * 64 + chunk * 16);
            const uint2 a = value(x.x), c = value(x.y), d = value(x.z), e = value(x.w);
            const uint32_t line = ring + to * UNIT + blk * (TILE * 128) + r * 128;
            ptx::st_shared_v4(line + (((2 * chunk) ^ (r & 7)) << 4), a.x, a.y, c.x, c.y);
            ptx::st_shared_v4(line + (((2 * chunk + 1) ^ (r & 7)) << 4), d.x, d.y, e.x, e.y);
          }
        };
        if (is_v) turns([](uint32_t c) { return cache::quad_half<FORMAT>(c); });
        else turns([](uint32_t c) { return cache::quad<FORMAT>(c); });
        ptx::fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) { ptx::mbar_arrive(kv_full + 8 * to); ptx::mbar_arrive(raw_empty + 8 * from); }
        __syncwarp();
      }
      unit += 2 * g.n;
    }
  }
#undef WAIT
#undef WAIT_ONE
#undef NEXT
  ptx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc(tmem, TM_COLS);
  }
}

// The unfinished items of a launch put together.  A warp has eight query rows x 16 dims (a line of every 16 bytes of a part), of which `split` warps of a
// block take every split-th part each, eight at a time: what bounds it is how many loads are on their way (with four at a time and no more than eight warps a row 13
// queries over 30001 tokens, 148 parts, took 36.4 us, now 32).
constexpr int COMBINE_THREADS = 512, AT_ONCE = 8;
template <int DIM>
__global__ void __launch_bounds__(COMBINE_THREADS) combine_kernel(const __grid_constant__ Args p, int split) {
  constexpr int WARPS = COMBINE_THREADS / 32;
  __shared__ float2 s_ml[WARPS][8];
  __shared__ float4 s_o[WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, share = warp % split;
  const int flat = p.s.batch * p.s.tokens * p.group, groups = (flat + 7) / 8;
  const int work = blockIdx.x * (WARPS / split) + warp / split, hg = work / (DIM / 16);
  const int column = (work & (DIM / 16 - 1)) * 4 + (lane & 3);           // of four dims
  const int h = hg / groups, f = (hg - h * groups) * 8 + row;
  const bool in = h < p.c.kv_heads && f < flat;
  const int bt = f / p.group, gi = f - bt * p.group, b = bt / p.s.tokens, t = bt - b * p.s.tokens;
  const int fs = f - b * p.s.tokens * p.group, r = fs / p.b_rows, b_row = fs - r * p.b_rows, a_items = p.joined ? 0 : p.a_tiles * p.c.kv_heads;
  ptx::grid_dep_wait();
  int2 a = make_int2(0, 0), o_ = make_int2(0, 0);
  if (in) {
    if (!p.joined) a = __ldcg(p.parts + h * p.a_tiles + f / ROWS);
    o_ = __ldcg(p.parts + a_items + (h * p.s.batch + b) * p.b_tiles + r);
  }
  const bool done = o_.y < 0;               // one CTA had it all
  const int n = done ? 0 : a.y + o_.y;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int k0 = share; k0 < n; k0 += AT_ONCE * split) {
    float2 ml[AT_ONCE];
    float4 v[AT_ONCE];
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const int at = k0 + k * split;
      const bool own = at >= a.y;
      const int rows = own ? p.b_slot : ROWS;
      const float* part = own ? p.b_parts + (long long)(o_.x + at - a.y) * rows * (DIM + 2) : p.a_parts + (long long)(a.x + at) * rows * (DIM + 2);
      const int pr = own ? b_row : f % ROWS;
      ml[k] = at < n ? __ldcg(reinterpret_cast<const float2*>(part + DIM * rows) + pr) : make_float2(-INFINITY, 0.f);
      v[k] = at < n ? __ldcg(reinterpret_cast<const float4*>(part) + column * rows + pr) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) top = fmaxf(top, ml[k].x);
    const float w = m == top ? 1.f : ptx::ex2_approx(m - top);
    l *= w; o.x *= w; o.y *= w; o.z *= w; o.w *= w;
    m = top;
#pragma unroll
    for (int k = 0; k < AT_ONCE; ++k) {
      const float u = ml[k].x == top ? 1.f : ptx::ex2_approx(ml[k].x - top);
      l += ml[k].y * u;
      o.x += v[k].x * u; o.y += v[k].y * u; o.z += v[k].z * u; o.w += v[k].w * u;
    }
  }
  if (split > 1) {
    if ((lane & 3) == 0) s_ml[warp][row] = make_float2(m, l);
    s_o[warp][lane] = o;
    __syncthreads();
    if (share) return;
    float top = m;
#pragma unroll 1
    for (int k = 1; k < split; ++k) top = fmaxf(top, s_ml[warp + k][row].x);
    const float w = m == top ? 1.f : ptx::ex2_approx(m - top);
    l *= w; o.x *= w; o.y *= w; o.z *= w; o.w *= w;
    m = top;
#pragma unroll 1
    for (int k = 1; k < split; ++k) {
      const float2 ml = s_ml[warp + k][row];
      const float4 v = s_o[warp + k][lane];
      const float u = ml.x == top ? 1.f : ptx::ex2_approx(ml.x - top);
      l += ml.y * u;
      o.x += v.x * u; o.y += v.y * u; o.z += v.z * u; o.w += v.w * u;
    }
  }
  if (!in || done) return;
  const float il = l == 0.f ? 0.f : 1.0f / l;
  const int head = h * p.group + gi;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.s.out) + b * p.s.out_batch_stride + t * p.s.out_token_stride + head * p.s.out_head_stride;
  *reinterpret_cast<uint2*>(out + column * 4) = make_uint2(cache::pack2(o.x * il, o.y * il), cache::pack2(o.z * il, o.w * il));
  if (column == 0 && p.s.lse) p.s.lse[((long long)b * p.s.tokens + t) * p.s.q_heads + head] = l == 0.f ? -INFINITY : ((m == -INFINITY ? 0.f : m) + log2f(l)) * 0.6931471805599453f;
}

}  // namespace shared
