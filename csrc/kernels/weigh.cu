// The attention weight that the rows of prefill chunks give to every key of the paged INT8 cache:
//   sums[slot][KV head][j] += sum over the chunk's rows i that see j, and the query heads h of the KV head,
//                             of exp(q_ih . k_j / sqrt D - lse_ih).
// A row's lse is known only behind all of its keys, and the sums run over rows, so the scores are
// made twice, by two kernels on tcgen05 tensor cores, neither of which writes any:
//   stats_kernel  S = Q K^T, a row per TMEM lane: maxima and sums of weights, one lse for each row;
//   sums_kernel   S^T = K Q^T, a key per lane: a thread adds the weights of its key, no lane to lane sums.
// Behind the first join_kernel makes a row's lse of its parts, once for all who use it; behind the
// second add_kernel adds the parts of a key's sum, in their order, to the sums so far.
//
// A query tile is 128 rows: P = 128 / rep positions of one request times the `rep` query heads that
// share a KV head.  K is the exact FP16 integers that the cache holds; products of each group of 64
// channels have an accumulator of their own and meet, times the key's group scales, in FP32, so
// that a score is as exact as FP32 products give it.
//
// Work is counted in units, 128 rows by 128 keys (64 in stats_kernel with heads of 256 channels), in the
// order (chunk, KV head, tile, step): row tiles walk their keys, key tiles the row tiles that see them.
// Every CTA takes as many units, wherever a tile begins or ends, and leaves a part of each tile that it
// had at place (tile + CTA) of a list, which is nobody else's; the tile's first and last CTA are noted.
//
// A CTA is persistent: a warp for copies (queries, and raw INT8 keys), one for products, one for scales,
// four that make FP16 integers of keys, and sixteen for weights, in two groups that have a product each
// in turn, half of its columns to a warp.  What bounds it is neither memory nor the tensor cores but the
// weights: a unit of 128 x 128 is 16384 exponentials, 1024 cycles of the SM's unit for them, and 512 of
// products; it takes about 1560 cycles in sums_kernel (that unit 72 % busy, half of the issue slots used)
// and 1850 in stats_kernel (60 %), which has other scales for each column and the reference beside.
// 32 / 8 heads of 128, 4096 rows: 131 and 111 us, join and add 5 and 7; six requests of 37 to 64 rows behind
// 11459 to 20000 keys: 98 and 126; two of 777 and 537 rows behind 3000 and 2073 keys, 16 / 2 heads of 256
// (twice the products' columns to a weight): 66 and 53.
//
// On the way, both kernels at 4096 rows: eight warps for weights 181 and 163; sixteen 169 and 156;
// products of 128 rows in sums 160 and 151; lse joined once (by every CTA for each unit it cost 35 us of
// sums) and scores kept in registers while they are weighed 176 and 140; two groups on alternate products
// 160 and 119; 32 columns in registers 136 and 113; one warp for scales 134 and 113.  Slower: polynomials
// for 2 or 4 of 8 pairs of exponentials (sums 122 and 139 for 116), TMEM read 16 or 32 columns at a time
// (116 to 130), eight warps for integers (147), a maximum of every few columns in stats (148 for 136), more
// registers for the weights' warps at the others' cost (spills).
#include <cuda.h>

#include <type_traits>

#include "api.h"
#include "common.cuh"
#include "tma.h"

namespace orinfer {
namespace kw {

constexpr int TILE = 128;                        // rows of a tile: positions x query heads; keys of a tile
constexpr int MAX_CHUNKS = 512;
// Softmax or sums: two groups, a product each in turn, so that one computes while the other waits and reads.
// Whoever waits on a barrier does so for each of its phases: one that came for every other one could not
// tell them apart.
constexpr int EP_WARPS = 16, EP_GROUP = 8, GROUPS = 2;
constexpr int DQ_WARPS = 4;                      // INT8 to FP16
constexpr int AUX_WARPS = 1;                     // scales
constexpr int AUX_WARP = EP_WARPS + DQ_WARPS, MMA_WARP = AUX_WARP + AUX_WARPS;
constexpr int TMA_WARP = MMA_WARP + 1, THREADS = (TMA_WARP + 1) * 32;
constexpr int CTAS = 148;
constexpr int PARTS = 4;                         // of a tile: two groups, two halves of the columns
constexpr int COLS = 32;                         // columns that a thread has in registers
constexpr int NS = 4;                            // places of scales, or of rows' lse
constexpr float FAR = 1.1529215046068470e18f;    // 2^60: weights under a reference that has to move

struct Chunk {            // of one request
  int row_start;          // first packed row
  int q_len;              // rows in the chunk
  int pos0;               // absolute position of the first row
  int slot;               // row of the page table
};

// First and last CTA of a tile.  (Where a kernel gave up waiting they are anything, and its status is set.)
__device__ __forceinline__ int2 span_of(const int* span, int index) {
  const int lo = span[2 * index], hi = span[2 * index + 1];
  return make_int2(max(0, min(lo, CTAS - 1)), max(0, min(hi, CTAS - 1)));
}

// What bounds a chunk, and how rows are packed.
struct Geometry {
  const Chunk* chunks;
  const int* page_table;
  int n_chunks, total_rows, slots, max_pages, num_pages;
  int longest, limit;                            // rows of a chunk, keys of a request at most
  int qh, kvh, rep, per;                         // per: positions of a row tile
  __device__ Chunk at(int c) const {             // without rows where it is out of bounds
    Chunk ch = chunks[c];
    if (ch.q_len <= 0 || ch.q_len > longest || ch.q_len > limit || ch.row_start < 0 ||
        ch.row_start > total_rows - ch.q_len || ch.pos0 < 0 || ch.pos0 > limit - ch.q_len ||
        ch.slot < 0 || ch.slot >= slots)
      ch.q_len = 0;
    return ch;
  }
};

// Tiles of a chunk and steps of a tile.  KT keys to a step of NT neighbouring row tiles; 0: key tiles, a
// step is a row tile, from the first one that sees the key tile on.
template <int KT, int NT = 1>
struct Order {
  __device__ static int tiles(const Geometry& g, const Chunk& ch) {
    if (ch.q_len <= 0) return 0;
    return KT ? (ch.q_len + NT * g.per - 1) / (NT * g.per) : (ch.pos0 + ch.q_len + TILE - 1) / TILE;
  }
  __device__ static int first(const Geometry& g, const Chunk& ch, int tile) {
    return KT ? 0 : max(tile * TILE - ch.pos0, 0) / g.per;
  }
  __device__ static int steps(const Geometry& g, const Chunk& ch, int tile) {
    if (KT) return (ch.pos0 + min((tile + 1) * NT * g.per, ch.q_len) + KT - 1) / (KT ? KT : 1);
    return (ch.q_len + g.per - 1) / g.per - first(g, ch, tile);
  }
};

// Per chunk: units and tiles of a KV head.  Filled by the CTA together.
struct Plan {
  int units[MAX_CHUNKS], tiles[MAX_CHUNKS];
};
template <int KT, int NT = 1>
__device__ __forceinline__ void make_plan(Plan& plan, const Geometry& g, int* status) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int c = warp; c < g.n_chunks; c += THREADS / 32) {
    const Chunk ch = g.at(c);
    if (ch.q_len == 0 && blockIdx.x == 0 && lane == 0 && g.chunks[c].q_len != 0)
      report_status(status, STATUS_BAD_INDEX, 0x70);
    const int tiles = Order<KT, NT>::tiles(g, ch);
    int sum = 0;
    for (int t = lane; t < tiles; t += 32) sum += Order<KT, NT>::steps(g, ch, t);
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == 0) {
      plan.units[c] = sum;
      plan.tiles[c] = tiles;
    }
  }
}

// A CTA's walk over its units, tile by tile.  All warps have one, a warp together.
template <int KT, int NT = 1>
struct Walk {
  const Geometry& g;
  const Plan& plan;
  Chunk ch;
  int c, h, tile, step, steps, left, first;      // first: the tile's first row tile (of key tiles)
  int index;                                     // of the tile, among all chunks' and heads'
  __device__ Walk(const Geometry& geo, const Plan& p) : g(geo), plan(p) {
    const int lane = threadIdx.x & 31;
    int total = 0;
    for (int i = lane; i < g.n_chunks; i += 32) total += plan.units[i];
    total = __reduce_add_sync(0xffffffffu, total) * g.kvh;
    const int share = (total + gridDim.x - 1) / gridDim.x;
    int at = blockIdx.x * share;
    left = max(min(total - at, share), 0);
    if (left == 0) return;
    index = 0;
    for (c = 0;; ++c) {
      const int here = plan.units[c] * g.kvh;
      if (at < here) break;
      at -= here;
      index += plan.tiles[c] * g.kvh;
    }
    h = at / plan.units[c];
    at -= h * plan.units[c];
    index += h * plan.tiles[c];
    ch = g.at(c);
    for (int t0 = 0;; t0 += 32) {                // the tile in which it lies, 32 at a time
      const int n = t0 + lane < plan.tiles[c] ? Order<KT, NT>::steps(g, ch, t0 + lane) : 0;
      int before = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      const unsigned later = __ballot_sync(0xffffffffu, before > at);
      if (later != 0) {
        const int who = __ffs(later) - 1;
        tile = t0 + who;
        steps = __shfl_sync(0xffffffffu, n, who);
        step = at - __shfl_sync(0xffffffffu, before, who) + steps;
        break;
      }
      at -= __shfl_sync(0xffffffffu, before, 31);
    }
    index += tile;
    first = Order<KT, NT>::first(g, ch, tile);
  }
  __device__ int here() const { return min(steps - step, left); }        // units of this tile
  __device__ void next_tile() {
    left -= here();
    if (left == 0) return;
    step = 0;
    ++index;
    if (++tile == plan.tiles[c]) {
      tile = 0;
      if (++h == g.kvh) {
        h = 0;
        do ++c; while (plan.units[c] == 0);
        ch = g.at(c);
      }
    }
    steps = Order<KT, NT>::steps(g, ch, tile);
    first = Order<KT, NT>::first(g, ch, tile);
  }
};
// The same unit by unit, for roles that go ahead of the others.
template <int KT, int NT = 1>
struct Units {
  Walk<KT, NT> w;
  int i;                                         // of the tile's
  __device__ Units(const Geometry& g, const Plan& p) : w(g, p), i(0) {}
  __device__ bool more() const { return w.left > 0; }
  __device__ int step() const { return w.step + i; }
  __device__ void next() {
    if (++i < w.here()) return;
    i = 0;
    w.next_tile();
  }
  __device__ void skip(int n) {
    for (; n > 0 && more(); --n) next();
  }
};

template <int D>
struct Shape {
  static constexpr int G = D / 64;               // scale groups of a key
  static constexpr int QSUB = TILE * 128;        // bytes of 64 channels of a tile of 128 rows or keys
  static constexpr int Q_BYTES = G * QSUB;
  static constexpr int N = D > 128 ? 64 : 128;   // columns of a product
  static constexpr int SLOT = G * N;             // and of TMEM, a group of channels after the other
  static constexpr int SLOTS = 512 / SLOT;       // products that have a place
  static constexpr int RK = D > 128 ? 64 : 128;  // keys that are copied at a time
  static constexpr int R_BYTES = RK * D;
  // ---- stats_kernel
  static constexpr int KT = RK;                  // keys of a step
  static constexpr int NT = D > 128 ? 1 : 2;     // row tiles of a step: converted keys serve them all
  static constexpr int KSUB = KT * 128, K_BYTES = G * KSUB, PER_A = KT / N;
  static constexpr int NQ = 1, NK = D > 128 ? 3 : 2, NR = 3;   // buffers of queries, keys, raw keys
  static constexpr int A_K = NQ * NT * Q_BYTES;
  static constexpr int A_R = A_K + NK * K_BYTES;
  static constexpr int A_SCALE = A_R + NR * R_BYTES;
  static constexpr int SCALES = KT * G * 4;
  static constexpr int A_BAR = A_SCALE + NS * SCALES;
  static constexpr int A_TOTAL = A_BAR + 512 + 1024;
  // ---- sums_kernel
  static constexpr int PER_B = TILE / N;         // products of a unit
  static constexpr int BQ = D > 128 ? 2 : 3, BK = D > 128 ? 1 : 2, BR = D > 128 ? 1 : 2;
  static constexpr int TSUB = TILE * 128, T_BYTES = G * TSUB;  // a tile of 128 keys
  static constexpr int B_Q = BK * T_BYTES;
  static constexpr int B_R = B_Q + BQ * Q_BYTES;
  static constexpr int B_LSE = B_R + BR * R_BYTES;
  static constexpr int B_SCALE = B_LSE + NS * TILE * 4;        // [NC][G][128]
  static constexpr int NC = 2;
  static constexpr int B_BAR = B_SCALE + NC * G * TILE * 4;
  static constexpr int B_TOTAL = B_BAR + 512 + 1024;
  static_assert(SLOTS % GROUPS == 0, "a slot is always the same group's");
  static_assert(A_TOTAL + sizeof(Plan) <= 227 * 1024 && B_TOTAL + sizeof(Plan) <= 227 * 1024,
                "exceeds the shared memory of one CTA");
};

constexpr int TMA_WAIT = STATUS_TMA_WAIT, MMA_WAIT = STATUS_MMA_WAIT;
constexpr int EPILOGUE_WAIT = STATUS_EPILOGUE_WAIT, DECODE_WAIT = STATUS_DECODE_WAIT;

// The bounded wait of common.cuh for warps that wait most of the time: each try may sleep for as long as
// the second number says, in nanoseconds, and takes no issue slots meanwhile.  (Twenty-eight warps that
// poll took half of them.)
__device__ __forceinline__ bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(100000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint64_t* bar, uint32_t parity, int* status, int code,
                                          int detail) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long limit = wait_limit(status), start = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (clock64() - start > limit) {
      report_status(status, code, detail);
      return false;
    }
  }
  return true;
}

// Descriptors by their lower words, which are where an operand starts; the upper one is the same for all
// tiles here (K-major rows of 128 bytes, swizzled, groups of eight 1024 bytes apart).
constexpr uint32_t DESC_HIGH = 1024 >> 4 | 1u << 14 | static_cast<uint32_t>(UMMA_SWIZZLE_128B) << 29;
__device__ __forceinline__ uint32_t desc_low(const void* tile) {
  return (smem_u32(tile) & 0x3ffff) >> 4 | 1u << 16;
}
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t tmem_d, uint32_t a_low, uint32_t b_low,
                                       uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      ".reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "mov.b64 a, {%1, %6};\n\t"
      "mov.b64 b, {%2, %6};\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(a_low), "r"(b_low), "r"(idesc), "r"(accumulate), "r"(leader), "r"(DESC_HIGH)
      : "memory");
}
// 32 lanes, a row each
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[16]) {       // 16 columns
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_rows(uint32_t taddr, uint32_t (&r)[8]) {        // 8 columns
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 pair_at(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}
// Eight INT8 values -> eight FP16 values, exactly: 0x64xx is 1024 + xx, and 1152 is subtracted.
__device__ __forceinline__ uint4 integers_fp16(uint32_t w0, uint32_t w1) {
  const __half2 bias = __half2half2(__ushort_as_half(0x6480));
  const uint32_t x0 = w0 ^ 0x80808080u, x1 = w1 ^ 0x80808080u;
  uint32_t h[4] = {__byte_perm(x0, 0x64646464u, 0x4140), __byte_perm(x0, 0x64646464u, 0x4342),
                   __byte_perm(x1, 0x64646464u, 0x4140), __byte_perm(x1, 0x64646464u, 0x4342)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h[i]), bias);
    h[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
}
// Sixteen channels (unit c of a key's D / 16) into swizzled tiles of 64 channels, `sub` bytes each.
// Lanes of every other group of channels store their second half first: eight lanes that store
// together then meet on no bank.
__device__ __forceinline__ void place(unsigned char* to, int sub, const uint4& raw, int key, int c) {
  unsigned char* dst = to + (c / 4) * sub;
  const bool swap = c & 4;
  const uint4 lo = integers_fp16(swap ? raw.z : raw.x, swap ? raw.w : raw.y);
  const uint4 hi = integers_fp16(swap ? raw.x : raw.z, swap ? raw.y : raw.w);
  *reinterpret_cast<uint4*>(dst + swz128(key, (c % 4) * 2 + swap)) = lo;
  *reinterpret_cast<uint4*>(dst + swz128(key, (c % 4) * 2 + !swap)) = hi;
}

// Keys as they were copied, rows of D bytes, to FP16 integers in swizzled tiles, from key `at` on.  By
// THREADS_ threads.
template <int D, int PER, int THREADS_>
__device__ __forceinline__ void convert(const unsigned char* from, unsigned char* to, int sub, int t, int at) {
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const int x = t + j * THREADS_;
    place(to, sub, *reinterpret_cast<const uint4*>(from + x * 16), at + x / (D / 16), x % (D / 16));
  }
}

// Where a role that goes ahead reads its next keys: their page, asked for a turn before, the first key's
// place on it and the head.  A page that does not exist is reported, and page 0 is read instead.
struct Ahead {
  int page = 0, at = 0, h = 0;
  __device__ void ask(const Geometry& g, const Chunk& ch, int key, int head) {
    page = g.page_table[static_cast<size_t>(ch.slot) * g.max_pages + (key >> 7)];
    at = key & 127;
    h = head;
  }
  __device__ int row(const Geometry& g, int* status) const {             // of the cache
    const bool there = page >= 0 && page < g.num_pages;
    if (!there) report_status(status, STATUS_BAD_INDEX, 0x71);
    return (there ? page * 128 : 0) + at;
  }
};

// The rows of the query tiles that no copy writes hold zeros: their scores are 0, not what was there.
__device__ __forceinline__ void clear_tails(unsigned char* q, int tiles, int rows) {
  const int tail = (TILE - rows) * 8;            // 16-byte units of 64 channels
  for (int i = threadIdx.x; i < tiles * tail; i += THREADS)
    *reinterpret_cast<uint4*>(q + i / tail * (TILE * 128) + rows * 128 + i % tail * 16) =
        make_uint4(0, 0, 0, 0);
  fence_proxy_async();
}

// lse: [tiles + CTAs][2 groups][2 halves][128], log2 of the sum of weights that a group has seen in half of the
// columns, of its row tile or of the one that there is; span: a tile's first and last CTA.
template <int D>
__global__ void __launch_bounds__(THREADS, 1) stats_kernel(
    const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
    const Geometry g, const __half* ks, float* lse, int* span, int* status) {
  using L = Shape<D>;
  constexpr int G = L::G, KT = L::KT, N = L::N, PER = L::PER_A, NQ = L::NQ, NK = L::NK, NR = L::NR;
  constexpr int SLOTS = L::SLOTS, NT = L::NT;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ Plan plan;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::A_BAR);
  uint64_t* q_full = bars;                       // [NQ] a tile's queries
  uint64_t* q_free = q_full + NQ;                // [NQ] its last product is through
  uint64_t* r_full = q_free + NQ;                // [NR] a unit's keys as the cache has them
  uint64_t* r_free = r_full + NR;                // [NR] they have been read
  uint64_t* k_full = r_free + NR;                // [NK] and as FP16 integers
  uint64_t* k_free = k_full + NK;                // [NK] its products are through
  uint64_t* s_full = k_free + NK;                // [SLOTS] scores of a product
  uint64_t* s_free = s_full + SLOTS;             // [SLOTS] they have been read (an arrival per warp)
  uint64_t* c_full = s_free + SLOTS;             // [NS] a unit's scales
  uint64_t* c_free = c_full + NS;                // [NS] they have been used (the same)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(c_free + NS);
  const int tid = threadIdx.x, warp = warp_same(tid >> 5), lane = tid & 31;
  if (tid == 0) {
    for (int b = 0; b < NQ; ++b) {
      mbar_init(&q_full[b], 1);
      mbar_init(&q_free[b], 1);
    }
    for (int b = 0; b < NR; ++b) {
      mbar_init(&r_full[b], 1);
      mbar_init(&r_free[b], DQ_WARPS);
    }
    for (int b = 0; b < NK; ++b) {
      mbar_init(&k_full[b], DQ_WARPS);
      mbar_init(&k_free[b], 1);
    }
    for (int b = 0; b < SLOTS; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&s_free[b], EP_GROUP);
    }
    for (int b = 0; b < NS; ++b) {
      mbar_init(&c_full[b], 1);
      mbar_init(&c_free[b], EP_GROUP * NT);
    }
    mbar_fence_init();
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
  }
  if (g.per * g.rep < TILE) clear_tails(smem, NQ * NT * G, g.per * g.rep);
  grid_wait();
  make_plan<KT, NT>(plan, g, status);
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_same(*tmem_slot);
  grid_release();
  bool ok = true;

  if (warp == TMA_WARP) {
    Units<KT, NT> u(g, plan);
    if (lane == 0) {
      int n = 0, i = 0;                            // tiles, units
      Ahead next;
      if (u.more()) next.ask(g, u.w.ch, u.step() * KT, u.w.h);
      bool fresh = true;
      while (u.more()) {
        if (fresh) {
          const int b = n % NQ;
          if (n >= NQ && !mbar_wait(&q_free[b], (n / NQ - 1) & 1, status, TMA_WAIT, 0x10)) break;
          mbar_expect_tx(&q_full[b], static_cast<uint32_t>(NT * G) * 64 * 2 * g.rep * g.per);
          for (int s = 0; s < NT * G; ++s)         // (rows behind the last are zeros)
            tma_load_3d(smem + (b * NT * G + s) * L::QSUB, &tmap_q, &q_full[b], s % G * 64, u.w.h * g.rep,
                        u.w.ch.row_start + (u.w.tile * NT + s / G) * g.per);
          ++n;
        }
        const int b = i % NR, h = next.h, row = next.row(g, status), tile = u.w.index;
        u.next();
        if (u.more()) next.ask(g, u.w.ch, u.step() * KT, u.w.h);
        fresh = u.w.index != tile;
        if (i >= NR && !mbar_wait(&r_free[b], (i / NR - 1) & 1, status, TMA_WAIT, 0x11)) break;
        mbar_expect_tx(&r_full[b], L::R_BYTES);
        tma_load_3d(smem + L::A_R + b * L::R_BYTES, &tmap_k, &r_full[b], 0, h, row);
        ++i;
      }
      for (int j = max(n - NQ, 0); j < n; ++j)     // our copies have landed before exit
        mbar_wait(&q_full[j % NQ], (j / NQ) & 1, status, TMA_WAIT, 0x12);
      for (int j = max(i - NR, 0); j < i; ++j)
        mbar_wait(&r_full[j % NR], (j / NR) & 1, status, TMA_WAIT, 0x13);
    }
  } else if (warp == MMA_WARP) {
    constexpr uint32_t idesc = umma_idesc(1, 0, 0, 0, 0, TILE, N);
    const uint32_t leader = elect_one();
    const uint32_t qd = desc_low(smem);
    const uint32_t kd = desc_low(smem + L::A_K);
    int n = 0, i = 0, x = 0;                       // tiles, units, products
    for (Walk<KT, NT> w(g, plan); warp_same(w.left) > 0 && ok; w.next_tile(), ++n) {
      const int last = i + warp_same(w.here());
      ok = warp_all(mbar_wait(&q_full[n % NQ], (n / NQ) & 1, status, MMA_WAIT, 0x14));
      const uint32_t qb = qd + n % NQ * NT * (L::Q_BYTES / 16);
      for (; i < last && ok; ++i) {
        const int b = i % NK;
        ok = warp_all(mbar_wait(&k_full[b], (i / NK) & 1, status, MMA_WAIT, 0x15));
        for (int p = 0; p < PER * NT && ok; ++p, ++x) {          // by turns of the row tiles
          const int s = x % SLOTS;
          if (x >= SLOTS) ok = mbar_wait(&s_free[s], (x / SLOTS - 1) & 1, status, MMA_WAIT, 0x16);
          ok = warp_all(ok);
          tc_fence_after();
          if (!ok) break;
          const uint32_t kb = kd + b * (L::K_BYTES / 16) + p / NT * (N * 128 / 16);
          const uint32_t qt = qb + p % NT * (L::Q_BYTES / 16);
#pragma unroll
          for (int c = 0; c < G; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ss(leader, tmem + L::SLOT * s + c * N, qt + (c * L::QSUB + k * 32) / 16,
                     kb + (c * L::KSUB + k * 32) / 16, idesc, k != 0 ? 1u : 0u);
          tc_commit_by(leader, &s_full[s]);
        }
        if (ok) tc_commit_by(leader, &k_free[b]);
      }
      if (ok) tc_commit_by(leader, &q_free[n % NQ]);
    }
    __syncwarp();
  } else if (warp >= AUX_WARP) {
    // ---------------- scales times log2 e / sqrt D, pairs of keys by groups
    constexpr int KS = KT * G / 32;
    const float qscale = rsqrtf(static_cast<float>(D)) * 1.4426950408889634f;
    __half raw[KS];
    Ahead next;
    Units<KT, NT> u(g, plan);
    auto ask = [&] {
      if (u.more()) next.ask(g, u.w.ch, u.step() * KT, u.w.h);
    };
    auto fetch = [&] {                             // what `next` names, and the page behind it
      const size_t cell = static_cast<size_t>(next.row(g, status)) * g.kvh + next.h;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const int x = lane + 32 * j;
        raw[j] = ks[(cell + static_cast<size_t>(x / G) * g.kvh) * G + x % G];
      }
      u.skip(AUX_WARPS);
      ask();
    };
    const int mine = warp - AUX_WARP, units = max(u.w.left, 0);
    u.skip(mine);
    ask();
    if (mine < units) fetch();
    for (int i = mine; i < units; i += AUX_WARPS) {
      const int b = i % NS;
      if (i >= NS) ok = mbar_wait(&c_free[b], (i / NS - 1) & 1, status, DECODE_WAIT, 0x17);
      ok = warp_all(ok);
      if (!ok) break;
      float* sk = reinterpret_cast<float*>(smem + L::A_SCALE + b * L::SCALES);
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const int x = lane + 32 * j, key = x / G, c = x % G;
        sk[((key >> 1) * G + c) * 2 + (key & 1)] = __half2float(raw[j]) * qscale;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&c_full[b]);
      if (i + AUX_WARPS < units) fetch();
    }
  } else if (warp >= EP_WARPS) {
    // ---------------- keys: INT8 to FP16 integers
    constexpr int DQ = DQ_WARPS * 32, KI = L::R_BYTES / 16 / DQ;
    const int t = tid - EP_WARPS * 32, units = max(Walk<KT, NT>(g, plan).left, 0);
    for (int i = 0; i < units; ++i) {
      const int b = i % NK, r = i % NR;
      ok = mbar_wait(&r_full[r], (i / NR) & 1, status, DECODE_WAIT, 0x18) &&
           (i < NK || mbar_wait(&k_free[b], (i / NK - 1) & 1, status, DECODE_WAIT, 0x19));
      ok = warp_all(ok);
      if (!ok) break;
      convert<D, KI, DQ>(smem + L::A_R + r * L::R_BYTES, smem + L::A_K + b * L::K_BYTES, L::KSUB, t, 0);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&k_full[b]);
        mbar_arrive(&r_free[r]);
      }
    }
  } else {
    // ---------------- a row per lane; a group has a row tile, or every other unit
    constexpr int CB = G > 1 ? 8 : 16;           // columns that are read at a time
    constexpr int EVERY = GROUPS / NT;
    const int group = warp >> 3, half = warp >> 2 & 1, at = (warp & 3) * 32 + lane;
    const uint32_t scores = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    static_assert(PER == 1, "a product for each row tile");
    int i = 0;
    for (Walk<KT, NT> w(g, plan); w.left > 0 && ok; w.next_tile()) {
      const int p = (w.tile * NT + group % NT) * g.per + at / g.rep;
      // keys that the row sees, and those that all rows of the warp see
      const int sees = at < g.per * g.rep && p < w.ch.q_len ? w.ch.pos0 + p + 1 : 0;
      const int all_see = __reduce_min_sync(0xffffffffu, sees);
      float m_ref = 0.f;
      float2 sum = make_float2(0.f, 0.f);
      const int n = w.here();
      bool start = true;
      for (int j0 = EVERY > 1 ? (i ^ group) & 1 : 0; j0 < n; j0 += EVERY) {
        const int u = i + j0, cb = u % NS, x = u * NT + group % NT, slot = x % SLOTS;
        ok = warp_all(mbar_wait(&c_full[cb], (u / NS) & 1, status, EPILOGUE_WAIT, 0x1b) &&
                      mbar_wait(&s_full[slot], (x / SLOTS) & 1, status, EPILOGUE_WAIT, 0x1a));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int p0 = 0; p0 < N / 2; p0 += COLS) {
          const int k0 = half * (N / 2) + p0, key0 = (w.step + j0) * KT + k0;
          const float2* scales =
              reinterpret_cast<const float2*>(smem + L::A_SCALE + cb * L::SCALES) + k0 / 2 * G;
          // ---- scores less the reference
          float2 y[COLS / 2];
          uint32_t raw[G][CB];
#pragma unroll
          for (int k = 0; k < COLS; k += CB) {
#pragma unroll
            for (int c = 0; c < G; ++c) tmem_ld_rows(scores + L::SLOT * slot + c * N + k0 + k, raw[c]);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < CB / 2; ++j) {
              const float2* f = scales + (k / 2 + j) * G;
              float2 fg[G];
              if (G == 1) {
                fg[0] = f[0];
              } else {
#pragma unroll
                for (int c = 0; c < G; c += 2) {
                  const float4 v = *reinterpret_cast<const float4*>(f + c);
                  fg[c] = make_float2(v.x, v.y);
                  fg[(c + 1) % G] = make_float2(v.z, v.w);
                }
              }
              float2 v = make_float2(-m_ref, -m_ref);
#pragma unroll
              for (int c = 0; c < G; ++c) v = fma2(pair_at(raw[c][2 * j], raw[c][2 * j + 1]), fg[c], v);
              y[k / 2 + j] = v;
            }
          }
          if (p0 + COLS == N / 2) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&s_free[slot]);
              mbar_arrive(&c_free[cb]);
            }
          }
          if (all_see < key0 + COLS) {
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) {
              if (key0 + 2 * j >= sees) y[j].x = -INFINITY;
              if (key0 + 2 * j + 1 >= sees) y[j].y = -INFINITY;
            }
          }
          // ---- weights.  The reference is the maximum of the row's first columns, and moves where weights are
          // far above 1: no maximum is taken but then.  (A row that sees none of the first sees none behind.)
          auto weights = [&] {                     // chains of sums of a quarter of the columns
            float2 v[4];
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) {
              const float2 e = make_float2(ex2(y[j].x), ex2(y[j].y));
              v[j & 3] = j < 4 ? e : add2(v[j & 3], e);
            }
            return add2(add2(v[0], v[1]), add2(v[2], v[3]));
          };
          float2 more = make_float2(0.f, 0.f);
          if (!start) more = weights();
          if (__any_sync(0xffffffffu, start || more.x + more.y > FAR)) {
            float top = fmaxf(y[0].x, y[0].y);
#pragma unroll
            for (int j = 1; j < COLS / 2; ++j) top = fmaxf(top, fmaxf(y[j].x, y[j].y));
            const float by = top == -INFINITY ? 0.f : start ? top : fmaxf(top, 0.f);
            const float f = start ? 0.f : ex2(-by);
            sum = mul2(sum, make_float2(f, f));
            m_ref += by;
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) y[j] = add2(y[j], make_float2(-by, -by));
            more = weights();
            start = false;
          }
          sum = add2(sum, more);
        }
      }
      if (!ok) break;
      i += n;
      const float l = sum.x + sum.y;
      lse[(static_cast<size_t>(w.index + blockIdx.x) * PARTS + group * 2 + half) * TILE + at] =
          l == 0.f ? -INFINITY : m_ref + log2f(l);
      if (tid == 0) {
        if (w.step == 0) span[2 * w.index] = blockIdx.x;
        if (w.step + n == w.steps) span[2 * w.index + 1] = blockIdx.x;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
}

// A CTA per row tile, KV head and chunk: what the tile's CTAs have left becomes the rows' lse, negative, at
// [row tiles][128]; a row that is none gets one that leaves no weight.  Few rows behind many keys leave as
// many parts as there are CTAs to a tile: those are joined in blockDim.y interleaved slices, eight loads
// at a time (16 rows behind 20000 keys, two tiles of 74 CTAs: 64 us one after the other, now 9.7).
constexpr int JOIN_SLICES = 8;
template <int NT>
__global__ void __launch_bounds__(TILE * JOIN_SLICES) join_kernel(const Geometry g, const float* lse,
                                                                  const int* span, float* rows) {
  __shared__ float2 s_part[JOIN_SLICES][TILE];
  grid_wait();
  grid_release();
  const int c = blockIdx.z, h = blockIdx.y, rt = blockIdx.x, at = threadIdx.x;
  const int slice = threadIdx.y, slices = blockDim.y;
  const Chunk ch = g.at(c);
  if (rt * g.per >= ch.q_len) return;
  int base = 0, tiles = 0;                         // of the chunks before: tiles, row tiles
  for (int d = 0; d < c; ++d) {
    const Chunk other = g.at(d);
    base += Order<1, NT>::tiles(g, other) * g.kvh;
    tiles += Order<1, 1>::tiles(g, other) * g.kvh;
  }
  const int index = base + h * Order<1, NT>::tiles(g, ch) + rt / NT;
  const int2 of = span_of(span, index);
  float m = -INFINITY, l = 0.f;
  auto join = [&](float v, float weight, float top) {
    return v == -INFINITY ? 0.f : weight * exp2f(v - top);
  };
  constexpr int OWN = NT > 1 ? 2 : PARTS, AHEAD = 8;             // parts of a CTA; loads in flight
  const float* from = lse + (static_cast<size_t>(index + of.x) * PARTS + rt % NT * 2) * TILE + at;
  const int n = (of.y - of.x + 1) * OWN;
  for (int x0 = slice; x0 < n; x0 += AHEAD * slices) {
    float v[AHEAD];
    float top = m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int x = x0 + k * slices;
      v[k] = x < n ? from[(x / OWN * PARTS + x % OWN) * TILE] : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) top = fmaxf(top, v[k]);
    l = join(m, l, top);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) l += join(v[k], 1.f, top);
    m = top;
  }
  if (slices > 1) {
    s_part[slice][at] = make_float2(m, l);
    __syncthreads();
    if (slice > 0) return;
    float top = m;
    for (int k = 1; k < slices; ++k) top = fmaxf(top, s_part[k][at].x);
    l = join(m, l, top);
    for (int k = 1; k < slices; ++k) l += join(s_part[k][at].x, s_part[k][at].y, top);
    m = top;
  }
  const bool there = at < min(g.per, ch.q_len - rt * g.per) * g.rep;
  rows[(static_cast<size_t>(tiles) + h * Order<1, 1>::tiles(g, ch) + rt) * TILE + at] =
      there ? -m - log2f(l) : -INFINITY;
}

// rows: join_kernel's.  parts: [key tiles + CTAs][2 groups][2 halves][128], sums of what they have seen;
// span_out: a key tile's first and last CTA.
template <int D>
__global__ void __launch_bounds__(THREADS, 1) sums_kernel(
    const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
    const Geometry g, const __half* ks, const float* rows, float* parts, int* span_out, int* status) {
  using L = Shape<D>;
  constexpr int G = L::G, N = L::N, PER = L::PER_B, BQ = L::BQ, BK = L::BK, BR = L::BR, NC = L::NC;
  constexpr int SLOTS = L::SLOTS, HALVES = TILE / L::RK;         // copies of a tile's keys
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  __shared__ Plan plan;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::B_BAR);
  uint64_t* r_full = bars;                       // [BR] keys as the cache has them
  uint64_t* r_free = r_full + BR;                // [BR] they have been read
  uint64_t* k_full = r_free + BR;                // [BK] a tile's keys as FP16 integers
  uint64_t* k_free = k_full + BK;                // [BK] its last product is through
  uint64_t* q_full = k_free + BK;                // [BQ] a unit's queries
  uint64_t* q_free = q_full + BQ;                // [BQ] its products are through
  uint64_t* s_full = q_free + BQ;                // [SLOTS] scores of a product
  uint64_t* s_free = s_full + SLOTS;             // [SLOTS] they have been read (an arrival per warp)
  uint64_t* l_full = s_free + SLOTS;             // [NS] a unit's lse
  uint64_t* l_free = l_full + NS;                // [NS] they have been used (an arrival per warp)
  uint64_t* c_full = l_free + NS;                // [NC] a tile's scales
  uint64_t* c_free = c_full + NC;                // [NC] they have been read (an arrival per warp)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(c_free + NC);
  const int tid = threadIdx.x, warp = warp_same(tid >> 5), lane = tid & 31;
  if (tid == 0) {
    for (int b = 0; b < BR; ++b) {
      mbar_init(&r_full[b], 1);
      mbar_init(&r_free[b], DQ_WARPS);
    }
    for (int b = 0; b < BK; ++b) {
      mbar_init(&k_full[b], DQ_WARPS);
      mbar_init(&k_free[b], 1);
    }
    for (int b = 0; b < BQ; ++b) {
      mbar_init(&q_full[b], 1);
      mbar_init(&q_free[b], 1);
    }
    for (int b = 0; b < SLOTS; ++b) {
      mbar_init(&s_full[b], 1);
      mbar_init(&s_free[b], EP_GROUP);
    }
    for (int b = 0; b < NS; ++b) {
      mbar_init(&l_full[b], 1);
      mbar_init(&l_free[b], EP_GROUP * PER);
    }
    for (int b = 0; b < NC; ++b) {
      mbar_init(&c_full[b], DQ_WARPS);
      mbar_init(&c_free[b], EP_WARPS);
    }
    mbar_fence_init();
    prefetch_tmap(&tmap_q);
    prefetch_tmap(&tmap_k);
  }
  if (g.per * g.rep < TILE) clear_tails(smem + L::B_Q, BQ * G, g.per * g.rep);
  grid_wait();
  make_plan<0>(plan, g, status);
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_same(*tmem_slot);
  grid_release();
  bool ok = true;

  if (warp == TMA_WARP) {
    Units<0> u(g, plan);
    if (lane == 0) {
      int n = 0, copied = 0, base_c = 0, base = 0;             // row tiles of the chunks before
      for (; u.more(); u.next(), ++n) {
        const int b = n % BQ, lb = n % NS, rt = u.w.first + u.step();
        for (; base_c < u.w.c; ++base_c) base += Order<1>::tiles(g, g.at(base_c)) * g.kvh;
        const int index = base + u.w.h * Order<1>::tiles(g, u.w.ch) + rt;
        if (n >= NS && !mbar_wait(&l_free[lb], (n / NS - 1) & 1, status, TMA_WAIT, 0x25)) break;
        mbar_expect_tx(&l_full[lb], TILE * 4);
        bulk_load(smem + L::B_LSE + lb * TILE * 4, rows + static_cast<size_t>(index) * TILE, TILE * 4,
                  &l_full[lb]);
        ++copied;
        if (n >= BQ && !mbar_wait(&q_free[b], (n / BQ - 1) & 1, status, TMA_WAIT, 0x20)) break;
        mbar_expect_tx(&q_full[b], static_cast<uint32_t>(G) * 64 * 2 * g.rep * g.per);
        for (int s = 0; s < G; ++s)
          tma_load_3d(smem + L::B_Q + b * L::Q_BYTES + s * L::QSUB, &tmap_q, &q_full[b], s * 64,
                      u.w.h * g.rep, u.w.ch.row_start + rt * g.per);
      }
      for (int i = max(n - BQ, 0); i < n; ++i)     // our copies have landed before exit
        mbar_wait(&q_full[i % BQ], (i / BQ) & 1, status, TMA_WAIT, 0x21);
      for (int i = max(copied - NS, 0); i < copied; ++i)
        mbar_wait(&l_full[i % NS], (i / NS) & 1, status, TMA_WAIT, 0x2e);
    }
  } else if (warp == MMA_WARP) {
    constexpr uint32_t idesc = umma_idesc(1, 0, 0, 0, 0, TILE, N);
    const uint32_t leader = elect_one();
    const uint32_t kd = desc_low(smem);
    const uint32_t qd = desc_low(smem + L::B_Q);
    int n = 0, i = 0, x = 0;                       // tiles, units, products
    for (Walk<0> w(g, plan); warp_same(w.left) > 0 && ok; w.next_tile(), ++n) {
      const int last = i + warp_same(w.here());
      ok = warp_all(mbar_wait(&k_full[n % BK], (n / BK) & 1, status, MMA_WAIT, 0x22));
      const uint32_t kb = kd + n % BK * (L::T_BYTES / 16);
      for (; i < last && ok; ++i) {
        const int b = i % BQ;
        ok = warp_all(mbar_wait(&q_full[b], (i / BQ) & 1, status, MMA_WAIT, 0x23));
        for (int p = 0; p < PER && ok; ++p, ++x) {
          const int s = x % SLOTS;
          if (x >= SLOTS) ok = mbar_wait(&s_free[s], (x / SLOTS - 1) & 1, status, MMA_WAIT, 0x24);
          ok = warp_all(ok);
          tc_fence_after();
          if (!ok) break;
          const uint32_t qb = qd + b * (L::Q_BYTES / 16) + p * (N * 128 / 16);
#pragma unroll
          for (int c = 0; c < G; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ss(leader, tmem + L::SLOT * s + c * N, kb + (c * L::TSUB + k * 32) / 16,
                     qb + (c * L::QSUB + k * 32) / 16, idesc, k != 0 ? 1u : 0u);
          tc_commit_by(leader, &s_full[s]);
        }
        if (ok) tc_commit_by(leader, &q_free[b]);
      }
      if (ok) tc_commit_by(leader, &k_free[n % BK]);
    }
    __syncwarp();
  } else if (warp >= AUX_WARP) {                   // (scales come with the keys)
  } else if (warp >= EP_WARPS) {
    // ---------------- keys: a tile, INT8 to FP16 integers, and their scales.  The copies are this role's
    // own, BR ahead: the first lane of its first warp asks for them.
    constexpr int DQ = DQ_WARPS * 32, KI = L::R_BYTES / 16 / DQ;
    const int t = tid - EP_WARPS * 32;
    const float qscale = rsqrtf(static_cast<float>(D)) * 1.4426950408889634f;
    __half scale[G];
    Ahead next;
    Walk<0> w(g, plan);
    int n = 0, y = 0, asked = 0;                   // tiles, copies used and asked for
    int tile_row[2] = {0, 0}, tile_h[2] = {0, 0};  // the tile at work and the next one
    int tiles = 0;                                 // known so far
    auto ask = [&] {
      if (w.left > 0) next.ask(g, w.ch, w.tile * TILE, w.h);
    };
    auto know = [&] {                              // the tile that `next` names, and the page behind it
      if (w.left <= 0) return;
      tile_row[tiles & 1] = next.row(g, status);
      tile_h[tiles & 1] = next.h;
      ++tiles;
      w.next_tile();
      ask();
    };
    // The copies of the tiles that are known, as far as buffers are free (their last use was BR copies ago).
    auto copy = [&] {
      if (t == 0) for (; asked < tiles * HALVES && asked < y + BR; ++asked) {
        const int r = asked % BR, of = asked / HALVES & 1;
        if (asked >= BR && !mbar_wait(&r_free[r], (asked / BR - 1) & 1, status, TMA_WAIT, 0x29)) return;
        mbar_expect_tx(&r_full[r], L::R_BYTES);
        tma_load_3d(smem + L::B_R + r * L::R_BYTES, &tmap_k, &r_full[r], 0, tile_h[of],
                    tile_row[of] + asked % HALVES * L::RK);
      }
    };
    ask();
    know();
    copy();
    for (; n < tiles; ++n) {
      const int b = n % BK, cb = n % NC;
      const size_t cell = (static_cast<size_t>(tile_row[n & 1]) + (t & (TILE - 1))) * g.kvh + tile_h[n & 1];
#pragma unroll
      for (int c = 0; c < G; ++c) scale[c] = ks[cell * G + c];
      know();
      copy();
      __syncwarp();
      ok = warp_all(n < BK || mbar_wait(&k_free[b], (n / BK - 1) & 1, status, DECODE_WAIT, 0x26));
      for (int part = 0; part < HALVES && ok; ++part) {
        const int r = y % BR;
        ok = warp_all(mbar_wait(&r_full[r], (y / BR) & 1, status, DECODE_WAIT, 0x2b));
        if (!ok) break;
        convert<D, KI, DQ>(smem + L::B_R + r * L::R_BYTES, smem + b * L::T_BYTES, L::TSUB, t, part * L::RK);
        __syncwarp();
        if (lane == 0) mbar_arrive(&r_free[r]);
        ++y;
        copy();
        __syncwarp();
      }
      if (!ok) break;
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[b]);
      if (n >= NC) ok = mbar_wait(&c_free[cb], (n / NC - 1) & 1, status, DECODE_WAIT, 0x2c);
      ok = warp_all(ok);
      if (!ok) break;
      float* sc = reinterpret_cast<float*>(smem + L::B_SCALE + cb * G * TILE * 4);
#pragma unroll
      for (int c = 0; c < G; ++c)
        if (t < TILE) sc[c * TILE + t] = __half2float(scale[c]) * qscale;
      __syncwarp();
      if (lane == 0) mbar_arrive(&c_full[cb]);
    }
    if (t == 0)                                    // our copies have landed before exit
      for (int i = y; i < asked; ++i)
        mbar_wait(&r_full[i % BR], (i / BR) & 1, status, TMA_WAIT, 0x2d);
    __syncwarp();
  } else {
    // ---------------- sums: a key per lane; a group has every other unit, or half of the rows of each
    constexpr int CB = G > 1 ? 8 : 16;             // columns that are read at a time
    constexpr int EVERY = GROUPS / PER;
    const int group = warp >> 3, half = warp >> 2 & 1, key_at = (warp & 3) * 32 + lane, part = group % PER * N;
    const uint32_t scores = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    int i = 0, n = 0;                              // units, tiles
    for (Walk<0> w(g, plan); w.left > 0 && ok; w.next_tile(), ++n) {
      const int cb = n % NC, here = w.here();
      ok = warp_all(mbar_wait(&c_full[cb], (n / NC) & 1, status, EPILOGUE_WAIT, 0x2a));
      if (!ok) break;
      float2 f[G];
#pragma unroll
      for (int c = 0; c < G; ++c) {
        const float v = *reinterpret_cast<const float*>(smem + L::B_SCALE + ((cb * G + c) * TILE + key_at) * 4);
        f[c] = make_float2(v, v);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&c_free[cb]);
      // of the chunk's rows times heads those from `see` on see the key
      const int see = (w.tile * TILE + key_at - w.ch.pos0) * g.rep, last = w.ch.q_len * g.rep;
      const int see_all = (w.tile * TILE + TILE - 1 - w.ch.pos0) * g.rep;    // and all keys of the tile
      float2 total = make_float2(0.f, 0.f);
      for (int j0 = EVERY > 1 ? (i ^ group) & 1 : 0; j0 < here; j0 += EVERY) {
        const int u = i + j0, lb = u % NS, x = PER * u + group % PER, slot = x % SLOTS;
        const int pos = (w.first + w.step + j0) * g.per;           // of the unit's first row
        ok = warp_all(mbar_wait(&l_full[lb], (u / NS) & 1, status, EPILOGUE_WAIT, 0x28) &&
                      mbar_wait(&s_full[slot], (x / SLOTS) & 1, status, EPILOGUE_WAIT, 0x27));
        if (!ok) break;
        tc_fence_after();
        const float* neg = reinterpret_cast<const float*>(smem + L::B_LSE + lb * TILE * 4) + part;
#pragma unroll
        for (int p0 = 0; p0 < N / 2; p0 += COLS) {
          const int k0 = half * (N / 2) + p0;
          float2 y[COLS / 2];                      // scores less the rows' lse
          uint32_t raw[G][CB];
#pragma unroll
          for (int k = 0; k < COLS; k += CB) {
#pragma unroll
            for (int c = 0; c < G; ++c) tmem_ld_rows(scores + L::SLOT * slot + c * N + k0 + k, raw[c]);
            tc_wait_ld();
#pragma unroll
            for (int j = 0; j < CB / 2; j += 2) {
              const float4 from = *reinterpret_cast<const float4*>(neg + k0 + k + 2 * j);
              float2 v[2] = {make_float2(from.x, from.y), make_float2(from.z, from.w)};
#pragma unroll
              for (int c = 0; c < G; ++c)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  v[e] = fma2(pair_at(raw[c][2 * (j + e)], raw[c][2 * (j + e) + 1]), f[c], v[e]);
              y[k / 2 + j] = v[0];
              y[k / 2 + j + 1] = v[1];
            }
          }
          if (p0 + COLS == N / 2) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              mbar_arrive(&s_free[slot]);
              mbar_arrive(&l_free[lb]);
            }
          }
#pragma unroll
          for (int j = 0; j < COLS / 2; ++j) y[j] = make_float2(ex2(y[j].x), ex2(y[j].y));
          const int first = pos * g.rep + part + k0;
          if (first < see_all || first + COLS > last) {
#pragma unroll
            for (int j = 0; j < COLS / 2; ++j) {
              const int row = first + 2 * j;
              if (row < see || row >= last) y[j].x = 0.f;
              if (row + 1 < see || row + 1 >= last) y[j].y = 0.f;
            }
          }
          float2 v[4];                             // chains of sums of a quarter of the columns
#pragma unroll
          for (int j = 0; j < COLS / 2; ++j) v[j & 3] = j < 4 ? y[j] : add2(v[j & 3], y[j]);
          total = add2(total, add2(add2(v[0], v[1]), add2(v[2], v[3])));
        }
      }
      if (!ok) break;
      i += here;
      parts[(static_cast<size_t>(w.index + blockIdx.x) * PARTS + group * 2 + half) * TILE + key_at] =
          total.x + total.y;
      if (tid == 0) {
        if (w.step == 0) span_out[2 * w.index] = blockIdx.x;
        if (w.step + here == w.steps) span_out[2 * w.index + 1] = blockIdx.x;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
}

// A CTA per key tile, ADD_HEADS KV heads and chunk: chunks of one request are added in their order by the
// first's.  A chain of small loads (chunk, span, parts, sums); a thread asks for its heads' together.
constexpr int ADD_HEADS = 4, MORE = 8;           // MORE: of a tile's further CTAs at a time
__global__ void __launch_bounds__(TILE) add_kernel(
    const Geometry g, const float* parts, const int* span, const float* weights, long long slot_stride,
    long long head_stride, float* sums, long long sums_slot_stride, long long sums_head_stride) {
  grid_wait();
  grid_release();
  const int c = blockIdx.z, h0 = blockIdx.y * ADD_HEADS, tile = blockIdx.x, tid = threadIdx.x;
  const Chunk ch = g.at(c);
  if (ch.q_len <= 0) return;
  float total[ADD_HEADS] = {};
  int base = 0, seen = 0;                          // key tiles of the chunks before; keys that are seen
  for (int d = 0; d < g.n_chunks; ++d) {
    const Chunk other = g.at(d);
    const int tiles = Order<0>::tiles(g, other);
    if (other.q_len > 0 && other.slot == ch.slot) {
      if (d < c) return;
      if (tile < tiles) {
        int2 of[ADD_HEADS];
        float v[ADD_HEADS][PARTS];
        auto place = [&](int k, int x, int part) {
          return (static_cast<size_t>(base + (h0 + k) * tiles + tile + x) * PARTS + part) * TILE + tid;
        };
#pragma unroll
        for (int k = 0; k < ADD_HEADS; ++k)
          if (h0 + k < g.kvh) of[k] = span_of(span, base + (h0 + k) * tiles + tile);
#pragma unroll
        for (int k = 0; k < ADD_HEADS; ++k)
#pragma unroll
          for (int part = 0; part < PARTS; ++part)
            if (h0 + k < g.kvh && of[k].x <= of[k].y) v[k][part] = parts[place(k, of[k].x, part)];
#pragma unroll
        for (int k = 0; k < ADD_HEADS; ++k) {
          if (h0 + k >= g.kvh || of[k].x > of[k].y) continue;
          float sum = 0.f;
#pragma unroll
          for (int part = 0; part < PARTS; ++part) sum += v[k][part];
          for (int x0 = of[k].x + 1; x0 <= of[k].y; x0 += MORE) {
            float w[MORE][PARTS];
#pragma unroll
            for (int x = 0; x < MORE; ++x)
#pragma unroll
              for (int part = 0; part < PARTS; ++part)
                w[x][part] = x0 + x <= of[k].y ? parts[place(k, x0 + x, part)] : 0.f;
#pragma unroll
            for (int x = 0; x < MORE; ++x)
#pragma unroll
              for (int part = 0; part < PARTS; ++part) sum += w[x][part];
          }
          total[k] += sum;
        }
        seen = max(seen, other.pos0 + other.q_len);
      }
    }
    base += tiles * g.kvh;
  }
  const int key = tile * TILE + tid;
  if (key >= seen) return;
  const float* from = weights + ch.slot * slot_stride + h0 * head_stride + key;
  float* to = sums + ch.slot * sums_slot_stride + h0 * sums_head_stride + key;
  float before[ADD_HEADS];
#pragma unroll
  for (int k = 0; k < ADD_HEADS; ++k)
    if (h0 + k < g.kvh) before[k] = from[k * head_stride];
#pragma unroll
  for (int k = 0; k < ADD_HEADS; ++k)
    if (h0 + k < g.kvh) to[k * sums_head_stride] = before[k] + total[k];
}

// Tiles that a call may have at most, of rows and of keys, and its units.
struct Bounds {
  long long row_tiles, key_tiles, units;
};
static Bounds bounds(int n_chunks, int max_q_len, int kvh, int rep, int limit) {
  const long long per = TILE / rep;
  const long long rows = (max_q_len + per - 1) / per * n_chunks * kvh;
  const long long keys = (limit + TILE - 1LL) / TILE;
  return {rows, keys * n_chunks * kvh, rows * keys * 2};
}

static int ctas_for(long long units) { return units < CTAS ? static_cast<int>(units) : CTAS; }

template <int D>
static int launch(const __half* q, const Geometry& g, const int8_t* kc, const __half* ks,
                  const float* weights, long long slot_stride, long long head_stride, float* sums,
                  long long sums_slot_stride, long long sums_head_stride, float* work,
                  cudaStream_t stream) {
  using L = Shape<D>;
  PFN_encodeTiled enc = runtime_tma_encoder();
  if (!enc) return -3;
  CUtensorMap tq;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(g.qh),
                        static_cast<cuuint64_t>(g.total_rows)};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(g.qh) * D * 2};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(g.rep), static_cast<cuuint32_t>(g.per)};
  cuuint32_t estr[3] = {1, 1, 1};
  if (enc(&tq, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(q), dims, strides, box, estr,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return -3;
  CUtensorMap tk;                                  // the cache as [slots][heads][D] bytes
  cuuint64_t k_dims[3] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(g.kvh),
                          static_cast<cuuint64_t>(g.num_pages) * 128};
  cuuint64_t k_strides[2] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(g.kvh) * D};
  cuuint32_t k_box[3] = {static_cast<cuuint32_t>(D), 1, static_cast<cuuint32_t>(L::RK)};
  if (enc(&tk, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<int8_t*>(kc), k_dims, k_strides, k_box, estr,
          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
    return -3;
  static const int slot[2] = {runtime_new_slot(), runtime_new_slot()};
  if (const int e = runtime_allow_smem(slot[0], stats_kernel<D>, L::A_TOTAL)) return e;
  if (const int e = runtime_allow_smem(slot[1], sums_kernel<D>, L::B_TOTAL)) return e;
  const Bounds b = bounds(g.n_chunks, g.longest, g.kvh, g.rep, g.limit);
  float* lse = work;
  float* rows = lse + (b.row_tiles + CTAS) * PARTS * TILE;
  float* parts = rows + b.row_tiles * TILE;
  int* row_span = reinterpret_cast<int*>(parts + (b.key_tiles + CTAS) * PARTS * TILE);
  int* key_span = row_span + 2 * b.row_tiles;
  const int ctas = ctas_for(b.units);
  launch_early(stats_kernel<D>, dim3(ctas), THREADS, L::A_TOTAL, stream, tq, tk, g, ks, lse, row_span,
               runtime_status_ptr());
  // Slices by the parts that a tile has where all of the CTAs are at work on as many tiles as there can be.
  // us of the join in 1, 4 and 8 of them: 296 parts 30, 11.7, 9.5; 148 18.5, 9.2, 7.9; 74 8.1, 6.5, 6.1; 37
  // 7.9, 6.4, 5.9; 18 6.1, 5.1, 5.9; 6 6.2, 6.9, 7.9; 4 4.5, 5.1, 5.8; less than one (4096 rows) 5, 12.5, 21.7.
  const long long most = PARTS * static_cast<long long>(ctas) / b.row_tiles;
  const dim3 join(TILE, most >= 64 ? JOIN_SLICES : most >= 16 ? 4 : 1);
  launch_early(join_kernel<L::NT>, dim3((g.longest + g.per - 1) / g.per, g.kvh, g.n_chunks), join, 0, stream,
               g, static_cast<const float*>(lse), static_cast<const int*>(row_span), rows);
  launch_early(sums_kernel<D>, dim3(ctas), THREADS, L::B_TOTAL, stream, tq, tk, g, ks,
               static_cast<const float*>(rows), parts, key_span, runtime_status_ptr());
  launch_early(add_kernel, dim3((g.limit + TILE - 1) / TILE, (g.kvh + ADD_HEADS - 1) / ADD_HEADS, g.n_chunks),
               TILE, 0, stream, g,
               static_cast<const float*>(parts), static_cast<const int*>(key_span), weights, slot_stride,
               head_stride, sums, sums_slot_stride, sums_head_stride);
  return static_cast<int>(cudaGetLastError());
}

}  // namespace kw
}  // namespace orinfer

using namespace orinfer;

extern "C" size_t orinfer_prefill_weights_work_bytes(int n_chunks, int max_q_len, int kvh, int rep,
                                                     int limit) {
  if (n_chunks <= 0 || rep <= 0) return 0;
  const kw::Bounds b = kw::bounds(n_chunks, max_q_len, kvh, rep, limit);
  return ((b.row_tiles + kw::CTAS) * kw::PARTS + b.row_tiles + (b.key_tiles + kw::CTAS) * kw::PARTS) *
             kw::TILE * sizeof(float) +
         2 * (b.row_tiles + b.key_tiles) * sizeof(int);
}

extern "C" int orinfer_prefill_weights(const __half* q, const int* chunks, int n_chunks, int max_q_len,
                                       int total_rows, const int* page_table, int slots, int max_pages,
                                       const int8_t* kc, const __half* ks, int num_pages,
                                       const float* weights, long long slot_stride, long long head_stride,
                                       float* sums, long long sums_slot_stride,
                                       long long sums_head_stride, int limit, int qh, int kvh,
                                       int head_dim, float* work, cudaStream_t stream) {
  if (n_chunks <= 0 || max_q_len <= 0 || total_rows <= 0 || limit <= 0) return 0;
  if (n_chunks > kw::MAX_CHUNKS || kvh <= 0 || qh % kvh || qh / kvh > 16 || !work) return -1;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(kc) |
        reinterpret_cast<uintptr_t>(work)) & 15) != 0)
    return -1;
  if (limit > max_pages * 128LL) return -1;
  const kw::Bounds b = kw::bounds(n_chunks, max_q_len, kvh, qh / kvh, limit);
  if (num_pages <= 0 || num_pages > (1 << 24)) return -1;
  if (b.units > 0x3fffffffLL || b.key_tiles > 0x3fffffffLL) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  kw::Geometry g;
  g.chunks = reinterpret_cast<const kw::Chunk*>(chunks);
  g.page_table = page_table;
  g.n_chunks = n_chunks;
  g.total_rows = total_rows;
  g.slots = slots;
  g.max_pages = max_pages;
  g.num_pages = num_pages;
  g.longest = max_q_len;
  g.limit = limit;
  g.qh = qh;
  g.kvh = kvh;
  g.rep = qh / kvh;
  g.per = kw::TILE / g.rep;
#define CASE(D)                                                                                     \
  if (head_dim == D)                                                                                \
    return kw::launch<D>(q, g, kc, ks, weights, slot_stride, head_stride, sums,          \
                         sums_slot_stride, sums_head_stride, work, stream);
  CASE(64) CASE(128) CASE(256)
#undef CASE
  return -1;
}
