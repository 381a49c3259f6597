// Eviction from the paged cache: of a request that has outgrown its bound each layer and KV head keeps
// the keys that attention has given the most weight, beside the first and the last ones.
//
// The page table is one for all layers and heads, but which keys a page holds is a head's own matter: a
// request keeps as many keys in each, in their order, and attention goes on as over a shorter context
// (keys carry their rotary angle).  What is kept goes to fresh pages and the old ones lose a reference,
// so pages that others share are never written, the move needs no order, and a call repeats.
//
// The first kernel looks, the second changes.  In the first, one CTA does the bookkeeping of the pages (the
// lowest free ones, in the order of the requests), and beside it one per request, layer and KV head finds
// its threshold, the weight of the last key that stays, by three histograms of the weights' bits (11, 11,
// 10), and walks the keys once: those above the threshold, and of those equal to it the first so many, go
// to a list with their weights.  In the second a CTA fills a fresh page of a layer and head from the list.
//
// The second is bound by memory: 2 (D + D / 32) bytes of a kept key's key and value read and as many
// written, pieces of D bytes in no order of pages.  36 layers of 8 heads of 128: eleven requests of 1006 to
// 1450 keys cut to 1000 292 us, 5.6 TB/s (a CTA that walks its keys itself: 390); two of 8292 and 12000 to
// 2000 117 (199); seventeen of 1137 to 2100 to 1100, 12 layers of 2 heads of 256: 62.  The first, 46, 35 and
// 13 us of these, is a
// chain of passes over weights that lie in L2.  It took 47, 40 and 13 before its walk was shortened; then
// with weights in shared memory 53, 49 and 13, since fewer CTAs are at work beside each other, and with 512
// threads 70 and 50 of the first two.
//
// The pool is gone through by the one CTA that does the bookkeeping, 256 pages at a time, all of it: a small call
// (one request of 700 keys, 2 heads of 64) takes 34 us cold in a pool of 64 or 1500 pages, 50 in one of 15000
// and 103 in one of 60000.
#include <type_traits>

#include "api.h"
#include "common.cuh"

namespace orinfer {
namespace ev {

constexpr int PAGE = 128;                          // tokens
constexpr int THREADS = 256, WARPS = THREADS / 32;               // of the first kernel
constexpr int MOVE_THREADS = 256;                  // and of the second
constexpr int LANE_KEYS = 8, BLOCK = LANE_KEYS * THREADS;        // keys of a step of the walk
constexpr int BINS = 2048;                         // of a histogram
constexpr int WORK_HEAD = 4;                       // status, -, -, -

// What the first kernel leaves: the keys that stay and their weights [items][keep]; the first naming of a
// slot [slots]; per request its rank among those that are cut (-1: it stays as it is) [n]; fresh pages
// [n][pages of `keep`]; the table rows as they were [n][max_pages].
struct Work {
  int* head;
  int2* list;
  int *named, *len, *rank, *fresh, *rows;
  __host__ __device__ Work(int* w, int slots, int n, int kept, size_t items, int keep)
      : head(w), list(reinterpret_cast<int2*>(w + WORK_HEAD)),
        named(w + WORK_HEAD + 2 * items * keep), len(named + slots), rank(len + n), fresh(rank + n),
        rows(fresh + static_cast<size_t>(n) * kept) {}
};

struct Cache {
  const long long* bases;                          // [4][layers]: keys, values, their scales
  int layers, kvh, pages;
};

__device__ __forceinline__ int block_rank(bool flag, int* warp_sums, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned votes = __ballot_sync(0xffffffffu, flag);
  __syncthreads();
  if (lane == 0) warp_sums[warp] = __popc(votes);
  __syncthreads();
  const int own = warp_sums[lane];
  const unsigned lower = lane < warp ? 0xffffffffu : 0u;
  const int before = __reduce_add_sync(0xffffffffu, own & lower);
  total = __reduce_add_sync(0xffffffffu, own);
  return before + __popc(votes & ((1u << lane) - 1u));
}

// The bookkeeping, by one CTA: which requests are cut, their fresh pages, the references of all pages.
__device__ __forceinline__ void make_plan(const Work& w, const int* table, const int* lens, const int* refs,
                                          int* refs_out, const int* list, int n, int slots,
                                          int max_pages, int pages, int keep, int* status_out) {
  __shared__ int sums[32];
  __shared__ int s_wrong;
  const int kept = (keep + PAGE - 1) / PAGE, tid = threadIdx.x;
  if (tid < 32) sums[tid] = 0;                     // (fewer warps than the scan looks at)
  if (tid == 0) s_wrong = 0;
  for (int s = tid; s < slots; s += THREADS) w.named[s] = n;
  __syncthreads();
  for (int i = tid; i < n; i += THREADS) {
    const int s = list[i];
    if (s >= 0 && s < slots)
      atomicMin(&w.named[s], i);
    else
      s_wrong = 1;
  }
  __syncthreads();
  // ---- requests: lengths that fit the table, pages that somebody holds
  for (int i = tid / 16; i < n; i += THREADS / 16) {        // sixteen lanes per request
    const int s = list[i], lane = tid & 15;
    if (s < 0 || s >= slots) {
      if (lane == 0) w.len[i] = 0;
      continue;
    }
    const int len = lens[s];
    if (lane == 0) w.len[i] = w.named[s] == i ? len : 0;         // (named again: nothing to do)
    const int* row = table + static_cast<size_t>(s) * max_pages;
    bool wrong = len < 0 || len > max_pages * PAGE;
    for (int j = lane; !wrong && len > keep && j < max_pages; j += 16) {
      const int page = row[j];
      const bool needed = j < (len + PAGE - 1) / PAGE;
      wrong = page < 0 || page >= pages || (needed && page == 0) || (page > 0 && refs[page] <= 0);
    }
    if (wrong) s_wrong = 1;
  }
  __syncthreads();
  int status = s_wrong ? 2 : 0;
  int cut = 0;
  for (int i0 = 0; i0 < n; i0 += THREADS) {
    const int i = i0 + tid;
    const bool mine = i < n && status == 0 && w.len[i] > keep;
    int total;
    const int rank = cut + block_rank(mine, sums, total);
    if (i < n) w.rank[i] = mine ? rank : -1;
    cut += total;
  }
  // ---- the free pages in ascending order are theirs
  const long long need = static_cast<long long>(cut) * kept;
  int found = 0, next = tid < pages ? refs[tid] : 1;
  for (int p0 = 0; p0 < pages; p0 += THREADS) {
    const int p = p0 + tid, held = next;
    next = p + THREADS < pages ? refs[p + THREADS] : 1;
    int total;
    const int rank = found + block_rank(p > 0 && held <= 0, sums, total);
    if (p < pages && refs_out != refs) refs_out[p] = held;
    if (p > 0 && held <= 0 && rank < need) w.fresh[rank] = p;
    found += total;
  }
  if (status == 0 && found < need) status = 1;
  __syncthreads();
  if (status == 0) {
    for (int r = tid; r < need; r += THREADS) refs_out[w.fresh[r]] = 1;
    for (int i = tid / 32; i < n; i += THREADS / 32) {      // a warp per request
      const int rank = w.rank[i];
      if (rank < 0) continue;
      const size_t at = static_cast<size_t>(list[i]) * max_pages;
      for (int j = tid & 31; j < max_pages; j += 32) {
        const int page = table[at + j];
        w.rows[static_cast<size_t>(i) * max_pages + j] = page;
        if (page > 0) atomicSub(&refs_out[page], 1);
      }
    }
  }
  if (tid == 0) {
    w.head[0] = status;
    *status_out = status;
  }
}

// Weights as unsigned numbers in their order; -0 is 0, and what is no number is below all.
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Tokens that a CTA moves: all of a thread's loads are in flight at once, eight at most.
constexpr int move_tokens(int d) { return d > 128 ? PAGE / 2 : PAGE; }

// Item (request, layer, head): CTA 1 + item; CTA 0 does the bookkeeping.
__global__ void __launch_bounds__(THREADS) select_kernel(
    const Cache cache, const int* table, const int* lens, const int* refs, int* refs_out,
    const int* list, int n, int slots, int max_pages, int keep, int first, int recent,
    const float* weights, int capacity, int* work, int items, int* status_out) {
  __shared__ int s_hist[BINS];
  __shared__ int s_warp[WARPS], s_pick[3];
  const Work w(work, slots, n, (keep + PAGE - 1) / PAGE, items, keep);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_wait();
  grid_release();
  if (blockIdx.x == 0) {
    make_plan(w, table, lens, refs, refs_out, list, n, slots, max_pages, cache.pages, keep, status_out);
    return;
  }
  const int item = blockIdx.x - 1, h = item % cache.kvh, layer = item / cache.kvh % cache.layers;
  const int slot = list[item / cache.kvh / cache.layers];
  if (slot < 0 || slot >= slots) return;
  const int len = lens[slot], lo = first, hi = len - recent;
  if (len <= keep || len > capacity) return;       // (the latter is found wrong by the bookkeeping)
  const size_t line = (static_cast<size_t>(layer) * slots + slot) * cache.kvh + h;
  const float* from = weights + line * capacity;

  // ---- the threshold: `want` keys of [lo, hi) stay; of those whose bits begin as `prefix` (the upper 32 -
  // shift ones), the first `want`, and all above
  uint32_t prefix = 0u;
  int shift = 32, want = keep - first - recent;
  const bool none = want == 0;
  for (int pass = 0; pass < 3 && !none; ++pass) {
    const int next = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = 1 << (shift - next);
    for (int i = tid; i < BINS; i += THREADS) s_hist[i] = 0;
    __syncthreads();
    constexpr int AHEAD = 8;                       // loads in flight
    auto count = [&](float x) {
      const uint32_t u = ordered(x);
      if (pass == 0 || u >> shift == prefix) atomicAdd(&s_hist[u >> next & (bins - 1)], 1);
    };
    int i0 = lo + tid;
    for (; i0 + (AHEAD - 1) * THREADS < hi; i0 += AHEAD * THREADS) {
      float x[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) x[k] = from[i0 + k * THREADS];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) count(x[k]);
    }
    if (i0 < hi) {
      float x[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (i0 + k * THREADS < hi) x[k] = from[i0 + k * THREADS];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (i0 + k * THREADS < hi) count(x[k]);
    }
    __syncthreads();
    // the bin in which the `want`-th from the top lies
    constexpr int PER = BINS / THREADS;
    int mine = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) mine += s_hist[tid * PER + k];
    int above = mine;                              // in this thread's bins and all above
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_down_sync(0xffffffffu, above, o);
      if (lane + o < 32) above += v;
    }
    if (lane == 0) s_warp[warp] = above;
    __syncthreads();
    for (int k = warp + 1; k < WARPS; ++k) above += s_warp[k];
    above -= mine;
    if (above < want && above + mine >= want) {
      int b = PER - 1;
      for (; b > 0 && above + s_hist[tid * PER + b] < want; --b) above += s_hist[tid * PER + b];
      s_pick[0] = tid * PER + b;
      s_pick[1] = want - above;
      s_pick[2] = s_hist[tid * PER + b];
    }
    __syncthreads();
    prefix = prefix << (shift - next) | static_cast<uint32_t>(s_pick[0]);
    want = s_pick[1];
    shift = next;
    const bool whole = s_pick[2] == want;          // all of the bin stay
    __syncthreads();
    if (whole) break;
  }

  // ---- the walk
  int2* stays = w.list + static_cast<size_t>(item) * keep;
  int done = 0, equal = 0;                         // keys kept so far; of them or not, equal to the threshold
  // a warp takes 256 neighbouring keys, a lane eight of them 32 apart, the next ones ahead
  float ahead[LANE_KEYS];
  auto load = [&](int k0) {
#pragma unroll
    for (int k = 0; k < LANE_KEYS; ++k) {
      const int key = k0 + warp * (32 * LANE_KEYS) + k * 32 + lane;
      ahead[k] = key < len ? from[key] : 0.f;
    }
  };
  load(0);
  for (int k0 = 0; k0 < len; k0 += BLOCK) {
    float x[LANE_KEYS];
    unsigned over[LANE_KEYS], same[LANE_KEYS];
    int n_over = 0, n_same = 0;
#pragma unroll
    for (int k = 0; k < LANE_KEYS; ++k) x[k] = ahead[k];
    load(k0 + BLOCK);
#pragma unroll
    for (int k = 0; k < LANE_KEYS; ++k) {
      const int key = k0 + warp * (32 * LANE_KEYS) + k * 32 + lane;
      const bool between = static_cast<unsigned>(key - lo) < static_cast<unsigned>(hi - lo);
      const uint32_t u = shift < 32 ? ordered(x[k]) >> shift : 0u;
      over[k] = __ballot_sync(0xffffffffu, key < len && (!between || (!none && u > prefix)));
      same[k] = __ballot_sync(0xffffffffu, between && !none && u == prefix);
      n_over += __popc(over[k]);
      if (same[k]) n_same += __popc(same[k]);      // (few have any)
    }
    __syncthreads();                               // (the counts of the step before are read)
    if (lane == 0) s_warp[warp] = n_over | n_same << 16;
    __syncthreads();
    int o_before = 0, s_before = equal, o_all = 0, s_all = 0;
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const int v = s_warp[k];
      if (k < warp) {
        o_before += v & 0xffff;
        s_before += v >> 16;
      }
      o_all += v & 0xffff;
      s_all += v >> 16;
    }
    // (of the equal ones before a key, at most `want` are kept)
    const int base = done - min(equal, want);
    const unsigned lower = (1u << lane) - 1u;
    int at = base + o_before + min(s_before, want);          // of the next key that stays
#pragma unroll
    for (int k = 0; k < LANE_KEYS; ++k) {
      unsigned stay = over[k];
      if (same[k]) {
        // of the warp's equal ones the first that are still wanted
        const bool mine = (same[k] >> lane & 1u) && s_before + __popc(same[k] & lower) < want;
        stay |= __ballot_sync(0xffffffffu, mine);
        s_before += __popc(same[k]);
      }
      if (stay >> lane & 1u)
        stays[at + __popc(stay & lower)] =
            make_int2(k0 + warp * (32 * LANE_KEYS) + k * 32 + lane, __float_as_int(x[k]));
      at += __popc(stay);
    }
    done = base + o_all + min(equal + s_all, want);
    equal += s_all;
  }
}

// D: channels of a head.  CTA (request, layer, part of a fresh page, head): neighbours write what lies side by
// side.  Those behind them write the table and the lengths.
template <int D>
__global__ void __launch_bounds__(MOVE_THREADS) move_kernel(
    const Cache cache, const int* table, int* table_out, const int* lens, int* lens_out,
    const int* list, int n, int slots, int max_pages, int keep, const float* weights, float* sums,
    int capacity, int* work, int items) {
  constexpr int G = D / 64, UNITS = 2 * D / 16;    // 16-byte units of a key and its value
  constexpr int TOKENS = move_tokens(D);           // of a CTA
  constexpr int EACH = TOKENS * UNITS / MOVE_THREADS;
  static_assert(2 * TOKENS <= MOVE_THREADS, "a thread has the scales of a key or a value");
  using Scales = std::conditional_t<G == 1, unsigned short, std::conditional_t<G == 2, uint32_t, uint2>>;
  __shared__ int s_list[TOKENS];                   // sources: places in the cache
  const int kept = (keep + PAGE - 1) / PAGE, parts = (keep + TOKENS - 1) / TOKENS;
  const Work w(work, slots, n, kept, items, keep);
  const int tid = threadIdx.x;
  grid_wait();
  grid_release();
  const long long moves = static_cast<long long>(items) * parts;
  if (static_cast<long long>(blockIdx.x) >= moves) {
    const long long total = static_cast<long long>(slots) * max_pages;
    const int status = w.head[0], ctas = gridDim.x - static_cast<int>(moves);
    for (long long i = (blockIdx.x - moves) * MOVE_THREADS + tid; i < total + slots;
         i += static_cast<long long>(ctas) * MOVE_THREADS) {
      const int s = static_cast<int>(i < total ? i / max_pages : i - total), who = w.named[s];
      const int rank = status == 0 && who < n ? w.rank[who] : -1;
      if (i < total) {
        const int j = static_cast<int>(i % max_pages);
        if (rank >= 0)
          table_out[i] = j < kept ? w.fresh[static_cast<size_t>(rank) * kept + j] : 0;
        else if (table_out != table)
          table_out[i] = table[i];
      } else if (rank >= 0) {
        lens_out[s] = keep;
      } else if (lens_out != lens) {
        lens_out[s] = lens[s];
      }
    }
    return;
  }
  const int h = blockIdx.x % cache.kvh, part = blockIdx.x / cache.kvh % parts;
  const int layer = blockIdx.x / cache.kvh / parts % cache.layers;
  const int who = blockIdx.x / cache.kvh / parts / cache.layers;
  const int item = (who * cache.layers + layer) * cache.kvh + h;
  const int t0 = part * TOKENS, count = min(TOKENS, keep - t0);
  // (what does not wait for one another is asked for together: a CTA is a chain of loads)
  const int status = w.head[0], slot = list[who], ranked = w.rank[who];
  int2 mine = make_int2(0, 0);
  if (tid < count) mine = w.list[static_cast<size_t>(item) * keep + t0 + tid];
  if (slot < 0 || slot >= slots) return;
  const size_t line = (static_cast<size_t>(layer) * slots + slot) * cache.kvh + h;
  const float* from = weights + line * capacity;
  float* to = sums + line * capacity;
  const int rank = status == 0 ? ranked : -1;
  if (rank < 0) {                                  // it stays as it is, or is named again
    if (to != from && (status != 0 || w.named[slot] == who))
      for (int i = part * MOVE_THREADS + tid; i < capacity; i += parts * MOVE_THREADS) to[i] = from[i];
    return;
  }
  if (tid < count) {
    s_list[tid] = w.rows[static_cast<size_t>(who) * max_pages + (mine.x >> 7)] * PAGE + (mine.x & 127);
    to[t0 + tid] = __int_as_float(mine.y);
  }
  const int page = w.fresh[static_cast<size_t>(rank) * kept + t0 / PAGE];
  const size_t target = (static_cast<size_t>(page) * PAGE + t0 % PAGE) * cache.kvh + h;
  for (int i = keep + part * MOVE_THREADS + tid; i < capacity; i += parts * MOVE_THREADS) to[i] = 0.f;
  int8_t* kc = reinterpret_cast<int8_t*>(cache.bases[layer]);
  int8_t* vc = reinterpret_cast<int8_t*>(cache.bases[cache.layers + layer]);
  Scales* scales = reinterpret_cast<Scales*>(cache.bases[(tid & 1 ? 3 : 2) * cache.layers + layer]);
  __syncthreads();
  // all of a thread's loads ahead of its stores
  uint4 v[EACH];
  Scales sc;
#pragma unroll
  for (int b = 0; b < EACH; ++b) {
    const int t = (b * MOVE_THREADS + tid) / UNITS, c = tid % UNITS;
    if (t < count)
      v[b] = *reinterpret_cast<const uint4*>((c < UNITS / 2 ? kc : vc) +
                                             (static_cast<size_t>(s_list[t]) * cache.kvh + h) * D +
                                             c % (UNITS / 2) * 16);
  }
  if (tid >> 1 < count) sc = scales[static_cast<size_t>(s_list[tid >> 1]) * cache.kvh + h];
#pragma unroll
  for (int b = 0; b < EACH; ++b) {
    const int t = (b * MOVE_THREADS + tid) / UNITS, c = tid % UNITS;
    if (t < count)
      *reinterpret_cast<uint4*>((c < UNITS / 2 ? kc : vc) +
                                (target + static_cast<size_t>(t) * cache.kvh) * D +
                                c % (UNITS / 2) * 16) = v[b];
  }
  if (tid >> 1 < count) scales[target + static_cast<size_t>(tid >> 1) * cache.kvh] = sc;
}

}  // namespace ev
}  // namespace orinfer

using namespace orinfer;

extern "C" size_t orinfer_evict_work_words(int layers, int kvh, int slots, int n, int max_pages, int keep) {
  const size_t kept = (static_cast<size_t>(keep) + ev::PAGE - 1) / ev::PAGE;
  return ev::WORK_HEAD + 2 * static_cast<size_t>(n) * layers * kvh * keep + slots + 2 * static_cast<size_t>(n) +
         n * (kept + max_pages);
}

extern "C" int orinfer_evict_keys(const long long* bases, int layers, int kvh, int head_dim, int pages,
                                  const int* table, int* table_out, const int* lens, int* lens_out,
                                  const int* refs, int* refs_out, const int* list, int n, int slots,
                                  int max_pages, int keep, int first, int recent,
                                  const float* weights, float* sums, int capacity, int* work,
                                  int* status_out, cudaStream_t stream) {
  if (layers <= 0 || kvh <= 0 || pages <= 0 || n < 0 || slots <= 0 || max_pages <= 0) return -1;
  if (keep < 1 || first < 0 || recent < 0 || static_cast<long long>(first) + recent > keep) return -1;
  if (keep > max_pages * static_cast<long long>(ev::PAGE) ||
      capacity < max_pages * static_cast<long long>(ev::PAGE))
    return -1;
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return -1;
  if ((reinterpret_cast<uintptr_t>(work) & 7) != 0) return -1;
  const int kept = (keep + ev::PAGE - 1) / ev::PAGE;
  const long long items = static_cast<long long>(n) * layers * kvh;
  if (items * kept > (1 << 29) || static_cast<long long>(slots) * (max_pages + 1LL) > (1 << 30) ||
      static_cast<long long>(pages) * ev::PAGE > 0x7fffffffLL)
    return -1;
  const ev::Cache cache{bases, layers, kvh, pages};
  launch_early(ev::select_kernel, dim3(1 + static_cast<unsigned>(items)), ev::THREADS, 0, stream, cache, table,
               lens, refs, refs_out, list, n, slots, max_pages, keep, first, recent, weights, capacity, work,
               static_cast<int>(items), status_out);
  if (const cudaError_t e = cudaGetLastError()) return static_cast<int>(e);
  const int more = (slots * max_pages + slots + 4 * ev::MOVE_THREADS - 1) / (4 * ev::MOVE_THREADS);
  const int tokens = ev::move_tokens(head_dim), parts = (keep + tokens - 1) / tokens;
  const dim3 grid(static_cast<unsigned>(items * parts + more));
#define CASE(D)                                                                                   \
  if (head_dim == D)                                                                              \
    launch_early(ev::move_kernel<D>, grid, ev::MOVE_THREADS, 0, stream, cache, table, table_out, lens, \
                 lens_out, list, n, slots, max_pages, keep, weights, sums, capacity, work,        \
                 static_cast<int>(items));
  CASE(64) CASE(128) CASE(256)
#undef CASE
  return static_cast<int>(cudaGetLastError());
}
