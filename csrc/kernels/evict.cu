// Eviction from the paged cache: of a request that has outgrown its bound each layer and KV head keeps
// the keys that attention has given the most weight, beside the first and the last ones.
//
// The page table is one for all layers and heads, but which keys a page holds is a head's own matter: a
// request keeps as many keys in each, in their order, and attention goes on as over a shorter context
// (keys carry their rotary angle).  What is kept goes to fresh pages and the old ones lose a reference,
// so pages that others share are never written, the move needs no order, and a call repeats.
//
// One CTA does the bookkeeping of the pages (the lowest free ones, in the order of the requests).  Then a
// CTA per request, layer and KV head finds its threshold, the weight of the last key that stays, by
// three histograms of the weights' bits (11, 11, 10) and walks the keys once: those above the
// threshold, and of those equal to it the first so many, are copied as they are found.
#include "api.h"
#include "common.cuh"

namespace orinfer {
namespace ev {

constexpr int PAGE = 128;                          // tokens
constexpr int PLAN_THREADS = 1024;
constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int BLOCK = 4 * THREADS;                 // keys of a step of the walk
constexpr int BINS = 2048;                         // of a histogram
constexpr int WORK_HEAD = 4;                       // status, -, -, -

// What the bookkeeping leaves: the first naming of a slot [slots]; per request its tokens [n], its rank
// among those that are cut (-1: it stays as it is) [n]; fresh pages [n][pages of `keep`]; the table
// rows as they were [n][max_pages].
struct Work {
  int *head, *named, *len, *rank, *fresh, *rows;
  __host__ __device__ Work(int* w, int slots, int n, int kept)
      : head(w), named(w + WORK_HEAD), len(named + slots), rank(len + n), fresh(rank + n),
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

__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(
    const int* table, int* table_out, const int* lens, int* lens_out, const int* refs,
    int* refs_out, const int* list, int n, int slots, int max_pages, int pages, int keep,
    int* work, int* status_out) {
  __shared__ int sums[PLAN_THREADS / 32];
  __shared__ int s_wrong;
  const int kept = (keep + PAGE - 1) / PAGE, tid = threadIdx.x;
  const Work w(work, slots, n, kept);
  grid_wait();
  grid_release();
  if (tid == 0) s_wrong = 0;
  for (int s = tid; s < slots; s += PLAN_THREADS) w.named[s] = n;
  __syncthreads();
  for (int i = tid; i < n; i += PLAN_THREADS) {
    const int s = list[i];
    if (s >= 0 && s < slots)
      atomicMin(&w.named[s], i);
    else
      s_wrong = 1;
  }
  __syncthreads();
  // ---- requests: lengths that fit the table, pages that somebody holds
  for (int i = tid / 16; i < n; i += PLAN_THREADS / 16) {        // sixteen lanes per request
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
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + tid;
    const bool mine = i < n && status == 0 && w.len[i] > keep;
    int total;
    const int rank = cut + block_rank(mine, sums, total);
    if (i < n) w.rank[i] = mine ? rank : -1;
    cut += total;
  }
  // ---- the free pages in ascending order are theirs
  const long long need = static_cast<long long>(cut) * kept;
  int found = 0;
  for (int p0 = 0; p0 < pages; p0 += PLAN_THREADS) {
    const int p = p0 + tid;
    const int held = p < pages ? refs[p] : 1;
    int total;
    const int rank = found + block_rank(p > 0 && held <= 0, sums, total);
    if (p < pages && refs_out != refs) refs_out[p] = held;
    if (p > 0 && held <= 0 && rank < need) w.fresh[rank] = p;
    found += total;
  }
  if (status == 0 && found < need) status = 1;
  if (lens_out != lens)
    for (int s = tid; s < slots; s += PLAN_THREADS) lens_out[s] = lens[s];
  __syncthreads();
  if (status == 0) {
    for (int r = tid; r < need; r += PLAN_THREADS) refs_out[w.fresh[r]] = 1;
    for (int i = tid / 32; i < n; i += PLAN_THREADS / 32) {      // a warp per request
      const int rank = w.rank[i];
      if (rank < 0) continue;
      const size_t at = static_cast<size_t>(list[i]) * max_pages;
      for (int j = tid & 31; j < max_pages; j += 32) {
        const int page = table[at + j];
        w.rows[static_cast<size_t>(i) * max_pages + j] = page;
        if (page > 0) atomicSub(&refs_out[page], 1);
        if (table_out == table)
          table_out[at + j] = j < kept ? w.fresh[static_cast<size_t>(rank) * kept + j] : 0;
      }
      if ((tid & 31) == 0) lens_out[list[i]] = keep;
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

// D: channels of a head.  Item (request, layer, head); the CTAs behind the items write the table where
// it is not changed in place.
template <int D>
__global__ void __launch_bounds__(THREADS) move_kernel(
    const Cache cache, const int* table, int* table_out, const int* list, int n, int slots,
    int max_pages, int keep, int first, int recent, const float* weights, float* sums,
    int capacity, int* work, int items) {
  constexpr int G = D / 64, UNITS = 2 * D / 16;    // 16-byte units of a key and its value
  __shared__ int s_hist[BINS];
  __shared__ int s_warp[WARPS], s_pick[3];
  __shared__ int s_from[BLOCK], s_to[BLOCK];       // places of the tokens to be copied
  const int kept = (keep + PAGE - 1) / PAGE;
  const Work w(work, slots, n, kept);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  grid_wait();
  grid_release();
  const int status = w.head[0];
  if (static_cast<int>(blockIdx.x) >= items) {
    const int total = slots * max_pages;
    for (int i = (blockIdx.x - items) * THREADS + tid; i < total;
         i += (gridDim.x - items) * THREADS) {
      const int s = i / max_pages, j = i % max_pages, who = w.named[s];
      const int rank = status == 0 && who < n ? w.rank[who] : -1;
      table_out[i] = rank < 0 ? table[i]
                     : j < kept ? w.fresh[static_cast<size_t>(rank) * kept + j] : 0;
    }
    return;
  }
  const int h = blockIdx.x % cache.kvh, layer = blockIdx.x / cache.kvh % cache.layers;
  const int who = blockIdx.x / cache.kvh / cache.layers;
  const int slot = list[who];
  if (slot < 0 || slot >= slots || w.named[slot] != who) return;
  const size_t line = (static_cast<size_t>(layer) * slots + slot) * cache.kvh + h;
  const float* from = weights + line * capacity;
  float* to = sums + line * capacity;
  const int rank = status == 0 ? w.rank[who] : -1;
  if (rank < 0) {                                  // it stays as it is
    if (to != from)
      for (int i = tid; i < capacity; i += THREADS) to[i] = from[i];
    return;
  }
  const int len = w.len[who], lo = first, hi = len - recent;

  // ---- the threshold: `want` keys of [lo, hi) stay; of those whose bits begin as `prefix` (the upper 32 -
  // shift ones), the first `want`, and all above
  uint32_t prefix = 0u;
  int shift = 32, want = keep - first - recent;
  const bool none = want == 0;
  for (int pass = 0; pass < 3 && !none; ++pass) {
    const int next = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = 1 << (shift - next);
    for (int i = tid; i < BINS; i += THREADS) s_hist[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += THREADS) {
      const uint32_t u = ordered(from[i]);
      if (pass == 0 || u >> shift == prefix) atomicAdd(&s_hist[u >> next & (bins - 1)], 1);
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
  const int8_t* kc = reinterpret_cast<const int8_t*>(cache.bases[layer]);
  const int8_t* vc = reinterpret_cast<const int8_t*>(cache.bases[cache.layers + layer]);
  const __half* ks = reinterpret_cast<const __half*>(cache.bases[2 * cache.layers + layer]);
  const __half* vs = reinterpret_cast<const __half*>(cache.bases[3 * cache.layers + layer]);
  const int* pages = w.rows + static_cast<size_t>(who) * max_pages;
  const int* fresh = w.fresh + static_cast<size_t>(rank) * kept;
  const size_t token = static_cast<size_t>(cache.kvh) * D;
  int done = 0, equal = 0;                         // keys kept so far; of them or not, equal to the threshold
  for (int k0 = 0; k0 < len; k0 += BLOCK) {
    // a warp takes 128 neighbouring keys, a lane four of them 32 apart
    float x[4];
    unsigned over[4], same[4];
    int n_over = 0, n_same = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int key = k0 + warp * 128 + k * 32 + lane;
      x[k] = key < len ? from[key] : 0.f;
      const bool between = key >= lo && key < hi;
      const uint32_t u = shift < 32 ? ordered(x[k]) >> shift : 0u;
      over[k] = __ballot_sync(0xffffffffu, key < len && (!between || (!none && u > prefix)));
      same[k] = __ballot_sync(0xffffffffu, between && !none && u == prefix);
      n_over += __popc(over[k]);
      n_same += __popc(same[k]);
    }
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
    const int base = min(equal, want);
    const unsigned lower = (1u << lane) - 1u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int eq = s_before + __popc(same[k] & lower);
      const bool stays = (over[k] >> lane & 1u) || ((same[k] >> lane & 1u) && eq < want);
      const int at = o_before + __popc(over[k] & lower) + min(eq, want) - base;
      if (stays) {
        const int key = k0 + warp * 128 + k * 32 + lane, out = done + at;
        s_from[at] = pages[key >> 7] * PAGE + (key & 127);
        s_to[at] = fresh[out >> 7] * PAGE + (out & 127);
        to[out] = x[k];
      }
      o_before += __popc(over[k]);
      s_before += __popc(same[k]);
    }
    const int count = o_all + min(equal + s_all, want) - base;
    equal += s_all;
    __syncthreads();
    // ---- copies
    constexpr int BATCH = 4;
    for (int u0 = tid; u0 < count * UNITS; u0 += BATCH * THREADS) {
      uint4 v[BATCH];
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int u = u0 + b * THREADS, t = u / UNITS, c = u % UNITS;
        if (t < count) {
          const int8_t* p = c < UNITS / 2 ? kc : vc;
          v[b] = *reinterpret_cast<const uint4*>(p + s_from[t] * token + h * D + c % (UNITS / 2) * 16);
        }
      }
#pragma unroll
      for (int b = 0; b < BATCH; ++b) {
        const int u = u0 + b * THREADS, t = u / UNITS, c = u % UNITS;
        if (t < count) {
          int8_t* p = const_cast<int8_t*>(c < UNITS / 2 ? kc : vc);
          *reinterpret_cast<uint4*>(p + s_to[t] * token + h * D + c % (UNITS / 2) * 16) = v[b];
        }
      }
    }
    for (int u = tid; u < count * 2 * G; u += THREADS) {
      const int t = u / (2 * G), c = u % (2 * G);
      const unsigned short* p = reinterpret_cast<const unsigned short*>(c < G ? ks : vs);
      unsigned short* o = const_cast<unsigned short*>(p);
      o[(static_cast<size_t>(s_to[t]) * cache.kvh + h) * G + c % G] =
          p[(static_cast<size_t>(s_from[t]) * cache.kvh + h) * G + c % G];
    }
    done += count;
    __syncthreads();                               // (the lists are used)
  }
  for (int i = keep + tid; i < capacity; i += THREADS) to[i] = 0.f;
}

template <int D>
static void launch_move(int blocks, int items, cudaStream_t stream, const Cache& cache, const int* table,
                        int* table_out, const int* list, int n, int slots, int max_pages, int keep,
                        int first, int recent, const float* weights, float* sums, int capacity,
                        int* work) {
  launch_early(move_kernel<D>, dim3(blocks), THREADS, 0, stream, cache, table, table_out, list, n,
               slots, max_pages, keep, first, recent, weights, sums, capacity, work, items);
}

}  // namespace ev
}  // namespace orinfer

using namespace orinfer;

extern "C" size_t orinfer_evict_work_words(int slots, int n, int max_pages, int keep) {
  const size_t kept = (static_cast<size_t>(keep) + ev::PAGE - 1) / ev::PAGE;
  return ev::WORK_HEAD + slots + 2 * static_cast<size_t>(n) + n * (kept + max_pages);
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
  if (static_cast<long long>(n) * layers * kvh > (1 << 30) ||
      static_cast<long long>(slots) * max_pages > (1 << 30) ||
      static_cast<long long>(pages) * ev::PAGE > 0x7fffffffLL)
    return -1;
  launch_early(ev::plan_kernel, dim3(1), ev::PLAN_THREADS, 0, stream, table, table_out, lens,
               lens_out, refs, refs_out, list, n, slots, max_pages, pages, keep, work, status_out);
  if (const cudaError_t e = cudaGetLastError()) return static_cast<int>(e);
  const ev::Cache cache{bases, layers, kvh, pages};
  const int items = n * layers * kvh;
  const int more = table_out == table ? 0 : (slots * max_pages + 4 * ev::THREADS - 1) / (4 * ev::THREADS);
  if (items + more == 0) return 0;
#define CASE(D)                                                                                    \
  if (head_dim == D)                                                                               \
    ev::launch_move<D>(items + more, items, stream, cache, table, table_out, list, n, slots, max_pages, \
                       keep, first, recent, weights, sums, capacity, work);
  CASE(64) CASE(128) CASE(256)
#undef CASE
  return static_cast<int>(cudaGetLastError());
}
