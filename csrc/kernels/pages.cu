// Pages of the cache: copying, forking, freeing and compacting.
//
// A cache is a list of tensors (keys, values and scales of every layer), each [pages, 128, ...]
// contiguous, so that a token is `token_bytes` of a tensor and a page 128 times that.  Beside it
// stand the page table int32 [slots, max_pages], the tokens of every slot (lens) and the references
// of every page (refs).  Page 0 is nobody's.
//
// The bookkeeping is one CTA's work (a few scans over the pages).  It leaves a list of (source
// page, target page, tokens), and a second kernel moves those bytes of all tensors and writes the
// table.  Outputs may be the inputs themselves.
//
// A copy is bound by memory: 8 requests of up to 1500 tokens, eight branches each, in 36 layers of 8 KV
// heads of 128 take 73 us (340 MB written, an eighth of it read, at 5.9 TB/s behind 8 us of
// bookkeeping), 64 of 256 pages moved within the cache 206 (1.24 GB at 6.1).  Small calls are launches:
// a fork of one request into four 6.4, a compaction of a few pages 4.2, a freed slot 2.4.
#include "api.h"
#include "common.cuh"

namespace orinfer {
namespace pg {

constexpr int PAGE = 128;                          // tokens
constexpr int PLAN_THREADS = 1024;
constexpr int COPY_THREADS = 256;
constexpr int WORK_HEAD = 4;                       // status, copies, -, -

// The cache: tensors' addresses and bytes per token, and a page's units (tensor, first token,
// tokens).
struct Cache {
  const long long* bases;
  const int* token_bytes;
  const int* units;
  int n_units, pages;
};

// Rank of `flag` among the CTA's set flags, in the order of the threads, and their number.
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

// ---------------------------------------------------------------- fork
// work: head; copies [n][3]; pairs in the order of their new pages [n]; pair of a child slot [slots];
// a pair of a parent slot [slots]; from there the next one of the same parent [n]; these first pairs [n]
__global__ void __launch_bounds__(PLAN_THREADS) fork_plan_kernel(
    const int* table, const int* lens, const int* refs, int* refs_out, const int* parents,
    const int* children, int n, int slots, int max_pages, int pages, int apart, int* work,
    int* status_out) {
  __shared__ int sums[PLAN_THREADS / 32];
  __shared__ int s_wrong, s_firsts;
  int* copies = work + WORK_HEAD;
  int* owner = copies + 3 * n;
  int* child_of = owner + n;
  int* pair_of = child_of + slots;
  int* chain = pair_of + slots;
  int* firsts = chain + n;
  const int tid = threadIdx.x;
  grid_wait();
  grid_release();
  if (tid == 0) s_wrong = s_firsts = 0;
  for (int s = tid; s < slots; s += PLAN_THREADS) child_of[s] = pair_of[s] = -1;
  __syncthreads();
  // ---- the pairs: slots that exist, a child that is empty and named once, pages that are held
  for (int i = tid / 16; i < n; i += PLAN_THREADS / 16) {        // sixteen lanes per pair
    const int p = parents[i], c = children[i], lane = tid & 15;
    bool wrong = p < 0 || p >= slots || c < 0 || c >= slots || p == c;
    if (!wrong) {
      const int len = lens[p];
      wrong = lens[c] != 0 || len < 0 || len > max_pages * PAGE;
      if (!wrong && lane == 0) wrong = atomicCAS(&child_of[c], -1, i) != -1;
      const int* row = table + static_cast<size_t>(p) * max_pages;
      for (int j = lane; !wrong && j < (len + PAGE - 1) / PAGE; j += 16) {
        const int page = row[j];
        wrong = page <= 0 || page >= pages || refs[page] <= 0;
      }
    }
    if (wrong) s_wrong = 1;
  }
  __syncthreads();
  const bool named = s_wrong == 0;                 // every slot is one: nobody is child and parent
  __syncthreads();
  if (named)
    for (int i = tid; i < n; i += PLAN_THREADS)
      if (child_of[parents[i]] != -1) s_wrong = 1;
  __syncthreads();
  int status = s_wrong ? 2 : 0;
  // ---- which pairs need a page
  int need = 0;
  for (int i0 = 0; i0 < n && status == 0; i0 += PLAN_THREADS) {
    const int i = i0 + tid;
    const int p = i < n ? parents[i] : 0, tail = i < n ? lens[p] % PAGE : 0;
    int total;
    const int rank = need + block_rank(tail != 0, sums, total);
    if (i < n) {
      copies[3 * i] = tail ? table[static_cast<size_t>(p) * max_pages + lens[p] / PAGE] : 0;
      copies[3 * i + 1] = 0;
      copies[3 * i + 2] = tail;
      if (tail) {
        owner[rank] = i;
        if (!apart) chain[i] = atomicExch(&pair_of[p], i);
      }
    }
    need += total;
  }
  __syncthreads();
  // ---- the free pages in ascending order are theirs
  int found = 0;
  for (int p0 = 0; p0 < pages; p0 += PLAN_THREADS) {
    const int p = p0 + tid;
    const int held = p < pages ? refs[p] : 1;
    int total;
    const int rank = found + block_rank(p > 0 && held <= 0, sums, total);
    if (p < pages && refs_out != refs) refs_out[p] = held;
    if (p > 0 && held <= 0 && rank < need) copies[3 * owner[rank] + 1] = p;
    found += total;
  }
  if (status == 0 && found < need) status = 1;
  if (status == 0 && !apart)
    for (int i = tid; i < n; i += PLAN_THREADS)
      if (copies[3 * i + 2] > 0 && pair_of[parents[i]] == i)
        firsts[atomicAdd(&s_firsts, 1)] = i;
  __syncthreads();
  if (status == 0)
    for (int r = tid; r < need; r += PLAN_THREADS) refs_out[copies[3 * owner[r] + 1]] = 1;
  if (tid == 0) {
    work[0] = status;
    work[1] = status != 0 ? 0 : apart ? n : s_firsts;
    *status_out = status;
  }
}

// ---------------------------------------------------------------- copies
// Four loads of a thread ahead of their stores (one at a time, 128 pages of 9.7 MB moved at 5.7 TB/s).
// `next` names the targets in turn: what several children get is read once.
template <class T, class Next>
__device__ __forceinline__ void copy_as(const unsigned char* from, int bytes, Next next) {
  constexpr int BATCH = 4;
  const int n = bytes / static_cast<int>(sizeof(T));
  const T* src = reinterpret_cast<const T*>(from);
  for (int i0 = threadIdx.x; i0 < n; i0 += BATCH * COPY_THREADS) {
    T v[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
      if (i0 + k * COPY_THREADS < n) v[k] = __ldcs(src + i0 + k * COPY_THREADS);
    int at = -1;
    while (unsigned char* to = next(at)) {
      T* dst = reinterpret_cast<T*>(to);
#pragma unroll
      for (int k = 0; k < BATCH; ++k)
        if (i0 + k * COPY_THREADS < n) __stcs(dst + i0 + k * COPY_THREADS, v[k]);
    }
  }
  const int rest = n * static_cast<int>(sizeof(T));
  if (rest + static_cast<int>(threadIdx.x) < bytes) {
    int at = -1;
    while (unsigned char* to = next(at)) to[rest + threadIdx.x] = from[rest + threadIdx.x];
  }
}

// copies [][3]: source page, target page, tokens from the page's first on; *count of them, or where
// there are `firsts` as many of those, each with the copies of the same source that `chain` leads to.
// By CTA `cta` of `ctas`.
__device__ __forceinline__ void copy_units(const Cache& cache, const int* copies, const int* count,
                                           int cta, int ctas, int* status,
                                           const int* firsts = nullptr, const int* chain = nullptr) {
  const long long total = static_cast<long long>(*count) * cache.n_units;
  for (long long w = cta; w < total; w += ctas) {
    const long long item = w / cache.n_units;
    const long long first = firsts ? firsts[item] : item;
    const int* c = copies + 3 * first;
    const int* u = cache.units + w % cache.n_units * 3;
    const int from = c[0], tokens = min(c[2] - u[1], u[2]);
    if (tokens <= 0) continue;
    if (from < 0 || from >= cache.pages || c[1] < 0 || c[1] >= cache.pages || c[2] > PAGE) {
      if (threadIdx.x == 0) report_status(status, STATUS_BAD_INDEX, 0x40);
      continue;
    }
    const long long per = cache.token_bytes[u[0]];
    unsigned char* base = reinterpret_cast<unsigned char*>(cache.bases[u[0]]) + u[1] * per;
    const unsigned char* src = base + from * PAGE * per;
    const int bytes = tokens * static_cast<int>(per);
    // (pages are multiples of 128 bytes: all targets are aligned as the source is)
    auto next = [&](int& at) -> unsigned char* {
      at = at < 0 ? static_cast<int>(first) : chain ? chain[at] : -1;
      if (at < 0) return nullptr;
      return base + static_cast<long long>(copies[3 * static_cast<long long>(at) + 1]) * PAGE * per;
    };
    const uintptr_t off = reinterpret_cast<uintptr_t>(src);
    if ((off & 15) == 0)
      copy_as<uint4>(src, bytes, next);
    else if ((off & 3) == 0)
      copy_as<uint32_t>(src, bytes, next);
    else
      copy_as<unsigned char>(src, bytes, next);
  }
}

__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(const Cache cache,
                                                                  const int* copies,
                                                                  const int* count, int* status) {
  grid_wait();
  grid_release();
  copy_units(cache, copies, count, blockIdx.x, gridDim.x, status);
}

// The table's rows, lens and the references of shared pages, a CTA per slot; the CTAs behind them copy.
__global__ void __launch_bounds__(COPY_THREADS) fork_apply_kernel(
    const int* table, int* table_out, const int* lens, int* lens_out, int* refs_out,
    const int* parents, int n, int slots, int max_pages, int apart, const int* work,
    const Cache cache, int* status) {
  grid_wait();
  grid_release();
  const int* copies = work + WORK_HEAD;
  if (static_cast<int>(blockIdx.x) >= slots) {
    const int* chain = copies + 4 * n + 2 * slots;
    copy_units(cache, copies, work + 1, blockIdx.x - slots, gridDim.x - slots, status,
               apart ? nullptr : chain + n, apart ? nullptr : chain);
    return;
  }
  const int s = blockIdx.x, pair = work[0] == 0 ? (copies + 4 * n)[s] : -1;
  const int from = pair < 0 ? s : parents[pair];
  const int len = lens[from], full = len / PAGE;
  const int* row = table + static_cast<size_t>(from) * max_pages;
  int* row_out = table_out + static_cast<size_t>(s) * max_pages;
  if (pair < 0) {
    if (table_out != table)
      for (int j = threadIdx.x; j < max_pages; j += blockDim.x) row_out[j] = row[j];
  } else {
    for (int j = threadIdx.x; j < max_pages; j += blockDim.x) {
      int page = 0;
      if (j < full) {
        page = row[j];
        atomicAdd(&refs_out[page], 1);
      } else if (j == full && len % PAGE) {
        page = copies[3 * pair + 1];
      }
      row_out[j] = page;
    }
  }
  if (threadIdx.x == 0 && (pair >= 0 || lens_out != lens)) lens_out[s] = len;
}

// ---------------------------------------------------------------- free
// CTAs [0, slots): the rows; the CTAs behind them: the references of RANGE pages each, less what the
// listed slots hold of them.  `parts`: 1 rows, 2 references, both where no row is read and written.
constexpr int RANGE = 2048;
constexpr int ROWS = 1, REFS = 2;
constexpr int FREE_THREADS = 512;
constexpr int FREE_MOST = 1 << 17;                 // slots and entries whose bits fit beside the counts

__global__ void __launch_bounds__(FREE_THREADS) free_kernel(const int* table, int* table_out, const int* lens,
                                                   int* lens_out, const int* refs, int* refs_out,
                                                   const int* gone, int n, int slots, int max_pages,
                                                   int pages, int parts, int* status) {
  extern __shared__ int marks[];                   // a bit per slot: listed, and not yet claimed
  int* claims = marks + (slots + 31) / 32;         // a bit per entry: it is its slot's first
  __shared__ int held[RANGE];
  grid_wait();
  grid_release();
  const int row_ctas = parts & ROWS ? slots : 0;
  if (static_cast<int>(blockIdx.x) < row_ctas) {
    const int s = blockIdx.x;
    bool listed = false;
    for (int i = threadIdx.x; i < n; i += blockDim.x) listed = listed || gone[i] == s;
    listed = __syncthreads_or(listed);
    if (!listed && table == table_out && lens == lens_out) return;
    const size_t row = static_cast<size_t>(s) * max_pages;
    for (int j = threadIdx.x; j < max_pages; j += blockDim.x)
      table_out[row + j] = listed ? 0 : table[row + j];
    if (threadIdx.x == 0) lens_out[s] = listed ? 0 : lens[s];
    return;
  }
  const int first = (blockIdx.x - row_ctas) * RANGE;
  const bool reports = first == 0;
  for (int i = threadIdx.x; i < (slots + 31) / 32 + (n + 31) / 32; i += FREE_THREADS) marks[i] = 0;
  for (int i = threadIdx.x; i < RANGE; i += FREE_THREADS) held[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += FREE_THREADS) {
    const int s = gone[i];
    if (s >= 0 && s < slots)
      atomicOr(&marks[s >> 5], 1 << (s & 31));
    else if (reports)
      report_status(status, STATUS_BAD_INDEX, 0x41);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += FREE_THREADS) {
    const int s = gone[i];
    if (s >= 0 && s < slots && atomicAnd(&marks[s >> 5], ~(1 << (s & 31))) >> (s & 31) & 1)
      atomicOr(&claims[i >> 5], 1 << (i & 31));
  }
  __syncthreads();
  const unsigned cells = static_cast<unsigned>(n) * max_pages;
  for (unsigned c0 = threadIdx.x; c0 < cells; c0 += 4 * FREE_THREADS) {
    int page[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const unsigned c = c0 + k * FREE_THREADS, i = c / max_pages;
      page[k] = c < cells && claims[i >> 5] >> (i & 31) & 1
                    ? table[static_cast<size_t>(gone[i]) * max_pages + (c - i * max_pages)]
                    : 0;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (page[k] < 0 || page[k] >= pages) {
        if (reports) report_status(status, STATUS_BAD_INDEX, 0x42);
      } else if (page[k] > 0 && page[k] >= first && page[k] < first + RANGE) {
        atomicAdd(&held[page[k] - first], 1);
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < RANGE && first + i < pages; i += FREE_THREADS) {
    const int left = refs[first + i] - held[i];
    if (held[i] > 0 && left < 0) report_status(status, STATUS_BAD_INDEX, 0x43);   // held less often
    if (held[i] > 0 || refs_out != refs) refs_out[first + i] = held[i] > 0 ? max(left, 0) : left;
  }
}

// ---------------------------------------------------------------- compact
// work: head; copies [pages / 2][3].  With L pages in use, the k-th of them above L goes to the k-th
// free page of 1..L.
__global__ void __launch_bounds__(PLAN_THREADS) compact_plan_kernel(const int* refs, int* refs_out,
                                                                    int* moved, int pages,
                                                                    int* work) {
  __shared__ int sums[PLAN_THREADS / 32];
  int* copies = work + WORK_HEAD;
  const int tid = threadIdx.x;
  grid_wait();
  grid_release();
  int live = 0;
  for (int p0 = 0; p0 < pages; p0 += PLAN_THREADS) {
    const int p = p0 + tid;
    int total;
    block_rank(p > 0 && p < pages && refs[p] > 0, sums, total);
    live += total;
  }
  int holes = 0, tops = 0;
  for (int p0 = 0; p0 < pages; p0 += PLAN_THREADS) {
    const int p = p0 + tid;
    const int held = p > 0 && p < pages ? max(refs[p], 0) : 0;
    const bool hole = p > 0 && p <= live && held == 0, top = p > live && held > 0;
    int more_holes, more_tops;
    const int h = holes + block_rank(hole, sums, more_holes);
    const int t = tops + block_rank(top, sums, more_tops);
    if (hole) copies[3 * h + 1] = p;
    if (top) {
      copies[3 * t] = p;
      copies[3 * t + 2] = PAGE;
    }
    if (p < pages) {
      moved[p] = p;
      refs_out[p] = held;
    }
    holes += more_holes;
    tops += more_tops;
  }
  __syncthreads();
  for (int k = tid; k < tops; k += PLAN_THREADS) {
    const int from = copies[3 * k], to = copies[3 * k + 1];
    moved[from] = to;
    refs_out[to] = refs_out[from];
    refs_out[from] = 0;
  }
  if (tid == 0) {
    work[0] = 0;
    work[1] = tops;
  }
}

// CTAs [0, remap_ctas) write the table, those behind them copy.
__global__ void __launch_bounds__(COPY_THREADS) compact_apply_kernel(
    const int* table, int* table_out, long long n, const int* moved, int pages, int remap_ctas,
    const int* work, const Cache cache, int* status) {
  grid_wait();
  grid_release();
  if (static_cast<int>(blockIdx.x) >= remap_ctas) {
    copy_units(cache, work + WORK_HEAD, work + 1, blockIdx.x - remap_ctas, gridDim.x - remap_ctas,
               status);
    return;
  }
  const long long step = static_cast<long long>(remap_ctas) * COPY_THREADS;
  for (long long i = static_cast<long long>(blockIdx.x) * COPY_THREADS + threadIdx.x; i < n; i += step) {
    const int page = table[i];
    const bool known = page >= 0 && page < pages;
    if (!known) report_status(status, STATUS_BAD_INDEX, 0x44);
    table_out[i] = known ? moved[page] : page;
  }
}

// CTAs that copy at most `most` pages: four times as many as there is room for, so that one that ends
// early makes room for the next (8 per SM: 8 parents with eight children each 80 us, 64 pages moved 228;
// 32: 73 and 206; 64: 73 and 204, and a CTA without work costs its start).
static int copy_ctas(const Cache& cache, int most) {
  const long long units = static_cast<long long>(most) * cache.n_units;
  return static_cast<int>(units < 32 * 148 ? units : 32 * 148);
}

static int grid_of(long long n) {
  const long long g = (n + COPY_THREADS - 1) / COPY_THREADS;
  return static_cast<int>(g < 592 ? g : 592);
}

}  // namespace pg
}  // namespace orinfer

using namespace orinfer;

// copies: int32 [*count, 3] on the device, at most `most` of them
extern "C" int orinfer_copy_pages(const long long* bases, const int* token_bytes, const int* units,
                                  int n_units, int pages, const int* copies, const int* count,
                                  int most, cudaStream_t stream) {
  if (most <= 0 || n_units <= 0) return most < 0 || n_units < 0 ? -1 : 0;
  if (!bases || !token_bytes || !units || !copies || !count || pages <= 0) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  const pg::Cache cache = {bases, token_bytes, units, n_units, pages};
  launch_early(pg::copy_pages_kernel, dim3(pg::copy_ctas(cache, most)), pg::COPY_THREADS, 0, stream,
               cache, copies, count, runtime_status_ptr());
  return static_cast<int>(cudaGetLastError());
}

// status: 0, 1 (not enough free pages) or 2 (a pair that cannot be); then nothing is changed.
// work: int32 [4 + 6 n + 2 slots].
extern "C" int orinfer_fork_pages(const long long* bases, const int* token_bytes, const int* units,
                                  int n_units, int pages, const int* table, int* table_out,
                                  const int* lens, int* lens_out, const int* refs, int* refs_out,
                                  const int* parents, const int* children, int n, int slots,
                                  int max_pages, int* work, int* status, cudaStream_t stream) {
  if (n < 0 || slots <= 0 || max_pages <= 0 || pages <= 0 || n_units < 0) return -1;
  if (max_pages > (1 << 24) || !work || !status) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  // Children of one parent get its page from one read (8 parents with eight each 110 -> 79 us), but by
  // CTAs of their own where all fit at once (a fork into four 7.3 -> 6.4).
  const pg::Cache cache = {bases, token_bytes, units, n_units, pages};
  const int apart = static_cast<long long>(n) * n_units <= 8 * 148;
  launch_early(pg::fork_plan_kernel, dim3(1), pg::PLAN_THREADS, 0, stream, table, lens, refs,
               refs_out, parents, children, n, slots, max_pages, pages, apart, work, status);
  launch_early(pg::fork_apply_kernel, dim3(slots + pg::copy_ctas(cache, n)), pg::COPY_THREADS, 0,
               stream, table, table_out, lens, lens_out, refs_out, parents, n, slots, max_pages, apart,
               work, cache, runtime_status_ptr());
  return static_cast<int>(cudaGetLastError());
}

extern "C" int orinfer_free_pages(const int* table, int* table_out, const int* lens, int* lens_out,
                                  const int* refs, int* refs_out, const int* gone, int n, int slots,
                                  int max_pages, int pages, cudaStream_t stream) {
  if (n < 0 || slots <= 0 || max_pages <= 0 || pages <= 0) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  if (slots > pg::FREE_MOST || n > pg::FREE_MOST) return -1;
  if (static_cast<long long>(n) * max_pages >= 1LL << 31) return -1;
  const size_t smem = ((slots + 31) / 32 + (n + 31) / 32) * sizeof(int);
  const int ranges = (pages + pg::RANGE - 1) / pg::RANGE;
  // in place the references come first: the rows that they are counted from are emptied
  const bool apart = table == table_out || lens == lens_out;
  auto start = [&](int parts) {
    const int ctas = (parts & pg::ROWS ? slots : 0) + (parts & pg::REFS ? ranges : 0);
    launch_early(pg::free_kernel, dim3(ctas), pg::FREE_THREADS, smem, stream, table, table_out, lens, lens_out,
                 refs, refs_out, gone, n, slots, max_pages, pages, parts, runtime_status_ptr());
  };
  if (apart) {
    start(pg::REFS);
    start(pg::ROWS);
  } else {
    start(pg::REFS | pg::ROWS);
  }
  return static_cast<int>(cudaGetLastError());
}

// moved: int32 [pages], where each page has gone.  work: int32 [4 + 3 (pages / 2 + 1)].
extern "C" int orinfer_compact_pages(const long long* bases, const int* token_bytes,
                                     const int* units, int n_units, int pages, const int* table,
                                     int* table_out, const int* refs, int* refs_out, int* moved,
                                     int slots, int max_pages, int* work, cudaStream_t stream) {
  if (slots < 0 || max_pages < 0 || pages <= 0 || n_units < 0 || !work || !moved) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  const long long cells = static_cast<long long>(slots) * max_pages;
  launch_early(pg::compact_plan_kernel, dim3(1), pg::PLAN_THREADS, 0, stream, refs, refs_out, moved,
               pages, work);
  const pg::Cache cache = {bases, token_bytes, units, n_units, pages};
  const int remap = pg::grid_of(cells), ctas = remap + pg::copy_ctas(cache, pages / 2);
  if (ctas > 0)
    launch_early(pg::compact_apply_kernel, dim3(ctas), pg::COPY_THREADS, 0, stream, table, table_out,
                 cells, moved, pages, remap, work, cache, runtime_status_ptr());
  return static_cast<int>(cudaGetLastError());
}
