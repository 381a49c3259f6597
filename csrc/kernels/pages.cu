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
// work: head; copies [n][3]; pairs in the order of their new pages [n]; pair of a child slot [slots]
__host__ __device__ inline size_t fork_work(int n, int slots) {
  return WORK_HEAD + 4 * static_cast<size_t>(n) + slots;
}

__global__ void __launch_bounds__(PLAN_THREADS) fork_plan_kernel(
    const int* table, const int* lens, const int* refs, int* refs_out, const int* parents,
    const int* children, int n, int slots, int max_pages, int pages, int* work, int* status_out) {
  __shared__ int sums[PLAN_THREADS / 32];
  __shared__ int s_wrong;
  int* copies = work + WORK_HEAD;
  int* owner = copies + 3 * n;
  int* child_of = owner + n;
  const int tid = threadIdx.x;
  grid_wait();
  grid_release();
  if (tid == 0) s_wrong = 0;
  for (int s = tid; s < slots; s += PLAN_THREADS) child_of[s] = -1;
  __syncthreads();
  // ---- the pairs: slots that exist, a child that is empty and named once, pages that are held
  for (int i = tid; i < n; i += PLAN_THREADS) {
    const int p = parents[i], c = children[i];
    bool wrong = p < 0 || p >= slots || c < 0 || c >= slots || p == c;
    if (!wrong) wrong = lens[c] != 0 || lens[p] < 0 || lens[p] > max_pages * PAGE;
    if (!wrong) wrong = atomicCAS(&child_of[c], -1, i) != -1;
    if (!wrong) {
      const int* row = table + static_cast<size_t>(p) * max_pages;
      for (int j = 0; j < (lens[p] + PAGE - 1) / PAGE; ++j) {
        const int page = row[j];
        wrong = wrong || page <= 0 || page >= pages || refs[page] <= 0;
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
      if (tail) owner[rank] = i;
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
  __syncthreads();
  if (status == 0 && found < need) status = 1;
  if (status == 0)
    for (int r = tid; r < need; r += PLAN_THREADS) refs_out[copies[3 * owner[r] + 1]] = 1;
  if (tid == 0) {
    work[0] = status;
    work[1] = status == 0 ? n : 0;
    *status_out = status;
  }
}

// The table's rows, lens and the references of shared pages; CTA per slot.
__global__ void __launch_bounds__(128) fork_rows_kernel(
    const int* table, int* table_out, const int* lens, int* lens_out, int* refs_out,
    const int* parents, int n, int slots, int max_pages, const int* work) {
  grid_wait();
  grid_release();
  const int* copies = work + WORK_HEAD;
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

// ---------------------------------------------------------------- copies
template <class T>
__device__ __forceinline__ void copy_as(const unsigned char* from, unsigned char* to, int bytes) {
  const int n = bytes / static_cast<int>(sizeof(T));
  for (int i = threadIdx.x; i < n; i += COPY_THREADS)
    reinterpret_cast<T*>(to)[i] = reinterpret_cast<const T*>(from)[i];
  for (int i = n * static_cast<int>(sizeof(T)) + threadIdx.x; i < bytes; i += COPY_THREADS)
    to[i] = from[i];
}

// copies [*count][3]: source page, target page, tokens from the page's first on
__global__ void __launch_bounds__(COPY_THREADS) copy_pages_kernel(const Cache cache,
                                                                  const int* copies,
                                                                  const int* count, int* status) {
  grid_wait();
  grid_release();
  const long long total = static_cast<long long>(*count) * cache.n_units;
  for (long long w = blockIdx.x; w < total; w += gridDim.x) {
    const int* c = copies + w / cache.n_units * 3;
    const int* u = cache.units + w % cache.n_units * 3;
    const int from = c[0], to = c[1], tokens = min(c[2] - u[1], u[2]);
    if (tokens <= 0) continue;
    if (from < 0 || from >= cache.pages || to < 0 || to >= cache.pages || c[2] > PAGE) {
      if (threadIdx.x == 0) report_status(status, STATUS_BAD_INDEX, 0x40);
      continue;
    }
    const long long per = cache.token_bytes[u[0]];
    unsigned char* base = reinterpret_cast<unsigned char*>(cache.bases[u[0]]) + u[1] * per;
    const unsigned char* src = base + from * PAGE * per;
    unsigned char* dst = base + to * PAGE * per;
    const int bytes = tokens * static_cast<int>(per);
    const uintptr_t off = reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst);
    if ((off & 15) == 0)
      copy_as<uint4>(src, dst, bytes);
    else if ((off & 3) == 0)
      copy_as<uint32_t>(src, dst, bytes);
    else
      copy_as<unsigned char>(src, dst, bytes);
  }
}

// ---------------------------------------------------------------- free
__global__ void __launch_bounds__(256) copy_ints_kernel(const int* a, int* a_out, long long na,
                                                        const int* b, int* b_out, long long nb,
                                                        const int* c, int* c_out, long long nc) {
  grid_wait();
  grid_release();
  const long long at = blockIdx.x * 256LL + threadIdx.x, step = gridDim.x * 256LL;
  if (a != a_out)
    for (long long i = at; i < na; i += step) a_out[i] = a[i];
  if (b != b_out)
    for (long long i = at; i < nb; i += step) b_out[i] = b[i];
  if (c != c_out)
    for (long long i = at; i < nc; i += step) c_out[i] = c[i];
}

// CTA per listed slot; a slot that is named again is left to the first
__global__ void __launch_bounds__(128) free_kernel(int* table, int* lens, int* refs,
                                                   const int* gone, int slots, int max_pages,
                                                   int pages, int* status) {
  grid_wait();
  grid_release();
  const int s = gone[blockIdx.x];
  bool again = false;
  for (int i = threadIdx.x; i < static_cast<int>(blockIdx.x); i += blockDim.x)
    again = again || gone[i] == s;
  if (__syncthreads_or(again)) return;
  if (s < 0 || s >= slots) {
    if (threadIdx.x == 0) report_status(status, STATUS_BAD_INDEX, 0x41);
    return;
  }
  int* row = table + static_cast<size_t>(s) * max_pages;
  for (int j = threadIdx.x; j < max_pages; j += blockDim.x) {
    const int page = row[j];
    row[j] = 0;
    if (page == 0) continue;
    if (page < 0 || page >= pages) {
      report_status(status, STATUS_BAD_INDEX, 0x42);
    } else if (atomicSub(&refs[page], 1) <= 0) {       // released more often than held
      atomicAdd(&refs[page], 1);
      report_status(status, STATUS_BAD_INDEX, 0x43);
    }
  }
  if (threadIdx.x == 0) lens[s] = 0;
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

__global__ void __launch_bounds__(256) remap_kernel(const int* table, int* table_out, long long n,
                                                    const int* moved, int pages, int* status) {
  grid_wait();
  grid_release();
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) {
    const int page = table[i];
    const bool known = page >= 0 && page < pages;
    if (!known) report_status(status, STATUS_BAD_INDEX, 0x44);
    table_out[i] = known ? moved[page] : page;
  }
}

static void launch_copies(const Cache& cache, const int* copies, const int* count, int most,
                          cudaStream_t stream) {
  const long long units = static_cast<long long>(most) * cache.n_units;
  const int grid = static_cast<int>(units < 8 * 148 ? units : 8 * 148);
  if (grid > 0)
    launch_early(copy_pages_kernel, dim3(grid), COPY_THREADS, 0, stream, cache, copies, count,
                 runtime_status_ptr());
}

static int grid_of(long long n) {
  const long long g = (n + 255) / 256;
  return static_cast<int>(g < 1 ? 1 : g < 592 ? g : 592);
}

}  // namespace pg
}  // namespace orinfer

using namespace orinfer;

extern "C" size_t orinfer_fork_work(int n, int slots) {
  return n < 0 || slots < 0 ? 0 : pg::fork_work(n, slots);
}
extern "C" size_t orinfer_compact_work(int pages) {
  return pages < 0 ? 0 : pg::WORK_HEAD + 3 * (static_cast<size_t>(pages) / 2 + 1);
}

// copies: int32 [*count, 3] on the device, at most `most` of them
extern "C" int orinfer_copy_pages(const long long* bases, const int* token_bytes, const int* units,
                                  int n_units, int pages, const int* copies, const int* count,
                                  int most, cudaStream_t stream) {
  if (most <= 0 || n_units <= 0) return most < 0 || n_units < 0 ? -1 : 0;
  if (!bases || !token_bytes || !units || !copies || !count || pages <= 0) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  pg::launch_copies(pg::Cache{bases, token_bytes, units, n_units, pages}, copies, count, most,
                    stream);
  return static_cast<int>(cudaGetLastError());
}

// status: 0, 1 (not enough free pages) or 2 (a pair that cannot be); then nothing is changed.
// work: int32 [orinfer_fork_work(n, slots)].
extern "C" int orinfer_fork_pages(const long long* bases, const int* token_bytes, const int* units,
                                  int n_units, int pages, const int* table, int* table_out,
                                  const int* lens, int* lens_out, const int* refs, int* refs_out,
                                  const int* parents, const int* children, int n, int slots,
                                  int max_pages, int* work, int* status, cudaStream_t stream) {
  if (n < 0 || slots <= 0 || max_pages <= 0 || pages <= 0 || n_units < 0) return -1;
  if (max_pages > (1 << 24) || !work || !status) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  launch_early(pg::fork_plan_kernel, dim3(1), pg::PLAN_THREADS, 0, stream, table, lens, refs,
               refs_out, parents, children, n, slots, max_pages, pages, work, status);
  launch_early(pg::fork_rows_kernel, dim3(slots), 128, 0, stream, table, table_out, lens, lens_out,
               refs_out, parents, n, slots, max_pages, work);
  pg::launch_copies(pg::Cache{bases, token_bytes, units, n_units, pages}, work + pg::WORK_HEAD,
                    work + 1, n, stream);
  return static_cast<int>(cudaGetLastError());
}

extern "C" int orinfer_free_pages(const int* table, int* table_out, const int* lens, int* lens_out,
                                  const int* refs, int* refs_out, const int* gone, int n, int slots,
                                  int max_pages, int pages, cudaStream_t stream) {
  if (n < 0 || slots <= 0 || max_pages <= 0 || pages <= 0) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  const long long cells = static_cast<long long>(slots) * max_pages;
  if (table != table_out || lens != lens_out || refs != refs_out)
    launch_early(pg::copy_ints_kernel, dim3(pg::grid_of(cells)), 256, 0, stream, table, table_out,
                 cells, lens, lens_out, static_cast<long long>(slots), refs, refs_out,
                 static_cast<long long>(pages));
  if (n > 0)
    launch_early(pg::free_kernel, dim3(n), 128, 0, stream, table_out, lens_out, refs_out, gone,
                 slots, max_pages, pages, runtime_status_ptr());
  return static_cast<int>(cudaGetLastError());
}

// moved: int32 [pages], where each page has gone.  work: int32 [orinfer_compact_work(pages)].
extern "C" int orinfer_compact_pages(const long long* bases, const int* token_bytes,
                                     const int* units, int n_units, int pages, const int* table,
                                     int* table_out, const int* refs, int* refs_out, int* moved,
                                     int slots, int max_pages, int* work, cudaStream_t stream) {
  if (slots < 0 || max_pages < 0 || pages <= 0 || n_units < 0 || !work || !moved) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  const long long cells = static_cast<long long>(slots) * max_pages;
  launch_early(pg::compact_plan_kernel, dim3(1), pg::PLAN_THREADS, 0, stream, refs, refs_out, moved,
               pages, work);
  if (cells > 0)
    launch_early(pg::remap_kernel, dim3(pg::grid_of(cells)), 256, 0, stream, table, table_out,
                 cells, moved, pages, runtime_status_ptr());
  pg::launch_copies(pg::Cache{bases, token_bytes, units, n_units, pages}, work + pg::WORK_HEAD,
                    work + 1, pages / 2, stream);
  return static_cast<int>(cudaGetLastError());
}
