// Penalties for repeated tokens, biases and grammar masks on logits, ahead of the device's arg-max
// and sampler.
//
// The arithmetic is the host law's (csrc/core/sampling_core.cpp), in 64 bits and rounded once to
// FP32: with c the occurrences of a token in the row's history,
//   s = logit;  c > 0: s = s < 0 ? s * repetition : s / repetition, s -= presence;
//   s -= frequency * c;  s += bias;  a token that the row's mask does not permit gets `masked`.
// Only tokens that occur or have a bias need any of it; the others are copied.
//
// It is a pass over memory, 8 bytes a token.  A cluster of eight CTAs takes a row.  Each CTA streams an
// eighth of the vocabulary, copying what is permitted, four tokens to a load.  Of the tokens that occur
// or have a bias it looks after those that leave its rank modulo eight: it counts them in a table in
// shared memory and lists them, and when the row has been streamed it computes their scores, which
// whole warps then do, whichever tokens are frequent.  Of a long history each CTA sorts an eighth by
// the CTA that looks after a token, and fetches its own tokens from all eight.  The barriers between
// these steps are in halves, with the streaming or the counting between them, and all that a row needs
// besides its logits is asked for at the start: under load each round trip is 2500 cycles.
//
// 256 rows of 151936 tokens: 56 us without penalties and masks (a copy takes 49), 58 with a mask for
// half of the rows, 64 with histories of 250 tokens, 83 with 8000, 88 with 150 biases too; 64 rows 29,
// 16 rows 14.5, one row with 900 tokens 6.5.  What bounds it is memory first, then the chain of a CTA
// (a third of its time streams), of which three share an SM.
// Tried: scores as a branch of the streaming loop (a slice's few tokens one by one: 256 rows 210),
// slices of neighbouring tokens counted by atomics in each other's shared memory (155, and 200 where
// most of the history falls to one slice), the CTA that met a token first looking after it (158), each
// CTA reading the whole history (118), that by half of its warps while the others stream (121), whole
// barriers between the steps (97).
#include "api.h"
#include "common.cuh"

namespace orinfer {
namespace lp {

constexpr int CTAS = 8;                            // per row
constexpr int TABLE = 24576;                       // tokens that a CTA looks after at a time, at most
constexpr int LIST = 4096;                         // of which so many are listed
constexpr int BIASES = 32768;                      // of a row, at most
constexpr int BATCH = 5;                           // loads of a thread in flight
constexpr int SEG = 2048;                          // tokens of a history that a CTA sorts at a time
constexpr int SHORT = 32767;                       // tokens of a history whose counts take 16 bits

struct Args {
  const float* logits;
  long long row_stride;
  const int* history;
  long long history_stride;
  const int* history_len;
  int history_cap;
  const double *repetition, *presence, *frequency;
  const int *bias_start, *bias_ids;
  const double* bias_values;
  const unsigned int* mask;
  long long mask_stride;
  const int* mask_rows;
  int mask_count;
  float masked;
  float* out;
  long long out_stride;
  int* flags;
  int rows, vocab, bias_total;
};

// A word per token: its occurrences, and in the top bit whether it has a bias, whose thread then writes
// it.  Words of 16 bits, for histories that cannot count further, leave the L1 cache, through which the
// logits come, the room to have them in flight (256 rows of 151936 without a history, of 49 us for a
// copy: 59 with it, 69 without).
template <class W>
struct Words {
  static constexpr unsigned BIASED = 1u << (8 * sizeof(W) - 1);
  W* at;
  __device__ __forceinline__ unsigned operator[](unsigned i) const { return at[i]; }
  __device__ __forceinline__ void set(unsigned i, unsigned v) { at[i] = static_cast<W>(v); }
  // adds one, and returns what was there
  __device__ __forceinline__ unsigned count(unsigned i) {
    if (sizeof(W) == 4) return atomicAdd(reinterpret_cast<unsigned*>(at) + i, 1u);
    const unsigned shift = (i & 1) * 16;
    return atomicAdd(reinterpret_cast<unsigned*>(at) + i / 2, 1u << shift) >> shift & 0xffffu;
  }
  __device__ __forceinline__ void raise(unsigned i, unsigned v) {
    unsigned* word = reinterpret_cast<unsigned*>(at) + (sizeof(W) == 4 ? i : i / 2);
    const unsigned shift = sizeof(W) == 4 ? 0 : (i & 1) * 16, all = sizeof(W) == 4 ? ~0u : 0xffffu;
    unsigned old = *word;
    while ((old >> shift & all) < v) {
      const unsigned was = atomicCAS(word, old, (old & ~(all << shift)) | v << shift);
      if (was == old) break;
      old = was;
    }
  }
};

// Tokens that a CTA looks after at a time, and its dynamic shared memory: their words, the mask's words
// of its slice and one more, the list.
__host__ __device__ inline int table_words(int vocab) {
  const int own = (vocab + CTAS - 1) / CTAS;
  return ((own < TABLE ? own : TABLE) + 7) / 8 * 8;
}
__host__ __device__ inline int slice_of(int vocab) {
  return (vocab + 32 * CTAS - 1) / (32 * CTAS) * 32;
}
constexpr int MASK_WORDS = 1024;                   // of a slice, held in shared memory

// The cluster's barrier in two halves, whole warps each: what a thread wrote before it arrived, the
// others see past the wait.
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// What the CTA `rank` of the cluster has at the place of `p`.
__device__ __forceinline__ int cluster_load(const int* p, int rank) {
  int v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_u32(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ unsigned cluster_load(const unsigned short* p, int rank) {
  unsigned short v;
  asm volatile("ld.shared::cluster.u16 %0, [%1];" : "=h"(v) : "r"(mapa_u32(smem_u32(p), rank)) : "memory");
  return v;
}

template <class W, int THREADS, int RESIDENT>
__global__ void __launch_bounds__(THREADS, RESIDENT) process_logits_kernel(const Args a) {
  constexpr int WINS = (BIASES / THREADS + 64) / 64;       // words of a bit per bias entry of a thread
  constexpr int TAKES = (SEG / 4 + THREADS - 1) / THREADS; // fours of tokens that a thread sorts
  constexpr int HOLDS = (MASK_WORDS + THREADS - 1) / THREADS;
  constexpr unsigned BIASED = Words<W>::BIASED;
  extern __shared__ __align__(16) unsigned char space[];
  __shared__ unsigned s_mask[MASK_WORDS + 1];
  __shared__ unsigned short list[LIST];
  __shared__ unsigned short sorted[SEG];           // what this CTA sorted, by the CTA that looks after it
  __shared__ int s_count[CTAS], s_start[CTAS + 1]; // tokens for each of them, and where they begin
  __shared__ int s_at[CTAS], s_sum[CTAS + 1];      // what the CTAs sorted for this one
  __shared__ int s_flags[CTAS];
  __shared__ int s_listed;
  grid_wait();
  grid_release();
  cluster_arrive();                                // 1: all CTAs have started
  const int row = blockIdx.x / CTAS, rank = blockIdx.x % CTAS, tid = threadIdx.x;
  const int words = table_words(a.vocab);
  const unsigned most = words;
  Words<W> table{reinterpret_cast<W*>(space)};
  const float* x = a.logits + row * a.row_stride;
  float* out = a.out + row * a.out_stride;
  // ---- the slice that is streamed: four tokens at a time behind the first 16-byte boundary, where
  // both rows have theirs together
  const int slice = slice_of(a.vocab);
  const int lo = rank * slice, n = max(0, min(slice, a.vocab - lo));
  const bool vectors =
      ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  const int first =
      vectors ? static_cast<int>((16 - (reinterpret_cast<uintptr_t>(x + lo) & 15)) / 4 & 3) : 0;
  const int groups = vectors ? max(0, n - first) / 4 : 0;
  const float4* x4 = reinterpret_cast<const float4*>(x + lo + first);
  float4* out4 = reinterpret_cast<float4*>(out + lo + first);
  float4 v[BATCH];
  auto load = [&](int g0) {
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
      if (g0 + k * THREADS < groups) v[k] = x4[g0 + k * THREADS];
  };
  load(tid);                                       // on their way while the table is made

  const double rep = a.repetition ? a.repetition[row] : 1.0;
  const double pres = a.presence ? a.presence[row] : 0.0;
  const double freq = a.frequency ? a.frequency[row] : 0.0;
  const int len = a.history ? min(max(a.history_len[row], 0), a.history_cap) : 0;
  const int* history = a.history + row * a.history_stride;
  const int b_lo = a.bias_start ? max(a.bias_start[row], 0) : 0;
  const int entries = a.bias_start ? min(a.bias_start[row + 1], a.bias_total) - b_lo : 0;
  const int which = a.mask ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
  const int seen = rep != 1.0 || pres != 0.0 || freq != 0.0 ? len : 0;
  const unsigned* mask =
      which >= 0 && which < a.mask_count ? a.mask + which * a.mask_stride : nullptr;
  // (a mask that does not exist, more biases than the winners' bits)
  const bool odd = (which >= 0 && !mask) || entries > BIASES;
  const bool biased = entries > 0 && !odd, special = seen > 0 || biased;
  const bool sorts = seen > 4 * THREADS;           // (else each CTA looks through all of them)

  // What a row needs besides its logits is asked for at once, and used as it comes: the slice's
  // permissions (from global memory later where they are too many), tokens, the first bias.
  const bool held = slice <= 32 * MASK_WORDS;
  const int mask_words = mask ? (n + 31) / 32 : 0;
  unsigned bits[HOLDS];
#pragma unroll
  for (int k = 0; k < HOLDS; ++k)
    bits[k] = held && tid + k * THREADS < mask_words ? mask[lo / 32 + tid + k * THREADS] : 0u;
  const bool wide = (reinterpret_cast<uintptr_t>(history) & 15) == 0;
  auto tokens_at = [&](int i) {                    // four of the history
    int4 t = make_int4(-1, -1, -1, -1);
    if (wide && i + 3 < seen) {
      t = *reinterpret_cast<const int4*>(history + i);
    } else {
      if (i < seen) t.x = history[i];
      if (i + 1 < seen) t.y = history[i + 1];
      if (i + 2 < seen) t.z = history[i + 2];
      if (i + 3 < seen) t.w = history[i + 3];
    }
    return t;
  };
  int4 next[TAKES];
  auto ask = [&](int from) {                       // this CTA's part of the tokens from there on
    const int part =
        sorts ? min(SEG, ((seen - from + CTAS - 1) / CTAS + 3) / 4 * 4) : 4 * THREADS;
#pragma unroll
    for (int k = 0; k < TAKES; ++k) {
      const int i = 4 * (tid + k * THREADS);
      next[k] = i < part ? tokens_at((sorts ? from + rank * part : 0) + i)
                         : make_int4(-1, -1, -1, -1);
    }
  };
  ask(0);
  const int bias_id = biased && tid < entries ? a.bias_ids[b_lo + tid] : -1;

  // ---- the words of tokens rank + 8 (done .. done + words): occurrences, and which have a bias
  unsigned long long wins[WINS] = {};              // this thread's bias entries that count
  auto won = [&](int k) { return (WINS > 1 && k > 63 ? wins[WINS - 1] : wins[0]) >> (k & 63) & 1; };
  auto own_at = [&](int token, int done) {         // a token's word, or something past the table
    const unsigned id = token;
    return id < static_cast<unsigned>(a.vocab) && id % CTAS == static_cast<unsigned>(rank)
               ? id / CTAS - done
               : 0xffffffffu;
  };
  auto make_table = [&](int done) {                // without the history
    if (tid == 0) s_listed = 0;
    for (int q = tid; q < words * static_cast<int>(sizeof(W)) / 16; q += THREADS)
      reinterpret_cast<uint4*>(space)[q] = make_uint4(0u, 0u, 0u, 0u);
    __syncthreads();
    if (!biased) return;                           // the last entry of a token is the one that counts
#pragma unroll
    for (int w = 0; w < WINS; ++w) wins[w] = 0;
    auto entry_at = [&](int i) { return own_at(i == tid ? bias_id : a.bias_ids[b_lo + i], done); };
    for (int i = tid; i < entries; i += THREADS)
      if (entry_at(i) < most) table.raise(entry_at(i), i + 1u);
    __syncthreads();
    for (int i = tid, k = 0; i < entries; i += THREADS, ++k)
      if (entry_at(i) < most && table[entry_at(i)] == i + 1u) {
        (k > 63 ? wins[WINS - 1] : wins[0]) |= 1ull << (k & 63);
        table.set(entry_at(i), BIASED);            // (no other entry of the token has this number)
      }
    __syncthreads();
  };
  auto count = [&](unsigned at) {                  // tokens met for the first time are listed
    if (at >= most || table.count(at) != 0) return;
    const int to = atomicAdd(&s_listed, 1);
    if (to < LIST) list[to] = static_cast<unsigned short>(at);
  };
  auto look_through = [&](int done) {
    count(own_at(next[0].x, done));
    count(own_at(next[0].y, done));
    count(own_at(next[0].z, done));
    count(own_at(next[0].w, done));
  };
  auto sort = [&](int done) {
    if (tid < CTAS) s_count[tid] = 0;
    __syncthreads();
    unsigned own[4 * TAKES];                       // the token's word, and above it its place
    auto place = [&](int e, int token) {
      const unsigned id = token, at = id / CTAS - done;
      own[e] = 0xffffffffu;
      if (id < static_cast<unsigned>(a.vocab) && at < most)
        own[e] = at | static_cast<unsigned>(atomicAdd(&s_count[id % CTAS], 1)) << 16;
    };
#pragma unroll
    for (int k = 0; k < TAKES; ++k) {
      place(4 * k, next[k].x);
      place(4 * k + 1, next[k].y);
      place(4 * k + 2, next[k].z);
      place(4 * k + 3, next[k].w);
    }
    __syncthreads();
    if (tid < 32) {                                // (a warp: lane c has CTA c's)
      int sum = tid < CTAS ? s_count[tid] : 0;
      for (int d = 1; d < CTAS; d *= 2) {
        const int below = __shfl_up_sync(0xffffffffu, sum, d);
        if (tid >= d) sum += below;
      }
      if (tid < CTAS) s_start[tid + 1] = sum;
      if (tid == 0) s_start[0] = 0;
    }
    __syncthreads();
    auto put = [&](int e, int token) {
      if (own[e] != 0xffffffffu)
        sorted[s_start[static_cast<unsigned>(token) % CTAS] + (own[e] >> 16)] =
            static_cast<unsigned short>(own[e]);
    };
#pragma unroll
    for (int k = 0; k < TAKES; ++k) {
      put(4 * k, next[k].x);
      put(4 * k + 1, next[k].y);
      put(4 * k + 2, next[k].z);
      put(4 * k + 3, next[k].w);
    }
  };
  auto gather = [&] {                              // counts what the CTAs have sorted for this one
    if (tid < 32) {
      const int at = tid < CTAS ? cluster_load(&s_start[rank], tid) : 0;
      int sum = tid < CTAS ? cluster_load(&s_start[rank + 1], tid) - at : 0;
      for (int d = 1; d < CTAS; d *= 2) {
        const int below = __shfl_up_sync(0xffffffffu, sum, d);
        if (tid >= d) sum += below;
      }
      if (tid < CTAS) {
        s_at[tid] = at;
        s_sum[tid + 1] = sum;
      }
      if (tid == 0) s_sum[0] = 0;
    }
    __syncthreads();
    for (int i = tid; i < s_sum[CTAS]; i += THREADS) {
      int c = 0;
#pragma unroll
      for (int k = 1; k < CTAS; ++k) c += i >= s_sum[k];
      count(cluster_load(&sorted[s_at[c] + i - s_sum[c]], c));
    }
  };
  auto sort_and_gather = [&](int from, int done) { // with all CTAs past the last of them
    for (; from < seen; from += CTAS * SEG) {
      __syncthreads();
      cluster_sync_all();
      ask(from);
      sort(done);
      __syncthreads();
      cluster_sync_all();
      gather();
    }
  };
  if (special) {
    make_table(0);
    if (sorts)
      sort(0);
    else
      look_through(0);
  }
  unsigned any = mask ? 0u : 1u;
  for (int w = tid, k = 0; w < mask_words; w += THREADS, ++k) {
    unsigned word = 0;
#pragma unroll
    for (int i = 0; i < HOLDS; ++i)
      if (i == k) word = bits[i];
    if (held)
      s_mask[w] = word;
    else
      word = mask[lo / 32 + w];
    any |= n - 32 * w < 32 ? word & ((1u << (n - 32 * w)) - 1u) : word;
  }
  __syncthreads();
  cluster_wait();                                  // 1
  if (sorts) cluster_arrive();                     // 2: the first tokens have been sorted

  // ---- the slice
  float nothing = 0.f;                             // 0, or NaN once a logit was not finite
  for (int g0 = tid; g0 < groups; g0 += BATCH * THREADS) {
    if (g0 > tid) load(g0);
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int g = g0 + k * THREADS;
      if (g >= groups) break;
      float4 y = v[k];
      nothing = fmaf(y.x, 0.f, fmaf(y.y, 0.f, fmaf(y.z, 0.f, fmaf(y.w, 0.f, nothing))));
      if (mask) {
        const int i = first + 4 * g, at = i & 31;
        const unsigned* m = held ? s_mask + (i >> 5) : mask + (lo + i >> 5);
        unsigned allowed = m[0] >> at;
        if (at > 28) allowed |= m[1] << (32 - at);                       // (of tokens of the group)
        if (!(allowed & 1u)) y.x = a.masked;
        if (!(allowed & 2u)) y.y = a.masked;
        if (!(allowed & 4u)) y.z = a.masked;
        if (!(allowed & 8u)) y.w = a.masked;
      }
      out4[g] = y;
    }
  }
  auto mask_at = [&](int id) { return mask ? mask[id >> 5] >> (id & 31) & 1u : 1u; };
  for (int j = tid; j < n - 4 * groups; j += THREADS) {          // ahead of the groups and behind them
    const int id = lo + (j < min(first, n) ? j : j + 4 * groups);
    const float f = x[id];
    nothing = fmaf(f, 0.f, nothing);
    out[id] = mask_at(id) ? f : a.masked;
  }
  __syncwarp();
  if (sorts) cluster_wait();                       // 2
  const bool bad = __syncthreads_or(odd || !(nothing == 0.f));
  const bool some = __syncthreads_or(any);
  if (tid == 0) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_u32(smem_u32(&s_flags[rank]), 0)),
                 "r"((bad ? 2 : 0) | (some ? 1 : 0))
                 : "memory");
    if (rank == 0) a.flags[row] = 0;
  }
  __syncthreads();
  cluster_arrive();                                // 3: the row has been streamed
  if (sorts) gather();
  __syncthreads();
  cluster_wait();                                  // 3
  if (rank == 0 && tid == 0) {
    int all = 0;
    for (int c = 0; c < CTAS; ++c) all |= *reinterpret_cast<volatile int*>(&s_flags[c]);
    if (all != 1) atomicMax(a.flags + row, all & 2 ? 2 : 1);
  }
  if (!special) return;

  // ---- scores of tokens that occur or have a bias, in 64 bits and each operation rounded by itself, as
  // on the host: a product that goes into a difference unrounded (which the compiler would do) leaves
  // 1e-17 where the host has 0, and breaks a tie.  What is permitted has been copied, so that its logit
  // is still there where out is the logits.
  auto write_score = [&](int id, unsigned word, unsigned permitted, float logit, double bias) {
    if (!permitted) return;
    const int times = word & (BIASED - 1u);
    double s = logit;
    if (times > 0) s = __dsub_rn(s < 0.0 ? __dmul_rn(s, rep) : s / rep, pres);
    s = __dsub_rn(s, __dmul_rn(freq, times));
    if (word & BIASED) s = __dadd_rn(s, bias);
    const float f = static_cast<float>(s);
    out[id] = f;
    if (!isfinite(f)) atomicMax(a.flags + row, 2);
  };
  if (sorts) {
    sort_and_gather(CTAS * SEG, 0);
    __syncthreads();
    cluster_arrive();                              // 4: what was sorted has been read
  }
  for (int done = 0;; done += words) {
    // the first bias is on its way beside the first of the list
    const bool leads = biased && won(0);
    const unsigned lead_may = leads ? mask_at(bias_id) : 0u;
    const float lead_logit = leads ? x[bias_id] : 0.f;
    const double lead_bias = leads ? a.bias_values[b_lo + tid] : 0.0;
    auto look_after = [&](unsigned i) {
      const int id = (done + static_cast<int>(i)) * CTAS + rank;
      const unsigned may = mask_at(id);
      write_score(id, table[i], may, x[id], 0.0);
    };
    if (s_listed <= LIST) {
      for (int i = tid; i < s_listed; i += THREADS) look_after(list[i]);
    } else {                                       // the list has no room: all that occur
      for (int i = tid; i < words; i += THREADS)
        if (table[i] != 0 && !(table[i] & BIASED)) look_after(i);
    }
    if (leads)
      write_score(bias_id, table[own_at(bias_id, done)], lead_may, lead_logit, lead_bias);
    for (int i = tid + THREADS, k = 1; i < entries && biased; i += THREADS, ++k)
      if (won(k)) {
        const int id = a.bias_ids[b_lo + i];
        const unsigned may = mask_at(id);
        const float logit = x[id];
        write_score(id, table[own_at(id, done)], may, logit, a.bias_values[b_lo + i]);
      }
    __syncwarp();
    if (sorts && done == 0) cluster_wait();        // 4
    if ((done + words) * CTAS >= a.vocab) {
      if (sorts && done > 0) {
        __syncthreads();
        cluster_sync_all();
      }
      return;
    }
    __syncthreads();
    make_table(done + words);
    if (sorts)
      sort_and_gather(0, done + words);
    else
      look_through(done + words);
    __syncthreads();
  }
}

}  // namespace lp
}  // namespace orinfer

using namespace orinfer;

// logits, out: fp32 [rows, vocab] with row strides in elements (out may be logits itself).
// history: int32 [rows, history_cap]; repetition, presence, frequency: fp64 [rows] or null (1, 0,
// 0).  Biases of row r are entries bias_start[r] .. bias_start[r + 1] of bias_total; the last one of
// a token counts.  mask: rows of (vocab + 31) / 32 words, bit set = permitted; row r uses row
// mask_rows[r] (none below 0), or row r where mask_rows is null.  flags[r]: 0, 1 where nothing is
// permitted, 2 where a logit or a permitted token's score is not finite, the mask does not exist or
// the row has more than 32768 biases.
extern "C" int orinfer_process_logits(
    const float* logits, long long row_stride, const int* history, long long history_stride,
    int history_cap, const int* history_len, const double* repetition, const double* presence,
    const double* frequency, const int* bias_start, const int* bias_ids, const double* bias_values,
    int bias_total, const int* mask, long long mask_stride, const int* mask_rows, int mask_count,
    float masked, float* out, long long out_stride, int* flags, int rows, int vocab,
    cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (rows > (1 << 27) || vocab <= 0 || row_stride < vocab || out_stride < vocab || !logits || !out || !flags) return -1;
  if (history && (!history_len || history_cap < 0 || history_cap > 1 << 29)) return -1;
  if (bias_start && (bias_total < 0 || (bias_total > 0 && (!bias_ids || !bias_values)))) return -1;
  if (mask && (mask_stride < (vocab + 31) / 32 || mask_count < (mask_rows ? 0 : rows))) return -1;
  const lp::Args a = {logits, row_stride, history, history_stride, history_len, history_cap,
                      repetition, presence, frequency, bias_start, bias_ids, bias_values,
                      reinterpret_cast<const unsigned int*>(mask), mask_stride, mask_rows,
                      mask_count, masked, out, out_stride, flags, rows, vocab, bias_total};
  const bool narrow = !history || history_cap <= lp::SHORT;
  // Threads of a CTA, and with them CTAs of an SM: 512 and two where one such wave takes all rows (32
  // rows 17 us, with 320 threads 20), else 320 and three (256 rows 88 us, with 512 threads 98).
  const bool few = rows * static_cast<long long>(lp::CTAS) <= 2 * 148;
  auto kernel = few ? (narrow ? lp::process_logits_kernel<uint16_t, 512, 2>
                              : lp::process_logits_kernel<uint32_t, 512, 2>)
                    : (narrow ? lp::process_logits_kernel<uint16_t, 320, 3>
                              : lp::process_logits_kernel<uint32_t, 320, 3>);
  static const int slot[4] = {runtime_new_slot(), runtime_new_slot(), runtime_new_slot(),
                              runtime_new_slot()};
  if (const int e = runtime_allow_smem(slot[2 * few + narrow], kernel, 4 * lp::TABLE)) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(rows) * lp::CTAS);
  cfg.blockDim = dim3(few ? 512 : 320);
  cfg.dynamicSmemBytes = (narrow ? 2 : 4) * static_cast<size_t>(lp::table_words(vocab));
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;       // see launch_early
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = lp::CTAS;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = rows <= EARLY_CTAS / lp::CTAS ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  return static_cast<int>(e != cudaSuccess ? e : cudaGetLastError());
}
