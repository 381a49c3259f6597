// Penalties for repeated tokens, biases and grammar masks on logits, ahead of the device's arg-max
// and sampler.
//
// The arithmetic is the host law's (csrc/core/sampling_core.cpp), in 64 bits and rounded once to
// FP32: with c the occurrences of a token in the row's history,
//   s = logit;  c > 0: s = s < 0 ? s * repetition : s / repetition, s -= presence;
//   s -= frequency * c;  s += bias;  a token that the row's mask does not permit gets `masked`.
// Only tokens that occur or have a bias need any of it; the others are copied.
//
// One CTA per row walks the vocabulary in tiles and counts the history's tokens of a tile in shared
// memory.
#include "api.h"
#include "common.cuh"

namespace orinfer {
namespace lp {

constexpr int THREADS = 512;
constexpr int TILE = 4096;                         // tokens whose counts are held at a time

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

__global__ void __launch_bounds__(THREADS) process_logits_kernel(const Args a) {
  __shared__ int count[TILE], entry[TILE];         // occurrences; the last bias entry, plus one
  __shared__ int s_bad, s_any;
  const int row = blockIdx.x, tid = threadIdx.x;
  const float* x = a.logits + row * a.row_stride;
  float* out = a.out + row * a.out_stride;
  const double rep = a.repetition ? a.repetition[row] : 1.0;
  const double pres = a.presence ? a.presence[row] : 0.0;
  const double freq = a.frequency ? a.frequency[row] : 0.0;
  const bool counted = a.history && (rep != 1.0 || pres != 0.0 || freq != 0.0);
  const int seen = counted ? min(max(a.history_len[row], 0), a.history_cap) : 0;
  const int* history = a.history + row * a.history_stride;
  const int b_lo = a.bias_start ? max(a.bias_start[row], 0) : 0;
  const int b_hi = a.bias_start ? min(a.bias_start[row + 1], a.bias_total) : 0;
  const int which = a.mask ? (a.mask_rows ? a.mask_rows[row] : row) : -1;
  const unsigned int* mask =
      which >= 0 && which < a.mask_count ? a.mask + which * a.mask_stride : nullptr;
  if (tid == 0) s_bad = s_any = 0;
  bool bad = which >= a.mask_count, any = false;   // (a mask that does not exist)
  for (int lo = 0; lo < a.vocab; lo += TILE) {
    const int n = min(TILE, a.vocab - lo);
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) count[i] = entry[i] = 0;
    __syncthreads();
    for (int i = tid; i < seen; i += THREADS) {
      const unsigned id = static_cast<unsigned>(history[i]) - lo;
      if (id < static_cast<unsigned>(n)) atomicAdd(&count[id], 1);
    }
    for (int i = b_lo + tid; i < b_hi; i += THREADS) {
      const unsigned id = static_cast<unsigned>(a.bias_ids[i]) - lo;
      if (id < static_cast<unsigned>(n)) atomicMax(&entry[id], i - b_lo + 1);
    }
    __syncthreads();
    for (int i = tid; i < n; i += THREADS) {
      const int id = lo + i;
      const bool permitted = !mask || (mask[id >> 5] >> (id & 31) & 1u);
      float v = x[id];
      bad = bad || !isfinite(v);
      any = any || permitted;
      if (!permitted) {
        v = a.masked;
      } else if (count[i] || entry[i]) {
        const int c = count[i];
        double s = v;
        if (c > 0) {
          s = s < 0.0 ? s * rep : s / rep;
          s -= pres;
        }
        s -= freq * c;
        if (entry[i]) s += a.bias_values[b_lo + entry[i] - 1];
        v = static_cast<float>(s);
        bad = bad || !isfinite(v);
      }
      out[id] = v;
    }
  }
  if (bad) s_bad = 1;
  if (any) s_any = 1;
  __syncthreads();
  if (tid == 0) a.flags[row] = s_bad ? 2 : s_any ? 0 : 1;
}

}  // namespace lp
}  // namespace orinfer

using namespace orinfer;

// logits, out: fp32 [rows, vocab] with row strides in elements (out may be logits itself).
// history: int32 [rows, history_cap]; repetition, presence, frequency: fp64 [rows] or null (1, 0,
// 0).  Biases of row r are entries bias_start[r] .. bias_start[r + 1] of bias_total; the last one of
// a token counts.  mask: rows of (vocab + 31) / 32 words, bit set = permitted; row r uses row
// mask_rows[r] (none below 0), or row r where mask_rows is null.  flags[r]: 0, 1 where nothing is
// permitted, 2 where a logit or a permitted token's score is not finite or the mask does not exist.
extern "C" int orinfer_process_logits(
    const float* logits, long long row_stride, const int* history, long long history_stride,
    int history_cap, const int* history_len, const double* repetition, const double* presence,
    const double* frequency, const int* bias_start, const int* bias_ids, const double* bias_values,
    int bias_total, const int* mask, long long mask_stride, const int* mask_rows, int mask_count,
    float masked, float* out, long long out_stride, int* flags, int rows, int vocab,
    cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (vocab <= 0 || row_stride < vocab || out_stride < vocab || !logits || !out || !flags) return -1;
  if (history && (!history_len || history_cap < 0)) return -1;
  if (bias_start && (bias_total < 0 || (bias_total > 0 && (!bias_ids || !bias_values)))) return -1;
  if (mask && (mask_stride < (vocab + 31) / 32 || mask_count < (mask_rows ? 0 : rows))) return -1;
  const lp::Args a = {logits, row_stride, history, history_stride, history_len, history_cap,
                      repetition, presence, frequency, bias_start, bias_ids, bias_values,
                      reinterpret_cast<const unsigned int*>(mask), mask_stride, mask_rows,
                      mask_count, masked, out, out_stride, flags, rows, vocab, bias_total};
  lp::process_logits_kernel<<<rows, lp::THREADS, 0, stream>>>(a);
  return static_cast<int>(cudaGetLastError());
}
