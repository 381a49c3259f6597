// Attention of single rows whose contexts begin with the same pages (samples of one prompt,
// requests under one system prompt), over the paged INT8 cache.
//
// One CTA per (row, query head); its warps take the keys in turn, a lane holding the same channels
// of the query, of every key and of the output.  Online softmax in FP32, joined in shared memory.
#include "api.h"
#include "common.cuh"

namespace orinfer {
namespace sp {

constexpr int WARPS = 4;

template <int D>
__global__ void __launch_bounds__(WARPS * 32) rows_kernel(
    const __half* q, const __half* gate, const int* row_req, const int* row_pos,
    const int* page_table, int max_pages, const int8_t* kc, const int8_t* vc, const __half* ks,
    const __half* vs, __half* __restrict__ out, int qh, int kvh, int num_pages, int* status) {
  constexpr int PER = D / 32, G = D / 64;            // channels of a lane, scale groups
  grid_wait();
  grid_release();
  const int row = blockIdx.x, head = blockIdx.y, h = head / (qh / kvh);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = min(row_pos[row] + 1, max_pages * 128);
  const int* pages = page_table + static_cast<size_t>(row_req[row]) * max_pages;
  const size_t at = (static_cast<size_t>(row) * qh + head) * D + lane * PER;
  float qv[PER], acc[PER], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    qv[i] = __half2float(q[at + i]) * rsqrtf(static_cast<float>(D)) * 1.4426950408889634f;
    acc[i] = 0.f;
  }
  for (int key = warp; key < n; key += WARPS) {
    const int page = pages[key >> 7];
    if (page < 0 || page >= num_pages) {
      if (lane == 0) report_status(status, STATUS_BAD_INDEX, 0x50);
      continue;
    }
    const size_t slot = (static_cast<size_t>(page) * 128 + (key & 127)) * kvh + h;
    const int group = lane * PER / 64;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i) s = fmaf(qv[i], kc[slot * D + lane * PER + i], s);
    s = warp_sum(s * __half2float(ks[slot * G + group]));
    const float m_new = fmaxf(m, s), f = m == -INFINITY ? 0.f : exp2f(m - m_new);
    const float p = exp2f(s - m_new), scale = p * __half2float(vs[slot * G + group]);
    l = fmaf(l, f, p);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      acc[i] = fmaf(acc[i], f, scale * vc[slot * D + lane * PER + i]);
    m = m_new;
  }
  __shared__ float s_o[WARPS][D], s_m[WARPS], s_l[WARPS];
#pragma unroll
  for (int i = 0; i < PER; ++i) s_o[warp][lane * PER + i] = acc[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  float m_all = -INFINITY, l_all = 0.f;
  for (int w = 0; w < WARPS; ++w) m_all = fmaxf(m_all, s_m[w]);
  for (int d = threadIdx.x; d < D; d += WARPS * 32) {
    float o = 0.f;
    l_all = 0.f;
    for (int w = 0; w < WARPS; ++w) {
      const float f = s_m[w] == -INFINITY ? 0.f : exp2f(s_m[w] - m_all);
      o = fmaf(s_o[w][d], f, o);
      l_all = fmaf(s_l[w], f, l_all);
    }
    const size_t to = (static_cast<size_t>(row) * qh + head) * D + d;
    float v = l_all > 0.f ? o / l_all : 0.f;
    if (gate) v *= sigmoid_f32(__half2float(gate[to]));
    out[to] = __float2half_rn(v);
  }
}

}  // namespace sp
}  // namespace orinfer

using namespace orinfer;

extern "C" int orinfer_attention_shared(
    const __half* q, const __half* gate, const int* row_req, const int* row_pos,
    const int* page_table, int max_pages, const int8_t* kc, const int8_t* vc, const __half* ks,
    const __half* vs, __half* out, int rows, int qh, int kvh, int head_dim, int num_pages,
    cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (kvh <= 0 || qh % kvh || max_pages <= 0 || num_pages <= 0) return -1;
  const int rep = qh / kvh;
  if (rep != 1 && rep != 2 && rep != 4 && rep != 8 && !(rep == 5 && head_dim == 128)) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
#define CASE(D)                                                                                 \
  if (head_dim == D)                                                                            \
    launch_early(sp::rows_kernel<D>, dim3(rows, qh), sp::WARPS * 32, 0, stream, q, gate,        \
                 row_req, row_pos, page_table, max_pages, kc, vc, ks, vs, out, qh, kvh, num_pages, \
                 runtime_status_ptr());
  CASE(64) else CASE(128) else CASE(256) else return -1;
#undef CASE
  return static_cast<int>(cudaGetLastError());
}
