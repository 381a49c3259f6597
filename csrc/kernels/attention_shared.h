// What attention over a shared prefix hands to the row kernels: which keys of a row are its own, and
// where the parts of its shared keys stand.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace orinfer {

struct SharedParts {
  int pending = 0;                 // the kernel in front makes the parts; the row kernel runs beside it
  const int4* rows = nullptr;      // per row: shared keys, first part, parts, -
  const float* o = nullptr;        // [parts][query heads][D]: sums of weighted values
  const float2* ml = nullptr;      // [parts][query heads]: the weights' reference and their sum
  int* ready = nullptr;            // 1 where the kernel in front has waited for what lies before it
};

// Attention of single rows over the keys behind row.x, joined with the parts; see orinfer_attention.
int attention_own_keys(const __half* q, const __half* gate, const int* row_req, const int* row_pos,
                       const int* page_table, int max_pages, const int8_t* kc, const int8_t* vc,
                       const __half* ks, const __half* vs, __half* out, int rows, int qh, int kvh,
                       int head_dim, int splits, float* scratch, int context,
                       const SharedParts& parts, cudaStream_t stream);

}  // namespace orinfer
