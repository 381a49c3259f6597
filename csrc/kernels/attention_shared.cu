// Attention of single rows whose contexts begin with the same pages (samples of one prompt,
// requests under one system prompt), over the paged INT8 cache.
//
// The shared keys of a group of rows are read once: the group's rows times the `rep` query heads of
// a KV head are the M axis of one product with the prefix, on tcgen05 tensor cores with TMEM
// accumulators.  A CTA takes a tile of 128 such rows and a range of the keys, and leaves each row's
// part of the softmax (reference, sum of weights, sum of weighted values) for the row kernels of
// attention.cu, which add the row's own keys and join the parts.
//
//   S_g = Q K_g^T   a sum of its own per group of 64 channels, K as the exact FP16 integers that the
//                   cache holds;  score = sum_g S_g x key scale_g in FP32;
//   O_g = P_g V_g   P_g = weight x value scale_g as the sum of two BF16 numbers, V as the exact BF16
//                   integers that the cache holds.
// So a weight is off by 2^-18 of it at most, whatever the other keys' weights and value scales are: BF16
// has FP32's range.  (One FP16 number under a unit that follows the value scales left 2.9e-4 against 64
// bits where the output's own rounding is 2.07e-4, and lost the bits of keys beside one with a large
// scale and no weight.)
//
// Scores of three steps have a place in TMEM, so that the products run ahead of the eight softmax warps
// (sixteen rows each), which go from step to step without a wait.  The weights replace the scores that
// they are made of.  Two teams of dequantising warps take a step each in turn.
//
// 64 rows of 32 query heads behind 16384 keys of 4 KV heads of 128: 38.7 us, 445 TFLOP/s, with the rows' own
// keys and the join 50.2 (each row reading all keys 237); 6.6 us of the 38.7 are the start and the end.
// What bounds it is a step of 64 keys, 2170 cycles, in which nothing is at work for long: a scheduler
// issues in 57 % of its cycles, the tensor pipe works for a third, conversions and logic for 42 %,
// exponentials for 22 %, DRAM for 5 %.  Without the weights (exponentials, halves, stores) a step takes
// 1560 cycles, without the dequantisation 1870, with neither 1230: each is a chain in few warps, and they
// wait for one another.  The weights' second halves cost 3.6 us (without their arithmetic 46.6): two
// conversions and two differences for each two weights.  (With those made behind all exponentials of a
// step, the range looked after by the weights' sum, 51.6; with the first halves cut off, not rounded,
// 0.6 less and two bits worse.)
// Tried with one FP16 number to a weight (46 us): two tiles to a CTA, sixteen softmax warps that exchange
// maxima and sums, raw tiles by bulk copies ahead of the dequantisation (each slower by 5 to 20 %);
// scores read from TMEM ahead of the exponentials of the step before (50 to 53); all dequantising warps
// on each step (47), four teams (47); a second warp for the scales (46).
#include "api.h"
#include "attention_shared.h"
#include "common.cuh"

#include <climits>
#include <cuda_bf16.h>

namespace orinfer {
namespace sp {

constexpr int TILE = 128;                        // rows of a tile: positions x query heads
constexpr int SOFTMAX_WARPS = 8, DQ_WARPS = 8, DQ_TEAMS = 2;
constexpr int MMA_WARP = SOFTMAX_WARPS + DQ_WARPS, SCALE_WARP = MMA_WARP + 1;
constexpr int THREADS = (SCALE_WARP + 1) * 32;
constexpr float LEAD = 60.f;                     // of a score above the reference, in binades

template <int D>
struct Shape {
  static constexpr int G = D / 64;               // scale groups of a key
  static constexpr int DV = D > 128 ? 128 : D;   // value channels of a CTA
  static constexpr int GV = DV / 64, PARTS = D / DV;
  static constexpr int KT = D > 128 ? 32 : 64;   // keys of a step: at most 128 score columns
  static constexpr int NB = 5;                   // buffers of keys and values
  static constexpr int QSUB = TILE * 128, KSUB = KT * 128;     // bytes of 64 channels of a tile
  static constexpr int K_BYTES = G * KSUB, V_BYTES = GV * KSUB;
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = G * QSUB;
  static constexpr int SCALE_OFF = KV_OFF + NB * (K_BYTES + V_BYTES);
  static constexpr int SCALES = KT * (G + GV) * 4;             // key and value scales
  static constexpr int STAT_OFF = SCALE_OFF + NB * SCALES;     // [sum, reference][128]
  static constexpr int ODD_OFF = STAT_OFF + 2 * TILE * 4;      // [GV] first key whose value scale is no number
  static constexpr int BAR_OFF = ODD_OFF + 16;
  static constexpr int CS = 16;                  // keys whose weights are stored at a time
  static constexpr int TOTAL = BAR_OFF + 256 + 1024;
  static constexpr int SUB = DV / 2;             // channels that a warp writes, of 32 rows: in the ring
  static_assert(SOFTMAX_WARPS * 32 * SUB * 4 <= NB * (K_BYTES + V_BYTES), "results fit the ring");
  static_assert(TOTAL <= 227 * 1024, "exceeds the shared memory of one CTA");
  static_assert(SCALES % 16 == 0, "scales are read sixteen bytes at a time");
  static_assert(GV <= G, "both halves of the weights, 16 bits each, fit the places of their scores");
};

// Rows and keys of a CTA (as many as the plan has), per KV head.
struct Item {
  int row, rows;                                 // the first row of the tile, and how many
  int step_lo, step_hi;                          // its steps of KT keys
  int shared;                                    // keys that the group shares
  int part;                                      // its part of a row's parts
  int unused[2];
};

__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t tmem_d, uint64_t adesc,
                                       uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t tmem_d, uint32_t tmem_a,
                                       uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// Sixteen TMEM lanes as the fragments of a warp's matrix product: per eight columns lane (g = lane /
// 4, t = lane % 4) holds columns 2t and 2t + 1 of rows g and g + 8.
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[16]) {       // 32 columns
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[32]) {       // 64 columns
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_frag(uint32_t taddr, uint32_t (&r)[8]) {        // 16 columns
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_frag(uint32_t taddr, const uint32_t (&r)[8]) {  // 16 columns
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x2.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
      : "memory");
}
// The same rows and columns as pairs of BF16 values, half as many columns: per four columns lane (g,
// t) holds column t of rows g and g + 8.
__device__ __forceinline__ void tmem_st_pairs(uint32_t taddr, const uint32_t (&r)[4]) { // 8 columns
  asm volatile("tcgen05.st.sync.aligned.16x128b.x2.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3])
               : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}
__device__ __forceinline__ float2 pair_at(uint32_t a, uint32_t b) {
  return make_float2(__uint_as_float(a), __uint_as_float(b));
}
// Two values as BF16 numbers and as BF16 numbers for what those leave: off by 2^-18 of them at most.
__device__ __forceinline__ void split_bf16(const float2& v, uint32_t& big, uint32_t& rest) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(v.x, v.y);
  big = *reinterpret_cast<const uint32_t*>(&b);
  float2 left;                                   // (an FP32 number less a half of a word: one instruction)
  asm("{\n\t.reg .b16 l, h, m;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "mov.b16 m, 0xbf80;\n\t"
      "fma.rn.f32.bf16 %0, l, m, %3;\n\t"
      "fma.rn.f32.bf16 %1, h, m, %4;\n\t}"
      : "=f"(left.x), "=f"(left.y)
      : "r"(big), "f"(v.x), "f"(v.y));
  const __nv_bfloat162 r = __floats2bfloat162_rn(left.x, left.y);
  rest = *reinterpret_cast<const uint32_t*>(&r);
}

// Eight INT8 values -> eight BF16 values, exactly: 0x43xx is 128 + xx for seven bits, from which 128 is
// subtracted, or 256 where the eighth is set.
__device__ __forceinline__ uint4 integers_bf16(uint32_t w0, uint32_t w1) {
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? w0 : w1, at = i % 2 ? 0x4342u : 0x4140u;
    const uint32_t low = __byte_perm(w & 0x7f7f7f7fu, 0x43434343u, at);
    const uint32_t off = __byte_perm(w & 0x80808080u, 0x43434343u, at);
    const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&low),
                                     *reinterpret_cast<const __nv_bfloat162*>(&off));
    h[i] = *reinterpret_cast<const uint32_t*>(&v);
  }
  return make_uint4(h[0], h[1], h[2], h[3]);
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

template <int D>
__global__ void __launch_bounds__(THREADS, 1) prefix_kernel(
    const __half* q, const int* row_req, const int* row_pos, const int* page_table, int slots,
    int max_pages, const int8_t* kc, const int8_t* vc, const __half* ks, const __half* vs,
    const Item* items, const int4* info, float* __restrict__ part_o, float2* __restrict__ part_ml,
    int* ready, int qh, int kvh, int rep, int num_pages, int* status) {
  using L = Shape<D>;
  constexpr int G = L::G, GV = L::GV, KT = L::KT, NB = L::NB, CS = L::CS;
  constexpr int NS = 3;                  // steps whose scores have a place
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR_OFF);
  uint64_t* kv_full = bars;              // [NB] keys, values and scales of a step are there
  uint64_t* kv_free = bars + NB;         // [NB] the last product that reads them is through
  uint64_t* s_full = bars + 2 * NB;      // [NS] scores of a step
  uint64_t* p_ready = s_full + NS;       // [NS] its weights (an arrival per softmax warp)
  uint64_t* o_done = p_ready + NS;       // [NS] the product with them is through
  uint64_t* q_full = o_done + NS;         // the query rows are there (an arrival per softmax warp)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 1);

  const int tid = threadIdx.x, warp = warp_same(tid >> 5), lane = tid & 31;
  grid_wait();
  // The row kernel runs beside this one (attn_start_beside): it is let go by grid_release, and by this
  // word it sees what lies before the wait.  So the wait comes first, in every CTA, and both behind it.
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
    asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(ready), "r"(1) : "memory");
  const Item it = items[blockIdx.x];
  const int h = blockIdx.y / L::PARTS, vpart = blockIdx.y % L::PARTS;
  int request_of_lane[TILE / 32], pos_of_lane[TILE / 32];      // of the tile's rows
#pragma unroll
  for (int i = 0; i < TILE / 32; ++i) {
    const bool there = lane + 32 * i < it.rows;
    request_of_lane[i] = there ? row_req[it.row + lane + 32 * i] : -1;
    pos_of_lane[i] = there ? row_pos[it.row + lane + 32 * i] : -1;
  }

  int* odd = reinterpret_cast<int*>(smem + L::ODD_OFF);
  if (tid == 0) {
    for (int g = 0; g < GV; ++g) odd[g] = INT_MAX;
    for (int b = 0; b < NB; ++b) {
      mbar_init(&kv_full[b], DQ_WARPS / DQ_TEAMS + 1);
      mbar_init(&kv_free[b], 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], SOFTMAX_WARPS);
      mbar_init(&o_done[i], 1);
    }
    mbar_init(q_full, SOFTMAX_WARPS);
    mbar_fence_init();
  }
  if (warp == MMA_WARP) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = warp_same(*tmem_slot);
  grid_release();
  const uint32_t tmem_o = tmem + 128 * NS;       // scores at 128 (step modulo NS)

  // The pages are read from the table row of one that sees the most of the tile's rows, and no further than
  // that: the others may end before, and their table rows may be empty from there on.
  int req = 0, last_pos = -1;
#pragma unroll
  for (int i = 0; i < TILE / 32; ++i)
    if (request_of_lane[i] >= 0 && request_of_lane[i] < slots && pos_of_lane[i] > last_pos) {
      req = request_of_lane[i];
      last_pos = pos_of_lane[i];
    }
  const int top_pos = __reduce_max_sync(0xffffffffu, last_pos);
  req = __shfl_sync(0xffffffffu, req, __ffs(__ballot_sync(0xffffffffu, last_pos == top_pos)) - 1);
  const int seen = min(it.shared, top_pos + 1);  // shared keys that some row sees
  const int step_hi = min(it.step_hi, (seen + KT - 1) / KT);
  const int steps = max(step_hi - it.step_lo, 0);
  const int* pages = page_table + static_cast<size_t>(req) * max_pages;
  // A warp's page ids, a lane each, 32 at a time: one that is fetched when it is needed holds up what
  // is asked for by it.
  const int page_lo = it.step_lo * KT >> 7, page_hi = step_hi * KT - 1 >> 7;
  auto pages_from = [&](int i) { return page_lo + i + lane <= page_hi ? pages[page_lo + i + lane] : 0; };

  if (warp == MMA_WARP) {
    // ---------------- products, issued by the whole warp (see elect_one)
    constexpr uint32_t idesc_s = umma_idesc(1, 0, 0, 0, 0, TILE, KT);
    constexpr uint32_t idesc_o = umma_idesc(1, 1, 1, 0, 1, TILE, 64);
    const uint32_t leader = elect_one();
    const uint64_t qd = umma_desc(smem_u32(smem + L::Q_OFF), 16, 1024);
    const uint64_t kd = umma_desc(smem_u32(smem + L::KV_OFF), 16, 1024);
    const uint64_t vd = umma_desc(smem_u32(smem + L::KV_OFF + L::K_BYTES), L::KSUB, 1024);
    const int last = warp_same(steps);
    bool ok = __all_sync(0xffffffffu, mbar_wait(q_full, 0, status, STATUS_MMA_WAIT, 0x300));
    auto wait_kv = [&](int s) {
      if (ok && s < last)
        ok = __all_sync(0xffffffffu, mbar_wait(&kv_full[s % NB], (s / NB) & 1, status,
                                               STATUS_MMA_WAIT, 0x400 | (s & 0xff)));
    };
    auto issue_qk = [&](int s) {
      tc_fence_after();
      if (!ok) return;
      const uint64_t kb = kd + static_cast<uint64_t>(s % NB) * ((L::K_BYTES + L::V_BYTES) / 16);
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          mma_ss(leader, tmem + 128 * (s % NS) + g * KT, qd + (g * L::QSUB + k * 32) / 16,
                 kb + (g * L::KSUB + k * 32) / 16, idesc_s, k != 0 ? 1u : 0u);
      tc_commit_by(leader, &s_full[s % NS]);
    };
    for (int s = 0; s < NS && s < last; ++s) {
      wait_kv(s);
      issue_qk(s);
    }
    for (int s = 0; s < last && ok; ++s) {
      const int b = s % NB;
      wait_kv(s + NS);                           // (ahead of the weights, which come later)
      if (!ok) break;
      ok = __all_sync(0xffffffffu, mbar_wait(&p_ready[s % NS], (s / NS) & 1, status,
                                             STATUS_MMA_WAIT, 0x500 | (s & 0xff)));
      tc_fence_after();
      if (!ok) break;
      const uint64_t vb = vd + static_cast<uint64_t>(b) * ((L::K_BYTES + L::V_BYTES) / 16);
#pragma unroll
      for (int g = 0; g < GV; ++g)
#pragma unroll
        for (int k = 0; k < KT / 16; ++k)
#pragma unroll
          for (int part = 0; part < 2; ++part)   // of the weights
            mma_ts(leader, tmem_o + g * 64,
                   tmem + 128 * (s % NS) + g * KT + part * (KT / 2) + k * 8,
                   vb + (g * L::KSUB + k * 2048) / 16, idesc_o, (s | k | part) != 0 ? 1u : 0u);
      tc_commit_by(leader, &kv_free[b]);
      tc_commit_by(leader, &o_done[s % NS]);
      if (s + NS < last) issue_qk(s + NS);       // (in the place of the weights just used)
    }
    __syncwarp();
  } else if (warp == SCALE_WARP) {
    // ---------------- scales, of keys times log2 e / sqrt(D)
    constexpr int KS = KT * G / 32, VS = KT * GV / 32;
    const float qscale = rsqrtf(static_cast<float>(D)) * 1.4426950408889634f;
    bool ok = true;
    __half kraw[KS], vraw[VS];
    int ids = pages_from(0), ids_at = 0;
    auto load = [&](int s) {
      const int key0 = (it.step_lo + s) * KT, at = (key0 >> 7) - page_lo;
      if (at >= ids_at + 32) ids = pages_from(ids_at += 32);
      int page = __shfl_sync(0xffffffffu, ids, at - ids_at);
      if (page < 0 || page >= num_pages) {
        if (lane == 0) report_status(status, STATUS_BAD_INDEX, 0x50);
        page = 0;
      }
      const size_t slot = static_cast<size_t>(page) * 128 + (key0 & 127);
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int x = lane + 32 * i;
        kraw[i] = ks[((slot + x / G) * kvh + h) * G + x % G];
      }
#pragma unroll
      for (int i = 0; i < VS; ++i) {
        const int x = lane + 32 * i;
        vraw[i] = vs[((slot + x / GV) * kvh + h) * G + vpart * GV + x % GV];
      }
    };
    if (steps > 0) load(0);
    for (int s = 0; s < steps; ++s) {
      const int b = s % NB, live = seen - (it.step_lo + s) * KT;
      if (s >= NB)
        ok = ok && mbar_wait(&kv_free[b], (s / NB - 1) & 1, status, STATUS_DECODE_WAIT, 0x600);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      float* sk = reinterpret_cast<float*>(smem + L::SCALE_OFF + b * L::SCALES);
      float* sv = sk + KT * G;
      // Slots behind the keys that are seen may never have been written: they get no scale.  Nor do values
      // whose scale is no number, or rows that do not see them would get 0 times it: those that do are
      // given theirs at the end.
#pragma unroll
      for (int i = 0; i < VS; ++i) {
        const int x = lane + 32 * i, key = x / GV;
        if ((__half_as_ushort(vraw[i]) & 0x7c00u) == 0x7c00u) {
          if (key < live) atomicMin(&odd[x % GV], (it.step_lo + s) * KT + key);
          vraw[i] = __ushort_as_half(0);
        }
      }
#pragma unroll
      for (int i = 0; i < KS; ++i) {
        const int x = lane + 32 * i, key = x / G, g = x % G;
        sk[((key >> 1) * G + g) * 2 + (key & 1)] =
            key < live ? __half2float(kraw[i]) * qscale : 0.f;
      }
#pragma unroll
      for (int i = 0; i < VS; ++i) {
        const int x = lane + 32 * i, key = x / GV, g = x % GV;
        sv[((key >> 1) * GV + g) * 2 + (key & 1)] = key < live ? __half2float(vraw[i]) : 0.f;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&kv_full[b]);
      if (s + 1 < steps) load(s + 1);
    }
  } else if (warp >= SOFTMAX_WARPS) {
    // ---------------- keys and values: INT8 from global memory (a step of the team's ahead, in
    // registers) to FP16 integers in swizzled tiles
    constexpr int DQ = DQ_WARPS / DQ_TEAMS * 32;
    constexpr int KI = KT * D / 16 / DQ, VI = KT * L::DV / 16 / DQ;
    const int u = (tid - SOFTMAX_WARPS * 32) % DQ, team = warp_same((tid - SOFTMAX_WARPS * 32) / DQ);
    uint4 kraw[KI], vraw[VI];
    int ids = pages_from(0), ids_at = 0;
    auto load = [&](int s, uint4(&kr)[KI], uint4(&vr)[VI]) {
      const int key0 = (it.step_lo + s) * KT, at = (key0 >> 7) - page_lo;
      if (at >= ids_at + 32) ids = pages_from(ids_at += 32);
      int page = __shfl_sync(0xffffffffu, ids, at - ids_at);
      if (page < 0 || page >= num_pages) page = 0;           // (the scale warp reports it)
      const size_t slot = static_cast<size_t>(page) * 128 + (key0 & 127);
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int x = u + i * DQ, key = x / (D / 16), c = x % (D / 16);
        kr[i] = *reinterpret_cast<const uint4*>(kc + ((slot + key) * kvh + h) * D + c * 16);
      }
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        const int x = u + i * DQ, key = x / (L::DV / 16), c = x % (L::DV / 16);
        vr[i] = *reinterpret_cast<const uint4*>(vc + ((slot + key) * kvh + h) * D +
                                                vpart * L::DV + c * 16);
      }
    };
    auto place = [&](unsigned char* to, const uint4& raw, int key, int c, auto integers) {
      // lanes of every other group of channels store their second half first: eight lanes that
      // store together then meet on no bank
      unsigned char* dst = to + (c / 4) * L::KSUB;
      const bool swap = c & 4;
      const uint4 lo = integers(swap ? raw.z : raw.x, swap ? raw.w : raw.y);
      const uint4 hi = integers(swap ? raw.x : raw.z, swap ? raw.y : raw.w);
      *reinterpret_cast<uint4*>(dst + swz128(key, (c % 4) * 2 + swap)) = lo;
      *reinterpret_cast<uint4*>(dst + swz128(key, (c % 4) * 2 + !swap)) = hi;
    };
    bool ok = true;
    if (team < steps) load(team, kraw, vraw);
    for (int s = team; s < steps; s += DQ_TEAMS) {
      const int b = s % NB;
      if (s >= NB)
        ok = ok && mbar_wait(&kv_free[b], (s / NB - 1) & 1, status, STATUS_DECODE_WAIT, s & 0xff);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      unsigned char* buf = smem + L::KV_OFF + b * (L::K_BYTES + L::V_BYTES);
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int x = u + i * DQ;
        place(buf, kraw[i], x / (D / 16), x % (D / 16), integers_fp16);
      }
#pragma unroll
      for (int i = 0; i < VI; ++i) {
        const int x = u + i * DQ;
        place(buf + L::K_BYTES, vraw[i], x / (L::DV / 16), x % (L::DV / 16), integers_bf16);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(&kv_full[b]);
      if (s + DQ_TEAMS < steps) load(s + DQ_TEAMS, kraw, vraw);
    }
  } else {
    // ---------------- softmax: sixteen rows per warp
    const int quad = warp & 3, half = warp >> 2;
    // ---- the query rows, 16 bytes at a time, zeros where a tile has none
    {
      const bool wide = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
      constexpr int CPR = D / 8, BATCH = D / 32; // 16-byte pieces of a row; loads in flight
      for (int i0 = tid; i0 < TILE * CPR; i0 += BATCH * SOFTMAX_WARPS * 32) {
        uint4 v[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const int i = i0 + k * SOFTMAX_WARPS * 32, qr = i / CPR, row = qr / rep;
          v[k] = make_uint4(0, 0, 0, 0);
          if (qr < TILE / rep * rep && row < it.rows) {
            const __half* from =
                q + (static_cast<size_t>(it.row + row) * qh + h * rep + qr % rep) * D + i % CPR * 8;
            if (wide) {
              v[k] = *reinterpret_cast<const uint4*>(from);
            } else {
              const unsigned short* f = reinterpret_cast<const unsigned short*>(from);
              v[k] = make_uint4(f[0] | f[1] << 16, f[2] | f[3] << 16, f[4] | f[5] << 16,
                                f[6] | f[7] << 16);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const int i = i0 + k * SOFTMAX_WARPS * 32, qr = i / CPR;
          if (qr < TILE)
            *reinterpret_cast<uint4*>(smem + L::Q_OFF + i % CPR / 8 * L::QSUB +
                                      swz128(qr, i % CPR % 8)) = v[k];
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // TMEM hands scores out as fragments: a thread holds columns 2 qt and 2 qt + 1 of every eight, of
    // rows qg and qg + 8, so that each scale that it loads serves two rows.
    const int qg = lane >> 2, qt = lane & 3;
    const int row0 = quad * 32 + half * 16;      // of the tile
    auto row_of = [&](int tr) {                  // of row `tr` of the tile, or none
      return tr < TILE / rep * rep && tr / rep < it.rows ? it.row + tr / rep : -1;
    };
    int sees[2];                                 // shared keys that its rows see
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row_of(row0 + qg + 8 * i);
      sees[i] = row < 0 ? 0 : min(seen, row_pos[row] + 1);
    }
    const int all_see = __reduce_min_sync(0xffffffffu, min(sees[0], sees[1]));
    const uint32_t lane_addr = static_cast<uint32_t>(row0) << 16;
    float m_ref[2] = {0.f, 0.f}, l_run[2] = {0.f, 0.f};
    bool ok = true;
    for (int s = 0; s < steps; ++s) {
      const int b = s % NB;
      // (the scales are the scale warp's plain stores: seen by whoever waits for them)
      ok = mbar_wait(&s_full[s % NS], (s / NS) & 1, status, STATUS_EPILOGUE_WAIT, s & 0xff) &&
           mbar_wait(&kv_full[b], (s / NB) & 1, status, STATUS_EPILOGUE_WAIT, 0x100);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t tmem_s = tmem + 128 * (s % NS) + lane_addr;
      // scales by pairs of keys and groups: those of this thread's pair `j`
      const float* sk = reinterpret_cast<const float*>(smem + L::SCALE_OFF + b * L::SCALES);
      const float* sv = sk + KT * G;
      const int key0 = (it.step_lo + s) * KT;
      // ---- scores less the reference, pair by pair of this thread's two rows
      float2 x[2][KT / 8];
      {
        uint32_t raw[G][KT / 2];
#pragma unroll
        for (int g = 0; g < G; ++g) tmem_ld_frag(tmem_s + g * KT, raw[g]);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < KT / 8; ++j) {
          const float2* w = reinterpret_cast<const float2*>(sk) + (4 * j + qt) * G;
          float2 wg[G];
          if (G == 1) {
            wg[0] = w[0];
          } else {
#pragma unroll
            for (int g = 0; g < G; g += 2) {
              const float4 v = *reinterpret_cast<const float4*>(w + g);
              wg[g] = make_float2(v.x, v.y);
              wg[(g + 1) % G] = make_float2(v.z, v.w);
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            x[i][j] = make_float2(-m_ref[i], -m_ref[i]);
#pragma unroll
            for (int g = 0; g < G; ++g)
              x[i][j] = fma2(pair_at(raw[g][4 * j + 2 * i], raw[g][4 * j + 2 * i + 1]), wg[g],
                             x[i][j]);
          }
        }
      }
      if (all_see < key0 + KT) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < KT / 8; ++j) {
            const int key = key0 + 8 * j + 2 * qt;
            if (key >= sees[i]) x[i][j].x = -INFINITY;
            if (key + 1 >= sees[i]) x[i][j].y = -INFINITY;
          }
      }
      // ---- the reference is the maximum of some step, and moves where a score is LEAD above it: weights,
      // their products with value scales and integers and a prefix's sums of them stay in FP32's range
      float top[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[i] = fmaxf(x[i][0].x, x[i][0].y);
#pragma unroll
        for (int j = 1; j < KT / 8; ++j) top[i] = max3(top[i], x[i][j].x, x[i][j].y);
      }
      if (__any_sync(0xffffffffu, s == 0 || fmaxf(top[0], top[1]) > LEAD)) {
        float corr[2];
#pragma unroll
        for (int o = 1; o < 4; o <<= 1)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // (a row that sees none of these keys stays; at first there is nothing to be lost)
          const float by = top[i] == -INFINITY ? 0.f : s == 0 ? top[i] : fmaxf(top[i], 0.f);
          corr[i] = s == 0 ? 0.f : ex2(-by);
          l_run[i] *= corr[i];
          m_ref[i] += by;
#pragma unroll
          for (int j = 0; j < KT / 8; ++j) x[i][j] = add2(x[i][j], make_float2(-by, -by));
        }
        if (s > 0) {
          // O has to stand still: the product before this one is through (the one before on its
          // barrier is, since scores that came behind that have been read)
          ok = __all_sync(0xffffffffu, mbar_wait(&o_done[(s - 1) % NS], ((s - 1) / NS) & 1, status,
                                                 STATUS_EPILOGUE_WAIT, 0x180));
          tc_fence_after();
          const uint32_t tmem_oc = tmem_o + lane_addr;
#pragma unroll
          for (int g = 0; g < GV; ++g)
#pragma unroll 1
            for (int d0 = 0; d0 < 64; d0 += 16) {
              uint32_t o[8];
              tmem_ld_frag(tmem_oc + g * 64 + d0, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i)
                o[i] = __float_as_uint(__uint_as_float(o[i]) * corr[i >> 1 & 1]);
              tmem_st_frag(tmem_oc + g * 64 + d0, o);
            }
        }
      }
      // ---- weights, times the value scales: each as a BF16 number and another for what that leaves, in
      // the place of the scores
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int c = 0; c < KT / CS; ++c) {
        uint32_t big[GV][CS / 4], rest[GV][CS / 4];
#pragma unroll
        for (int j = 0; j < CS / 8; ++j) {
          const float2* from =
              reinterpret_cast<const float2*>(sv) + (c * (CS / 2) + 4 * j + qt) * GV;
          float2 w[GV];
          if (GV == 1) {
            w[0] = from[0];
          } else {
            const float4 v = *reinterpret_cast<const float4*>(from);
            w[0] = make_float2(v.x, v.y);
            w[GV - 1] = make_float2(v.z, v.w);
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 at = x[i][c * (CS / 8) + j];
            const float2 p = make_float2(ex2(at.x), ex2(at.y));
            sum[i] = add2(sum[i], p);
#pragma unroll
            for (int g = 0; g < GV; ++g)
              split_bf16(mul2(p, w[g]), big[g][2 * j + i], rest[g][2 * j + i]);
          }
        }
#pragma unroll
        for (int g = 0; g < GV; ++g) {
          tmem_st_pairs(tmem_s + g * KT + c * (CS / 2), big[g]);
          tmem_st_pairs(tmem_s + g * KT + KT / 2 + c * (CS / 2), rest[g]);
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) l_run[i] += sum[i].x + sum[i].y;
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[s % NS]);
    }
    // ---- this part of the rows' softmax, from here on a row per lane: none where no row sees any of these
    // keys.  The ring is free when the last product is through: a warp puts 32 rows of half of the
    // channels there and writes whole lines.
    const int r = quad * 32 + lane, row = row_of(r);
    const int part = row < 0 ? -1 : info[row].y + it.part;
    ok = ok && steps > 0 && mbar_wait(&o_done[(steps - 1) % NS], ((steps - 1) / NS) & 1, status,
                         STATUS_EPILOGUE_WAIT, 0x200);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
#pragma unroll
    for (int o = 1; o < 4; o <<= 1)
#pragma unroll
      for (int i = 0; i < 2; ++i) l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], o);
    float* stat = reinterpret_cast<float*>(smem + L::STAT_OFF);
    if (qt < 2) {
      stat[row0 + qg + 8 * qt] = qt == 0 ? l_run[0] : l_run[1];
      stat[TILE + row0 + qg + 8 * qt] = qt == 0 ? m_ref[0] : m_ref[1];
    }
    asm volatile("bar.sync 1, %0;" ::"n"(SOFTMAX_WARPS * 32) : "memory");
    const size_t at = static_cast<size_t>(part) * qh + h * rep + r % rep;
    if (half == 0 && vpart == 0 && part >= 0)
      part_ml[at] = ok && stat[r] != 0.f ? make_float2(stat[TILE + r], stat[r])
                                         : make_float2(-INFINITY, 0.f);
    constexpr int SUB = L::SUB;
    const int d_lo = half * SUB;                 // this warp's channels, all of one group
    const int first_odd = odd[GV == 2 ? half : 0];
    const bool spoilt = first_odd != INT_MAX && row >= 0 && first_odd <= row_pos[row];
    auto value = [&](uint32_t v) {
      return !ok ? 0.f : spoilt ? __int_as_float(0x7fc00000) : __uint_as_float(v);
    };
    unsigned char* slab = smem + L::KV_OFF + warp * (32 * SUB * 4);
    auto cell = [](int row, int chunk) {
      return row * (SUB * 4) + (chunk ^ (row & (SUB / 4 - 1))) * 16;
    };
#pragma unroll
    for (int d0 = 0; d0 < SUB; d0 += 16) {
      uint32_t o[16];
      tmem_ld_x16(tmem_o + d_lo + d0 + (static_cast<uint32_t>(quad * 32) << 16), o);
      tc_wait_ld();
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(slab + cell(lane, (d0 + i) / 4)) =
            make_float4(value(o[i]), value(o[i + 1]), value(o[i + 2]), value(o[i + 3]));
    }
    __syncwarp();
    constexpr int CHUNKS = SUB / 4, ROWS = 32 / CHUNKS;          // rows that a warp writes at a time
#pragma unroll
    for (int i = 0; i < 32 / ROWS; ++i) {
      const int from = i * ROWS + lane / CHUNKS;
      const size_t to = __shfl_sync(0xffffffffu, static_cast<unsigned long long>(at), from);
      if (__shfl_sync(0xffffffffu, part, from) >= 0)
        *reinterpret_cast<float4*>(part_o + to * D + vpart * L::DV + d_lo + lane % CHUNKS * 4) =
            *reinterpret_cast<const float4*>(slab + cell(from, lane % CHUNKS));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) tmem_dealloc(tmem, 512);
}

template <int D>
static int launch_prefix(const __half* q, const int* row_req, const int* row_pos,
                         const int* page_table, int slots, int max_pages, const int8_t* kc,
                         const int8_t* vc, const __half* ks, const __half* vs, const Item* items,
                         int n_items, const SharedParts& parts, int qh, int kvh, int num_pages,
                         cudaStream_t stream) {
  using L = Shape<D>;
  static const int slot = runtime_new_slot();
  if (const int e = runtime_allow_smem(slot, prefix_kernel<D>, L::TOTAL)) return e;
  launch_early(prefix_kernel<D>, dim3(n_items, kvh * L::PARTS), THREADS, L::TOTAL, stream, q,
               row_req, row_pos, page_table, slots, max_pages, kc, vc, ks, vs, items, parts.rows,
               const_cast<float*>(parts.o), const_cast<float2*>(parts.ml), parts.ready, qh, kvh,
               qh / kvh, num_pages, runtime_status_ptr());
  return static_cast<int>(cudaGetLastError());
}

}  // namespace sp
}  // namespace orinfer

using namespace orinfer;

// Keys of a step, and rows of a tile: what a plan's items are counted in.
extern "C" int orinfer_shared_step(int head_dim) { return head_dim > 128 ? 32 : 64; }

// items: int32 [n_items, 8], see Item; rows_info: int32 [rows, 4] = (shared keys, first part, parts,
// 0); parts: FP32 [all parts, query heads, D], behind it [all parts, query heads, 2] and a word that is 0
// before the first call; scratch: for splits > 1, orinfer_attention_scratch_bytes.
extern "C" int orinfer_attention_shared(
    const __half* q, const __half* gate, const int* row_req, const int* row_pos,
    const int* page_table, int slots, int max_pages, const int8_t* kc, const int8_t* vc,
    const __half* ks, const __half* vs, __half* out, int rows, int qh, int kvh, int head_dim,
    int num_pages, const int* items, int n_items, const int* rows_info, float* parts, int n_parts,
    int splits, float* scratch, int context, cudaStream_t stream) {
  if (rows <= 0) return 0;
  if (kvh <= 0 || qh % kvh || max_pages <= 0 || num_pages <= 0 || slots <= 0) return -1;
  if (n_items < 0 || n_parts < 0 || (n_items > 0 && (!items || !parts)) || !rows_info) return -1;
  if (splits < 1 || (splits > 1 && !scratch)) return -1;
  if (((reinterpret_cast<uintptr_t>(kc) | reinterpret_cast<uintptr_t>(vc) |
        reinterpret_cast<uintptr_t>(parts)) & 15) != 0)
    return -1;
  const int rep = qh / kvh;
  if (rep != 1 && rep != 2 && rep != 4 && rep != 8 && !(rep == 5 && head_dim == 128)) return -1;
  if (runtime_ensure_init() != cudaSuccess) return -2;
  SharedParts shared;
  shared.pending = n_items > 0;
  shared.rows = reinterpret_cast<const int4*>(rows_info);
  shared.o = parts;
  const size_t cells = static_cast<size_t>(n_parts) * qh;
  shared.ml = reinterpret_cast<const float2*>(parts + cells * head_dim);
  shared.ready = reinterpret_cast<int*>(parts + cells * (head_dim + 2));
  const sp::Item* list = reinterpret_cast<const sp::Item*>(items);
  if (n_items > 0) {
    int e = -1;
#define CASE(D)                                                                                  \
  if (head_dim == D)                                                                             \
    e = sp::launch_prefix<D>(q, row_req, row_pos, page_table, slots, max_pages, kc, vc, ks, vs,  \
                             list, n_items, shared, qh, kvh, num_pages, stream);
    CASE(64) CASE(128) CASE(256)
#undef CASE
    if (e != 0) return e;
  }
  return attention_own_keys(q, gate, row_req, row_pos, page_table, max_pages, kc, vc, ks, vs, out,
                            rows, qh, kvh, head_dim, splits, scratch, context, shared, stream);
}
