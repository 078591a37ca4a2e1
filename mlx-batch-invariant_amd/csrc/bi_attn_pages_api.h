// bi_attn_pages_api.h — arguments and launchers of bi_attn_pages.h's kernels for the
// C ABI, instantiated in bi_attn_pages_{bf16,f16,f32}.hip.
#pragma once

#include "bi_attn_api.h"

namespace bi {

struct PagesArgs {
  const void *q, *k, *v, *kg, *vg;       // kg, vg: (scale, bias) of every group of codes
  const int32_t *kv_lens, *table, *starts, *slens;
  float *pm, *pl, *pacc;                 // partials of every (sequence, head, token) row and split
  int32_t* plan;                         // pages_plan_kernel's
  void* out;
  int64_t q_sb, q_sh, q_st, k_sp, k_sh, k_sl, v_sp, v_sh, v_sl;  // codes: bytes
  int64_t kg_sp, kg_sh, kg_sl, vg_sp, vg_sh, vg_sl, table_stride;
  int B, Hq, Hkv, Tq, L, nsplit, causal, groups, shared_len, page_shift, num_pages, gshift;
  int near;                              // codes: every byte of the pools lies below 2^32 from their start
  unsigned hkv_inv, rows1_inv, g_inv;    // inverse() of Hkv, of Tq G (rows of a sequence and kv head) and of G
  float scale_log2;
};

// 2^32 / d, rounded down (2^32 - 1 for 1): quotients by one product and a correction.
inline unsigned inverse(int64_t d) { return d == 1 ? 0xffffffffu : (unsigned)(((int64_t)1 << 32) / d); }

constexpr int kPlanWords = 5;            // of a segment in the plan

template <typename T, int D>
int launch_pages(const PagesArgs& a, int bits, hipStream_t st);

// Whether attn_pages takes a call (a workgroup per split, partials merged by a second
// launch), or the kernels of bi_attn_scored.
inline bool pages_few_rows(int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t L, int64_t D, int64_t groups, int bits,
                           int causal, int dtype) {
  return Tq == 1 || few_rows(B, Hq, Hkv, Tq, L, D, causal, dtype);
}

}  // namespace bi
