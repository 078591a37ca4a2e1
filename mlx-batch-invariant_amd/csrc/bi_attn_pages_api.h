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
  int slots;                             // workgroups of attn_pages that the device holds at once
  int near;                              // codes: every byte of the pools lies below 2^32 from their start
  unsigned hkv_inv, rows1_inv, g_inv;    // inverse() of Hkv, of Tq G (rows of a sequence and kv head) and of G
  float scale_log2;
};

__device__ __forceinline__ int pages_len(const PagesArgs& a, int b) {
  return a.kv_lens ? min(max(a.kv_lens[b], 0), a.L) : a.L;
}

__device__ __forceinline__ int plan_start(const PagesArgs& a, int n) {
  return a.starts ? min(max(a.starts[n], 0), a.B) : n ? a.B : 0;
}

// 2^32 / d, rounded down (2^32 - 1 for 1): quotients by one product and a correction.
inline unsigned inverse(int64_t d) { return d == 1 ? 0xffffffffu : (unsigned)(((int64_t)1 << 32) / d); }

constexpr int kPlanWords = 5;            // of a segment in the plan
constexpr int kPlanFused = 192;          // segments of a plan that every workgroup makes for itself (3.75 KB of LDS: with 5 KB three
                                         // workgroups of 64 dims would not fit a CU, 46 instead of 41 us for 64 sequences behind 8192 keys)

template <typename T, int D>
int launch_pages(const PagesArgs& a, int bits, hipStream_t st);

// Whether a call goes to the kernels of few rows (a workgroup per split, partials merged
// by a last launch), or to those of bi_attn_scored, which score a sequence's rows 64
// at a time over all keys and know neither codes nor shared prefixes (bi_attn_pages
// reads codes back and finds the shared pages for them). Besides single
// tokens and what few_rows splits anyway (32/8 heads of 128, 2648 keys, 2048 of them
// shared in 4 groups, us here and there):
//  - codes of up to 64 rows a sequence and kv head, as reading them back costs more:
//    32 sequences of 1, 2, 4 chunks of 16 rows 65 / 199, 125 / 196, 191 / 189, 4 sequences
//    24 / 45, 45 / 50, 55 / 62; of 8 chunks 300 / 210 and 78 / 84;
//  - one chunk of 16-bit rows, where the prefix is read four times less often and
//    sequences are not so few that the others would split their keys too: 32 sequences
//    67 / 91, 16 in 4 groups 47 / 53, 8 in 2 groups 41 / 37; of 2 chunks 101 / 90.
//    (fp32: 158 / 147.)
// It holds for other heads and lengths: codes of 14 / 2 heads of 64, 4000 keys, 56 rows, 32
// sequences 31 / 69; 8 / 8 of 128, 4000 keys, 16 sequences, 32 rows 45 / 124, 64 rows 62 / 118; 32 / 8
// of 128, 32768 keys, 16 sequences, 32 rows 239 / 1022; 16-bit rows of 16, 32 sequences in 4 groups
// behind 256 keys 28 / 38 and behind 8192 100 / 264, 8 / 8 heads behind 2048 43 / 90; of 64 rows, 64
// sequences in one group behind 8192, 620 / 289.
inline bool pages_few_rows(int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t L, int64_t D, int64_t groups, int bits,
                           int causal, int dtype) {
  if (Tq == 1 || few_rows(B, Hq, Hkv, Tq, L, D, causal, dtype)) return true;
  const int64_t G = Hq / Hkv;
  if (Tq > 64 || Tq * G > 64 || (double)B * Hq > 1e9 || rows_partial_bytes(B, Hq, Tq, L, D) > ((int64_t)2 << 30)) return false;
  if (bits) return true;
  return groups > 0 && dtype != BI_F32 && Tq * G <= 16 && B >= 4 * groups && B * Hkv >= 128;
}

}  // namespace bi
