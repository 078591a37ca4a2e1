// bi_attn_api.h — the attention launchers the C ABI calls, one instantiation
// per (element type, head dim) in bi_attn_{bf16,f16,f32}.hip.
#pragma once

#include <algorithm>

#include "bi_attn_common.h"

namespace bi {

// Query heads of one kv head that a decode work item scores together (the
// columns of its score tile): the largest of 16, 8, 4, 2, 1 dividing G.
inline int decode_gu(int G) {
  for (int gu : {16, 8, 4, 2, 1})
    if (G % gu == 0) return gu;
  return 1;
}

// Queries per per-key prefill unit: 4 up to D = 128, 2 up to 256, else 1 (a
// unit's rows and accumulators grow with D). A query's arithmetic does not
// depend on it (a query takes only its own keys and splits); the K / V rows
// of a key block are loaded and converted once for the unit's queries.
__host__ __device__ constexpr int pk_prefill_qb(int64_t D) { return D <= 128 ? 4 : D <= 256 ? 2 : 1; }

// Query heads a per-key decode unit scores together: 4, 2 or 1 (dividing G), and 1
// while the grid has fewer than 16384 (head, split) pairs, where every unit
// is wanted for parallelism.
inline int perkey_decode_nq(int64_t B, int Hq, int Hkv, int nsplit) {
  const int G = Hq / Hkv;
  if ((int64_t)B * Hq * nsplit < 16384) return 1;
  return G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1;
}

template <typename T, int D>
int launch_decode(DecodeArgs& a, hipStream_t st);
template <typename T, int D>
int launch_prefill(PrefillArgs& a, hipStream_t st);
// The same with ScoreMod (bi_attn_mod_{decode,mask,cap,bias,capbias,rows}_{bf16,f16,f32}.hip).
template <typename T, int D>
int launch_decode_mod(ModDecodeArgs& a, hipStream_t st);
template <typename T, int D, int MOD>
int launch_prefill_mod(ModPrefillArgs& a, hipStream_t st);
template <typename T, int D>
int launch_rows_mod(ModRowsArgs& a, hipStream_t st);

// Bytes of the partials (m, l, acc) of every row and split of a chunk of Tq tokens.
inline int64_t rows_partial_bytes(int64_t B, int64_t Hq, int64_t Tq, int64_t L, int64_t D) {
  const int64_t n = B * Hq * Tq * ((L + kSplit - 1) / kSplit);
  return ((n + 3) / 4 * 4 * 2 + n * D) * (int64_t)sizeof(float);
}
// Whether attn_rows_mod takes a chunk (a workgroup per split and 16 rows) or
// attn_prefill_mod (one that walks the splits of 64 rows). Walking costs the
// longest row's splits, whatever the rows, while these leave CUs idle; per split
// and 16 rows K and V come from the cache again. With R the 16-row chunks, less
// the half that a causal chunk's own triangle leaves out, and N the splits (us, walk
// / split; the turn moves up with N, as a second launch merges, and N = 1 walks):
// bf16, 32 / 8 heads of 128: R = 185, N = 3: 20.0 / 23.4; R = 190, N = 7: 43 / 40; R
// = 191, N = 16: 101 / 79; R = 246, N = 7: 45 / 52; R = 253, N = 17: 102 / 107; 14 / 2
// heads of 64: R = 216, N = 7: 32 / 31; R = 335, N = 18: 80 / 86. fp32, whose walk has
// no pipeline, 8 / 8 heads of 128: R = 426, N = 3: 102 / 79; R = 569, N = 18: 615 /
// 454; 32 / 8: R = 623, N = 4: 124 / 131; heads of 32 to 192 turn alike (192: R = 460,
// N = 3: 114 / 108; R = 623: 184 / 189), of 256, where the walk spills 554 registers
// and more, later: R = 885,
// N = 5: 841 / 529. The partials stay below 256 MB. N is what the cache can hold (the
// host does not know the lengths): a workgroup without keys costs 1.1 ns, so 300 keys
// in a table of 32768 take 39 us where walking takes 21 (R = 128), and 32768 keys 380
// where walking takes some 1000.
inline bool few_rows(int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t L, int64_t D, int causal, int dtype) {
  if ((double)Tq * Hq * B > 1e9) return false;           // (so that the products below stay in 64 bits)
  const int64_t n = (L + kSplit - 1) / kSplit;
  const int64_t chunks = (Tq * (Hq / Hkv) + 15) / 16 * Hkv * B;
  const int64_t r = causal ? chunks - chunks * std::min(Tq, L) / (2 * L) : chunks;
  const int64_t most = dtype != BI_F32 ? 250 - 250 / n : D > 192 ? 1200 : 580 - 300 / n;
  return r <= most && rows_partial_bytes(B, Hq, Tq, L, D) <= ((int64_t)256 << 20);
}
// The reference's per-key order on the vector ALUs (bi_attn_perkey.h).
template <typename T, int D>
int launch_decode_perkey(DecodeArgs& a, hipStream_t st);
template <typename T, int D>
int launch_prefill_perkey(PrefillArgs& a, hipStream_t st);

}  // namespace bi
