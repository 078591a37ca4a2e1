// bi_attn_mod_cap_f16.hip — prefill attention with ScoreMod for f16 elements: capped scores.
#include "bi_attn_mod_launch.h"

namespace bi {
#define BI_MOD(T, D) template int launch_prefill_mod<T, D, (kModAny | kModCap)>(ModPrefillArgs&, hipStream_t);
BI_ATTN_MOD_D(BI_MOD, f16)
}  // namespace bi
