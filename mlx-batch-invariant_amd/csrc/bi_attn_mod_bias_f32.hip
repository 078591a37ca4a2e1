// bi_attn_mod_bias_f32.hip — prefill attention with ScoreMod for f32 elements: a distance bias.
#include "bi_attn_mod_launch.h"

namespace bi {
#define BI_MOD(T, D) template int launch_prefill_mod<T, D, (kModAny | kModBias)>(ModPrefillArgs&, hipStream_t);
BI_ATTN_MOD_D(BI_MOD, float)
}  // namespace bi
