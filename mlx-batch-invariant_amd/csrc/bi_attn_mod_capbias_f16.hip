// bi_attn_mod_capbias_f16.hip — prefill attention with ScoreMod for f16 elements: capped scores and a distance bias.
#include "bi_attn_mod_launch.h"

namespace bi {
#define BI_MOD(T, D) template int launch_prefill_mod<T, D, (kModAny | kModCap | kModBias)>(ModPrefillArgs&, hipStream_t);
BI_ATTN_MOD_D(BI_MOD, f16)
}  // namespace bi
