// bi_attn_mod_decode_f32.hip — decode attention with ScoreMod for f32 elements, every head dim.
#include "bi_attn_mod_launch.h"

namespace bi {
BI_ATTN_MOD_D(BI_ATTN_MOD_DECODE, float)
}  // namespace bi
