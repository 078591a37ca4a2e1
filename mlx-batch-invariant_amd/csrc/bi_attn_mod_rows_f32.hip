// bi_attn_mod_rows_f32.hip — attention of few rows with ScoreMod for f32 elements, every head dim.
#include "bi_attn_mod_launch.h"

namespace bi {
BI_ATTN_MOD_D(BI_ATTN_MOD_ROWS, float)
}  // namespace bi
