// bi_attn_mod_rows_f16.hip — attention of few rows with ScoreMod for f16 elements, every head dim.
#include "bi_attn_mod_launch.h"

namespace bi {
BI_ATTN_MOD_D(BI_ATTN_MOD_ROWS, f16)
}  // namespace bi
