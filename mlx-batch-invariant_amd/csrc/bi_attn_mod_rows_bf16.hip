// bi_attn_mod_rows_bf16.hip — attention of few rows with ScoreMod for bf16 elements, every head dim.
#include "bi_attn_mod_launch.h"

namespace bi {
BI_ATTN_MOD_D(BI_ATTN_MOD_ROWS, bf16)
}  // namespace bi
