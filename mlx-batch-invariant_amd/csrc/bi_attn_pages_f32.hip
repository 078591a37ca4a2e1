// bi_attn_pages_f32.hip — attention over quantized pages and shared prefixes, fp32.
#include "bi_attn_pages_launch.h"

namespace bi {
BI_PAGES_INSTANTIATE(float)
}
