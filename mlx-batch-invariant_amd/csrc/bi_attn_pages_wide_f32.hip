// bi_attn_pages_wide_f32.hip — attention over quantized pages and shared prefixes, fp32, head dims 192 and 256.
#include "bi_attn_pages_launch.h"

namespace bi {
BI_PAGES_INSTANTIATE(float, 192)
BI_PAGES_INSTANTIATE(float, 256)
}
