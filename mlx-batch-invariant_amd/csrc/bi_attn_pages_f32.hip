// bi_attn_pages_f32.hip — attention over quantized pages and shared prefixes, fp32, head dims to 128.
#include "bi_attn_pages_launch.h"

namespace bi {
BI_PAGES_INSTANTIATE(float, 32)
BI_PAGES_INSTANTIATE(float, 64)
BI_PAGES_INSTANTIATE(float, 96)
BI_PAGES_INSTANTIATE(float, 128)
}
