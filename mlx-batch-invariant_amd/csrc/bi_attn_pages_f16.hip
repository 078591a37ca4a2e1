// bi_attn_pages_f16.hip — attention over quantized pages and shared prefixes, f16, head dims to 128.
#include "bi_attn_pages_launch.h"

namespace bi {
BI_PAGES_INSTANTIATE(f16, 32)
BI_PAGES_INSTANTIATE(f16, 64)
BI_PAGES_INSTANTIATE(f16, 96)
BI_PAGES_INSTANTIATE(f16, 128)
}
