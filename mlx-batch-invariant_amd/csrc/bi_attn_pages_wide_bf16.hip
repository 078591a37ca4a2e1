// bi_attn_pages_wide_bf16.hip — attention over quantized pages and shared prefixes, bf16, head dims 192 and 256.
#include "bi_attn_pages_launch.h"

namespace bi {
BI_PAGES_INSTANTIATE(bf16, 192)
BI_PAGES_INSTANTIATE(bf16, 256)
}
