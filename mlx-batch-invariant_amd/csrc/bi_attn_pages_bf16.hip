// bi_attn_pages_bf16.hip — attention over quantized pages and shared prefixes, bf16, head dims to 128.
#include "bi_attn_pages_launch.h"

namespace bi {
BI_PAGES_INSTANTIATE(bf16, 32)
BI_PAGES_INSTANTIATE(bf16, 64)
BI_PAGES_INSTANTIATE(bf16, 96)
BI_PAGES_INSTANTIATE(bf16, 128)
}
