// bi_attn_pages_bf16.hip — attention over quantized pages and shared prefixes, bf16.
#include "bi_attn_pages_launch.h"

namespace bi {
BI_PAGES_INSTANTIATE(bf16)
}
