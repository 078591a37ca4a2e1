// bi_attn_pages_f16.hip — attention over quantized pages and shared prefixes, f16.
#include "bi_attn_pages_launch.h"

namespace bi {
BI_PAGES_INSTANTIATE(f16)
}
