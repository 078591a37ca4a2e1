// bi_attn_pages_launch.h — host launcher of the kernels of bi_attn_pages.h, included by
// bi_attn_pages_{bf16,f16,f32}.hip, which instantiate it for every head dim.
#pragma once

#include "bi_attn_launch.h"
#include "bi_attn_pages.h"

namespace bi {

template <typename T, int D, int BITS, bool MULTI>
static int launch_pages_as(const PagesArgs& a, hipStream_t st) {
  static int cache[kMaxDev] = {};
  int grid = resident_grid(attn_pages<T, D, BITS, MULTI>, cache);
  if (grid <= 0) return bi_host::fail(BI_E_UNSUPPORTED, "bi_attn_pages: device occupancy query failed");
  if constexpr (MULTI) pages_plan_kernel<<<1, kPlanThreads, 0, st>>>(a, grid);
  const int64_t most = (int64_t)a.B * a.nsplit * a.Hkv * ((a.Tq * (a.Hq / a.Hkv) + 15) / 16);   // no segment has more
  grid = (int)((std::min<int64_t>(grid, most) + 7) / 8 * 8);
  attn_pages<T, D, BITS, MULTI><<<grid, 256, 0, st>>>(a);
  if (a.nsplit > 1) {
    const int64_t n = (int64_t)a.B * a.Hq * a.Tq * (D / 4);
    attn_pages_merge<T, D><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a);
  }
  return bi_host::launch_status("bi_attn_pages");
}

template <typename T, int D>
int launch_pages(const PagesArgs& a, int bits, hipStream_t st) {
  const bool multi = a.groups > 0 || a.Tq * (a.Hq / a.Hkv) > 16;
  if (bits == 0) return launch_pages_as<T, D, 0, true>(a, st);
  if (bits == 8) return multi ? launch_pages_as<T, D, 8, true>(a, st) : launch_pages_as<T, D, 8, false>(a, st);
  return multi ? launch_pages_as<T, D, 4, true>(a, st) : launch_pages_as<T, D, 4, false>(a, st);
}

#define BI_PAGES_INSTANTIATE(T)                                                   \
  template int launch_pages<T, 32>(const PagesArgs&, int, hipStream_t);           \
  template int launch_pages<T, 64>(const PagesArgs&, int, hipStream_t);           \
  template int launch_pages<T, 96>(const PagesArgs&, int, hipStream_t);           \
  template int launch_pages<T, 128>(const PagesArgs&, int, hipStream_t);          \
  template int launch_pages<T, 192>(const PagesArgs&, int, hipStream_t);          \
  template int launch_pages<T, 256>(const PagesArgs&, int, hipStream_t);

}  // namespace bi
