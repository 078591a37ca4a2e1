// bi_attn_pages_launch.h — host launcher of the kernels of bi_attn_pages.h, included by
// bi_attn_pages_{bf16,f16,f32}.hip (head dims to 128) and bi_attn_pages_wide_{...}.hip
// (192 and 256, whose registers go by other rules: see build.py).
#pragma once

#include "bi_attn_launch.h"
#include "bi_attn_pages.h"

namespace bi {

// Workgroups of a kernel with `lds` bytes of dynamic LDS that the device holds at once,
// a multiple of 8 (one share for each XCD), and no more than there can be items.
template <typename K>
static int pages_grid(K kern, size_t lds, int (&cache)[kMaxDev], int64_t most) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDev) return 0;
  if (cache[dev] <= 0) {                                  // (every writer stores the same value)
    int cus = 0, per_cu = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
        hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kern, 256, lds) != hipSuccess || cus <= 0 || per_cu <= 0)
      return 0;
    cache[dev] = cus * per_cu;
  }
  return (int)((std::min<int64_t>(cache[dev], most) + 7) / 8 * 8);
}

template <typename T, int D>
static int merge_pages(const PagesArgs& a, hipStream_t st) {
  if (a.nsplit > 1) {
    const int64_t n = (int64_t)a.B * a.Hq * a.Tq * MergeRow<D>::kLanes;
    attn_pages_merge<T, D><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a);
  }
  return bi_host::launch_status("bi_attn_pages");
}

constexpr const char* kNoOccupancy = "bi_attn_pages: device occupancy query failed";

template <typename T, int D, int BITS>
static int launch_planned(PagesArgs a, hipStream_t st) {
  static int cache[2][kMaxDev] = {};
  const int64_t most = (int64_t)a.B * a.nsplit * a.Hkv * ((a.Tq * (a.Hq / a.Hkv) + 15) / 16);   // no segment has more
  const int many = a.groups + a.B > kPlanFused;
  const size_t lds = (many ? kPlanCached : kPlanFused * kPlanWords) * sizeof(int);
  a.slots = pages_grid(attn_pages<T, D, BITS>, lds, cache[many], (int64_t)1 << 30);
  if (a.slots <= 0) return bi_host::fail(BI_E_UNSUPPORTED, kNoOccupancy);
  if (many) pages_plan_kernel<<<1, kPlanThreads, 0, st>>>(a);
  attn_pages<T, D, BITS><<<pages_grid(attn_pages<T, D, BITS>, lds, cache[many], most), 256, lds, st>>>(a);
  return merge_pages<T, D>(a, st);
}

template <typename T, int D, int BITS, int GS>
static int launch_codes_as(const PagesArgs& a, hipStream_t st) {
  static int cache[3][kMaxDev] = {};
  const int rc = codes_rows(a.Tq * (a.Hq / a.Hkv));
  const size_t lds = (size_t)rc * 4 * 2 * (kSplit / 32) * sizeof(u32x4);
  const int grid = pages_grid(attn_codes<T, D, BITS, GS>, lds, cache[rc / 8], (int64_t)a.B * a.nsplit * a.Hkv);
  if (grid <= 0) return bi_host::fail(BI_E_UNSUPPORTED, kNoOccupancy);
  attn_codes<T, D, BITS, GS><<<grid, 256, lds, st>>>(a);
  return merge_pages<T, D>(a, st);
}
template <typename T, int D, int BITS>
static int launch_codes(const PagesArgs& a, hipStream_t st) {
  if constexpr (D % 64 == 0)
    if (a.gshift == 6) return launch_codes_as<T, D, BITS, 64>(a, st);
  if constexpr (D % 128 == 0)
    if (a.gshift == 7) return launch_codes_as<T, D, BITS, 128>(a, st);
  return launch_codes_as<T, D, BITS, 32>(a, st);
}

template <typename T, int D>
int launch_pages(const PagesArgs& a, int bits, hipStream_t st) {
  if (bits == 0) return launch_planned<T, D, 0>(a, st);
  if (a.groups == 0 && a.Tq * (a.Hq / a.Hkv) <= 16)
    return bits == 8 ? launch_codes<T, D, 8>(a, st) : launch_codes<T, D, 4>(a, st);
  return bits == 8 ? launch_planned<T, D, 8>(a, st) : launch_planned<T, D, 4>(a, st);
}

#define BI_PAGES_INSTANTIATE(T, D) template int launch_pages<T, D>(const PagesArgs&, int, hipStream_t);

}  // namespace bi
