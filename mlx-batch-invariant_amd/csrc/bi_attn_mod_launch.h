// bi_attn_mod_launch.h — host launchers of the attention kernels with ScoreMod
// (capped scores, distance bias, document and prefix masks), included by the
// translation units bi_attn_mod_*.hip, which instantiate them per element type
// and score variant. Kernels: bi_attn_mfma.h (decode), bi_attn_mod.h (prefill).
#pragma once

#include "bi_attn_launch.h"
#include "bi_attn_mod.h"

namespace bi {

// attn_combine_kernel, but a split without a visible key (l = 0 at m = -inf) is
// not merged: its m would make the factors NaN; one at m = NaN has no acc. (A split
// whose scores are all NaN has l = NaN and is merged.) A sum that is not finite has
// its thread look through the V column for infinities and NaN that the query sees.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_combine_mod_kernel(ModDecodeArgs a) {
  const int64_t gid0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const bool live = gid0 < (int64_t)a.B * a.Hq * D;
  const int64_t gid = live ? gid0 : 0;
  const int64_t bh = gid / D;
  const int d = (int)(gid % D), b = (int)(bh / a.Hq);
  const int len = a.kv_lens ? min(max(a.kv_lens[b], 0), a.L) : a.L;
  const int ns = (len + kSplit - 1) / kSplit;
  float M = -INFINITY, Ls = 0.0f, A = 0.0f;
  bool look = false;                                    // a split passed over has an acc that is not finite
  auto merge = [&](float m, float l, float acc) {
    // (merge_split's operations, without a branch: a split passed over multiplies
    // by 1 and adds -0; its acc may be unwritten)
    const bool sees = m > -INFINITY || l != 0.0f;
    const float top = sees ? fmaxf(M, m) : M;
    const float c_old = sees ? __builtin_amdgcn_exp2f(M - top) : 1.0f;
    const float c_new = sees ? __builtin_amdgcn_exp2f(m - top) : -0.0f;
    Ls = __builtin_fmaf(Ls, c_old, l * c_new);
    A = __builtin_fmaf(A, c_old, sees ? acc * c_new : -0.0f);
    M = top;
  };
  auto passed_over = [](float m, float l, float acc) { return m == -INFINITY && l == 0.0f && v_kind(acc) != 0u; };
  int i = 0;
  for (; i + 8 <= ns; i += 8) {                         // partials loaded eight splits ahead, merged in order
    float pm[8], pl[8], pa[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int64_t po = bh * a.nsplit + i + j;
      pm[j] = a.pm[po];
      pl[j] = a.pl[po];
      pa[j] = a.pacc[po * D + d];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) merge(pm[j], pl[j], pa[j]);
    const float any = ((pa[0] + pa[1]) + (pa[2] + pa[3])) + ((pa[4] + pa[5]) + (pa[6] + pa[7]));
    if (!(fabsf(any) < INFINITY)) {
#pragma unroll
      for (int j = 0; j < 8; ++j) look = look || passed_over(pm[j], pl[j], pa[j]);
    }
  }
  for (; i < ns; ++i) {
    const int64_t po = bh * a.nsplit + i;
    const float m = a.pm[po], l = a.pl[po], acc = a.pacc[po * D + d];
    merge(m, l, acc);
    look = look || passed_over(m, l, acc);
  }
  float x = Ls != 0.0f ? A / Ls : 0.0f;
  if (live && Ls > 0.0f && (look || !(fabsf(x) < INFINITY))) {  // (l NaN: NaN, whatever V holds)
    const int32_t* docs = a.mod.docs ? a.mod.docs + (int64_t)b * a.mod.docs_sb : nullptr;
    const int hk = (int)(bh % a.Hq) / (a.Hq / a.Hkv);
    const T* v = static_cast<const T*>(a.v) + d;
    uint32_t kinds = 0;
    for (int key = 0; key < len; ++key)
      if (!docs || docs[key] == docs[len - 1])
        kinds |= v_kind(to_f32(v[kv_row_off(a, a.v_sb, a.v_sh, a.v_sl, b, hk, key)]));
    if (kinds) x = seen_value(kinds, Ls);
  }
  if (live) static_cast<T*>(a.out)[bh * D + d] = to_store<T>(x);
}

// One instantiation for both item orders, chosen as for the plain kernel: with at
// most kDynMinRounds rounds of the resident grid the static order, which needs no
// launch to zero a counter.
template <typename T, int D, int GU, int MODE>
static int launch_decode_mod_gu(ModDecodeArgs& a, hipStream_t st) {
  static int cache[kMaxDev] = {};
  const int64_t most = (int64_t)a.B * a.nsplit * a.Hkv * a.nchunk;
  const int grid = resident_grid(attn_decode_mfma<T, D, GU, true, MODE, kModAny>, cache);
  if (grid <= 0) return bi_host::fail(BI_E_UNSUPPORTED, "bi_attn_scored: device occupancy query failed");
  if (most > (int64_t)kDynMinRounds * grid) zero_counter_kernel<<<1, 1, 0, st>>>(a.ctr);
  else a.ctr = nullptr;
  attn_decode_mfma<T, D, GU, true, MODE, kModAny><<<(int)std::min<int64_t>(grid, most), 256, 0, st>>>(a);
  return 0;
}

template <typename T, int D, int GU>
static int launch_decode_mod_mode(ModDecodeArgs& a, hipStream_t st) {
  switch (kv_mode<T>(a)) {
    case kKvPaged: return launch_decode_mod_gu<T, D, GU, kKvPaged>(a, st);
    case kKvTilePaged: return launch_decode_mod_gu<T, D, GU, kKvTilePaged>(a, st);
    case kKvRowPaged: return launch_decode_mod_gu<T, D, GU, kKvRowPaged>(a, st);
    default: return launch_decode_mod_gu<T, D, GU, kKvContig>(a, st);
  }
}

template <typename T, int D>
int launch_decode_mod(ModDecodeArgs& a, hipStream_t st) {
  int rc = 0;
  switch (a.GU) {
    case 16: rc = launch_decode_mod_mode<T, D, 16>(a, st); break;
    case 8: rc = launch_decode_mod_mode<T, D, 8>(a, st); break;
    case 4: rc = launch_decode_mod_mode<T, D, 4>(a, st); break;
    case 2: rc = launch_decode_mod_mode<T, D, 2>(a, st); break;
    default: rc = launch_decode_mod_mode<T, D, 1>(a, st); break;
  }
  if (rc) return rc;
  if ((rc = bi_host::launch_status("bi_attn_scored")) || a.nsplit == 1) return rc;
  const int64_t n = (int64_t)a.B * a.Hq * D;
  attn_combine_mod_kernel<T, D><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a);
  return bi_host::launch_status("bi_attn_scored(combine)");
}

// Smallest and largest document number of each split's keys below the sequence's
// length: one wave per split.
static __global__ __launch_bounds__(64) void doc_ranges_kernel(const int32_t* __restrict__ docs, int64_t docs_sb,
                                                               const int32_t* kv_lens, int L, int nsplit,
                                                               int2* ranges) {
  const int b = blockIdx.x / nsplit, sp = blockIdx.x % nsplit;
  const int len = kv_lens ? min(max(kv_lens[b], 0), L) : L;
  int lo = 0x7fffffff, hi = -0x7fffffff - 1;
#pragma unroll
  for (int j = 0; j < kSplit / 64; ++j) {
    const int key = kSplit * sp + 64 * j + (int)threadIdx.x;
    if (key < len) {
      const int d = docs[b * docs_sb + key];
      lo = min(lo, d);
      hi = max(hi, d);
    }
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) {
    lo = min(lo, __shfl_xor(lo, off, kWave));
    hi = max(hi, __shfl_xor(hi, off, kWave));
  }
  if (threadIdx.x == 0) ranges[blockIdx.x] = int2{lo, hi};
}

template <typename T, int D, int MOD>
int launch_prefill_mod(ModPrefillArgs& a, hipStream_t st) {
  const int64_t wgs = ((int64_t)a.Tq * (a.Hq / a.Hkv) + 63) / 64;
  const int64_t items = wgs * a.Hkv * a.B;
  dim3 grid((unsigned)(8 * ((items + 7) / 8)));
  if (a.mod.docs) {
    const int ns = (a.L + kSplit - 1) / kSplit;
    doc_ranges_kernel<<<(unsigned)(a.B * ns), 64, 0, st>>>(a.mod.docs, a.mod.docs_sb, a.kv_lens, a.L, ns,
                                                           const_cast<int2*>(a.mod.ranges));
  }
  switch (kv_mode<T>(a)) {
    case kKvPaged: attn_prefill_mod<T, D, kKvPaged, MOD><<<grid, 256, 0, st>>>(a); break;
    case kKvTilePaged: attn_prefill_mod<T, D, kKvTilePaged, MOD><<<grid, 256, 0, st>>>(a); break;
    case kKvRowPaged: attn_prefill_mod<T, D, kKvRowPaged, MOD><<<grid, 256, 0, st>>>(a); break;
    default: attn_prefill_mod<T, D, kKvContig, MOD><<<grid, 256, 0, st>>>(a); break;
  }
  return bi_host::launch_status("bi_attn_scored");
}

template <typename T, int D>
int launch_rows_mod(ModRowsArgs& a, hipStream_t st) {
  const int64_t nchunks = ((int64_t)a.Tq * (a.Hq / a.Hkv) + 15) / 16;
  const unsigned grid = (unsigned)(8 * ((nchunks * a.nsplit * a.Hkv * a.B + 7) / 8));
  switch (kv_mode<T>(a)) {
    case kKvPaged: attn_rows_mod<T, D, kKvPaged><<<grid, 256, 0, st>>>(a); break;
    case kKvTilePaged: attn_rows_mod<T, D, kKvTilePaged><<<grid, 256, 0, st>>>(a); break;
    case kKvRowPaged: attn_rows_mod<T, D, kKvRowPaged><<<grid, 256, 0, st>>>(a); break;
    default: attn_rows_mod<T, D, kKvContig><<<grid, 256, 0, st>>>(a); break;
  }
  int rc = bi_host::launch_status("bi_attn_scored");
  if (rc || a.nsplit == 1) return rc;
  const int64_t n = (int64_t)a.B * a.Hq * a.Tq * (D / 4);
  attn_rows_combine<T, D><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(a);
  return bi_host::launch_status("bi_attn_scored(combine)");
}

#define BI_ATTN_MOD_D(X, T) X(T, 32) X(T, 64) X(T, 96) X(T, 128) X(T, 192) X(T, 256)
#define BI_ATTN_MOD_DECODE(T, D) template int launch_decode_mod<T, D>(ModDecodeArgs&, hipStream_t);
#define BI_ATTN_MOD_ROWS(T, D) template int launch_rows_mod<T, D>(ModRowsArgs&, hipStream_t);

}  // namespace bi
