// bi_attn_pages.hip — C ABI of attention over quantized pages and of batches that
// share prefixes (bi_attn_pages). Kernels of few rows: bi_attn_pages.h. Many rows go
// through the kernels of bi_attn_scored with nothing changed: quantized pages read
// back into the workspace first, a slice of the sequences at a time, shared prefixes
// by a block table of their own there.
#include <numeric>

#include "bi_attn_pages_api.h"

namespace bi_host {
int check_quant(const char* what, int64_t D, int64_t bits, int64_t group_size, const void* const* pointers, int n,
                const int64_t* strides, int dtype);
int read_quantized(const void* k_codes, const void* k_groups, const void* v_codes, const void* v_groups,
                   const int64_t* strides, const int32_t* block_table, int64_t table_stride, int64_t page_size,
                   int64_t num_pages, const int32_t* kv_lens, const int32_t* source, const int32_t* all, void* k_out,
                   void* v_out, int64_t B, int64_t Hkv, int64_t L, int64_t D, int bits, int64_t group_size, int fill,
                   int dtype, void* stream);
}

namespace bi {

// Where the first keys of a sequence lie, for the kernels of many rows: a workgroup per
// sequence. By the plan's rule (bi_attn_pages.h), sequence b is in group n, the first with
// starts[n + 1] > b, if no start up to starts[n] lies above b; the largest of those is
// the group's first sequence. cols 0: out [B, 2], that sequence and how many keys come from
// it. Else out [B, cols] is a block table of pages of `unit` = min(page size, 256) keys:
// pages as they are, or of a larger page's 256 keys the piece page * per_page + its
// number * per_split. (Entries behind a sequence's length are not written.)
__global__ __launch_bounds__(256) void shared_source_kernel(PagesArgs a, int32_t* out, int64_t cols, int per_page, int per_split) {
  __shared__ int part[2][4];
  const int b = blockIdx.x, tid = threadIdx.x;
  auto least = [&](int x, int at) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x = min(x, __shfl_xor(x, off, kWave));
    if (tid % kWave == 0) part[at][tid / kWave] = x;
    __syncthreads();
    return min(min(part[at][0], part[at][1]), min(part[at][2], part[at][3]));
  };
  int n = a.groups;
  for (int i = tid; i < n; i += 256)
    if (plan_start(a, i + 1) > b) n = i;
  n = least(n, 0);
  int lo = 0;
  for (int i = tid; i <= n && i < a.groups; i += 256) lo = max(lo, plan_start(a, i));
  lo = -least(-lo, 1);
  int keys = 0;
  if (n < a.groups && lo <= b && plan_start(a, n + 1) - lo > 1) {
    const int want = a.slens ? min(max(a.slens[n], 0), a.L) : a.shared_len;
    keys = min(want, pages_len(a, lo)) / kSplit * kSplit;
  }
  if (cols == 0) {
    if (tid == 0) {
      out[2 * b] = lo;
      out[2 * b + 1] = keys;
    }
    return;
  }
  const int split_shift = __builtin_ctz(kSplit), shift = min(a.page_shift, split_shift);
  const int used = (int)(((int64_t)pages_len(a, b) + (1 << shift) - 1) >> shift);
  for (int c = tid; c < used; c += 256) {
    const int pos = c << shift, row = pos < keys ? lo : b;
    const int page = (int)clamp_page(a.table[row * a.table_stride + (pos >> a.page_shift)], a.num_pages);
    const int piece = (pos & ((1 << a.page_shift) - 1)) >> split_shift;
    out[b * cols + c] = a.page_shift <= split_shift ? page : page * per_page + piece * per_split;
  }
}

}  // namespace bi

namespace {

// Bytes of sequences that are read back at a time (one sequence at least).
constexpr int64_t kDenseBytes = (int64_t)2 << 30;

int64_t dense_bytes(int64_t Hkv, int64_t L, int64_t D, int dtype) {
  return 2 * Hkv * L * D * (int64_t)bi_host::dtype_size(dtype);
}
int64_t dense_slice(int64_t B, int64_t Hkv, int64_t L, int64_t D, int dtype) {
  return std::max<int64_t>(1, std::min(B, kDenseBytes / dense_bytes(Hkv, L, D, dtype)));
}

// A page of more than a split as pages of one split: a page's and a split's strides in
// units, the largest one that K and V have in common up to a factor, which is each one's page stride
// then. False: there is none, or the last one's number is no int32.
struct Pieces {
  int64_t per_page, per_split, k, v, count;
};
bool pieces_of(int64_t k_sp, int64_t k_sl, int64_t v_sp, int64_t v_sl, int64_t num_pages, int64_t page_size, Pieces* p) {
  for (int64_t s : {k_sp, k_sl, v_sp, v_sl})
    if (s > ((int64_t)1 << 50)) return false;
  if (num_pages == 1) k_sp = v_sp = 0;
  k_sl *= bi::kSplit;
  v_sl *= bi::kSplit;
  p->k = std::gcd(k_sp, k_sl);
  p->v = std::gcd(v_sp, v_sl);
  if (p->k && p->v && (k_sp / p->k != v_sp / p->v || k_sl / p->k != v_sl / p->v)) return false;
  p->per_page = p->k ? k_sp / p->k : p->v ? v_sp / p->v : 0;
  p->per_split = p->k ? k_sl / p->k : p->v ? v_sl / p->v : 0;
  const double last = (double)(num_pages - 1) * p->per_page + (double)(page_size / bi::kSplit - 1) * p->per_split;
  if (last >= 2147483647.0) return false;
  p->count = (int64_t)last + 1;
  return true;
}

size_t partial_bytes(int64_t B, int64_t Hq, int64_t Tq, int64_t L, int64_t D) {
  return ((size_t)bi::rows_partial_bytes(B, Hq, Tq, L, D) + 15) / 16 * 16;
}

// What shared_source_kernel writes: a table of pages of at most a split, or (codes) two words a sequence.
int64_t table_cols(int64_t L, int64_t page_size) {
  const int64_t unit = std::min<int64_t>(page_size, bi::kSplit);
  return (L + unit - 1) / unit;
}
size_t source_bytes(int64_t B, int64_t L, int64_t groups, int bits, int64_t page_size) {
  return groups == 0 ? 0 : ((size_t)B * (bits ? 2 : table_cols(L, page_size)) * sizeof(int32_t) + 15) / 16 * 16;
}

bool bad_shape(int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t L, int64_t D, int64_t groups) {
  return B <= 0 || B > 65535 || Hq <= 0 || Hkv <= 0 || Hq > 0x7fffffffLL / 16 || Hq % Hkv || Hkv > 65535 || Tq <= 0 ||
         Tq > 0x7fffffffLL || L <= 0 || L > 0x7fffffffLL - bi::kSplit || D <= 0 || D > 65536 || groups < 0 || groups > 65535;
}

bool known(int64_t D, int dtype) {
  return (D == 32 || D == 64 || D == 96 || D == 128 || D == 192 || D == 256) &&
         (dtype == BI_BF16 || dtype == BI_F16 || dtype == BI_F32);
}

// Whether the kernels of few rows can count a call's items, rows and the merge's threads in
// 32 bits. (Products in an order in which none leaves 64 bits.)
bool few_fits(int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t L, int64_t groups) {
  const int64_t nsplit = (L + bi::kSplit - 1) / bi::kSplit, rows1 = Tq * (Hq / Hkv);
  return B * Hq * Tq <= 0x7fffffffLL && rows1 <= 0x7fffffffLL - 16 && B * rows1 <= 0x7fffffffLL - 1024 &&
         (double)nsplit * Hkv * ((double)B * ((rows1 + 15) / 16) + groups) <= 2e9 &&
         B * Hq * Tq * nsplit <= ((int64_t)1 << 36) && B * Hq * Tq * 64 <= ((int64_t)1 << 32) - 256;
}

}  // namespace

extern "C" size_t bi_attn_pages_workspace_bytes_paged(int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t L, int64_t D,
                                                      int64_t groups, int bits, int causal, int dtype, int64_t page_size) {
  if (bad_shape(B, Hq, Hkv, Tq, L, D, groups) || !known(D, dtype) || page_size <= 0) return 0;
  if (bi::pages_few_rows(B, Hq, Hkv, Tq, L, D, groups, bits, causal, dtype))
    return !few_fits(B, Hq, Hkv, Tq, L, groups) ? 0 : partial_bytes(B, Hq, Tq, L, D) + (size_t)(2 + bi::kPlanWords * (groups + B)) * sizeof(int32_t);
  const int64_t nb = bits ? dense_slice(B, Hkv, L, D, dtype) : B;
  size_t n = bi_attn_scored_workspace_bytes(nb, Hq, Hkv, Tq, L, D, causal, 0, dtype);
  if (bits) n = std::max(n, bi_attn_scored_workspace_bytes((B - 1) % nb + 1, Hq, Hkv, Tq, L, D, causal, 0, dtype));
  n = (n + 15) / 16 * 16 + source_bytes(B, L, groups, bits, page_size);
  return n + (bits ? (size_t)(nb * dense_bytes(Hkv, L, D, dtype)) : 0);
}

extern "C" size_t bi_attn_pages_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t L, int64_t D,
                                                int64_t groups, int bits, int causal, int dtype) {
  return bi_attn_pages_workspace_bytes_paged(B, Hq, Hkv, Tq, L, D, groups, bits, causal, dtype, 1);
}

extern "C" int bi_attn_pages(const void* q, const void* k, const void* k_groups, const void* v, const void* v_groups,
                             int bits, int64_t group_size, const int32_t* block_table, int64_t table_stride,
                             int64_t page_size, int64_t num_pages, const int32_t* kv_lens,
                             const int32_t* shared_starts, const int32_t* shared_lens, int64_t shared_len,
                             int64_t groups, void* out, int64_t B, int64_t Hq, int64_t Hkv, int64_t Tq, int64_t L,
                             int64_t D, const int64_t* strides, int causal, float scale, int dtype, void* ws,
                             size_t ws_bytes, void* stream) {
  using namespace bi_host;
  const char* what = "bi_attn_pages";
  if (B == 0) return BI_OK;
  if (Hq > 0 && Hkv > 0 && Hq % Hkv)
    return fail(BI_E_INVALID_ARG, "%s: Hq=%lld not a multiple of Hkv=%lld", what, (long long)Hq, (long long)Hkv);
  if (B < 0 || Hq <= 0 || Hkv <= 0 || Tq <= 0 || L <= 0 || groups < 0)
    return fail(BI_E_INVALID_ARG, "%s: bad shape B=%lld Hq=%lld Hkv=%lld Tq=%lld L=%lld groups=%lld", what, (long long)B,
                (long long)Hq, (long long)Hkv, (long long)Tq, (long long)L, (long long)groups);
  if (!known(D, BI_F32))
    return fail(BI_E_UNSUPPORTED, "%s: head dim %lld (supported: 32, 64, 96, 128, 192, 256)", what, (long long)D);
  if (!known(D, dtype))
    return fail(BI_E_UNSUPPORTED, "%s: unknown dtype %d", what, dtype);
  if (bad_shape(B, Hq, Hkv, Tq, L, D, groups)) return fail(BI_E_UNSUPPORTED, "%s: shape exceeds the grid limits", what);
  if (causal && Tq > L)
    return fail(BI_E_INVALID_ARG, "%s: causal needs Tq (%lld) <= L (%lld)", what, (long long)Tq, (long long)L);
  int shift = 0;
  if (page_size <= 0 || page_size > ((int64_t)1 << 24) || (page_size & (page_size - 1)))
    return fail(BI_E_INVALID_ARG, "%s: page size %lld must be a power of two in [1, 2^24]", what, (long long)page_size);
  while (((int64_t)1 << shift) < page_size) ++shift;
  if (num_pages <= 0 || num_pages > 0x7fffffffLL)
    return fail(BI_E_INVALID_ARG, "%s: num_pages %lld must be in [1, 2^31)", what, (long long)num_pages);
  if (table_stride < (L + page_size - 1) / page_size)
    return fail(BI_E_INVALID_ARG, "%s: table stride %lld < ceil(L / page size) = %lld", what, (long long)table_stride,
                (long long)((L + page_size - 1) / page_size));
  if (groups > 0 && ((!shared_starts && groups != 1) || (!shared_lens && (shared_len < 0 || groups != 1))))
    return fail(BI_E_INVALID_ARG, "%s: %lld groups need their starts and lengths", what, (long long)groups);
  if (!q || !k || !v || !block_table || !out || !strides)
    return fail(BI_E_INVALID_ARG, "%s: null pointer argument", what);
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(out))
    return fail(BI_E_INVALID_ARG, "%s: q, k, v, out must be 16-byte aligned", what);
  const int64_t es = (int64_t)dtype_size(dtype);
  for (int i = 0; i < 9; ++i)
    if (strides[i] < 0 || strides[i] * (bits && i >= 3 ? 1 : es) % 16)
      return fail(BI_E_INVALID_ARG, "%s: stride %d (%lld) must be >= 0 and 16-byte aligned", what, i,
                  (long long)strides[i]);
  int64_t qs[12];                                         // codes and pairs of K, then of V
  if (bits) {
    const void* pools[4] = {k, k_groups, v, v_groups};
    for (int i = 0; i < 3; ++i) {
      qs[i] = strides[3 + i];
      qs[3 + i] = strides[9 + i];
      qs[6 + i] = strides[6 + i];
      qs[9 + i] = strides[12 + i];
    }
    const int rc = check_quant(what, D, bits, group_size, pools, 4, qs, dtype);
    if (rc) return rc;
  }
  // (a lane finds its rows by 32-bit strides)
  const bool few = bi::pages_few_rows(B, Hq, Hkv, Tq, L, D, groups, bits, causal, dtype);
  for (int i = 0; i < 15; ++i)
    if ((i < 3 ? few : bits && i % 3 != 1) && strides[i] > 0xffffffffLL)
      return fail(BI_E_UNSUPPORTED, "%s: stride %d (%lld) must be below 2^32", what, i, (long long)strides[i]);
  Pieces pieces = {1, 0, strides[3], strides[6], num_pages};
  if (!few && !bits && groups > 0 && page_size > bi::kSplit &&
      !pieces_of(strides[3], strides[5], strides[6], strides[8], num_pages, page_size, &pieces))
    return fail(BI_E_UNSUPPORTED,
                "%s: shared prefixes of many rows over pages of %lld keys need K and V of one layout (page strides %lld, "
                "%lld, row strides %lld, %lld)", what, (long long)page_size, (long long)strides[3], (long long)strides[6],
                (long long)strides[5], (long long)strides[8]);
  if (few && !few_fits(B, Hq, Hkv, Tq, L, groups)) return fail(BI_E_UNSUPPORTED, "%s: grid too large", what);
  const size_t need = bi_attn_pages_workspace_bytes_paged(B, Hq, Hkv, Tq, L, D, groups, bits, causal, dtype, page_size);
  if (need > 0 && (!ws || ws_bytes < need || !aligned16(ws)))
    return fail(BI_E_WORKSPACE, "%s: 16-byte aligned workspace of %zu bytes required, got %zu", what, need,
                ws ? ws_bytes : (size_t)0);
  hipStream_t st = static_cast<hipStream_t>(stream);

  bi::PagesArgs a;
  a.kv_lens = kv_lens; a.table = block_table; a.starts = shared_starts; a.slens = shared_lens;
  a.table_stride = table_stride;
  a.B = (int)B; a.L = (int)L; a.groups = (int)groups;
  a.shared_len = (int)std::min(std::max<int64_t>(shared_len, 0), L);
  a.page_shift = shift; a.num_pages = (int)num_pages;

  if (!few) {
    const bi_score_mod none = {0.0f, nullptr, nullptr, 0, nullptr};
    const size_t source_n = source_bytes(B, L, groups, bits, page_size);
    int32_t* source = groups ? static_cast<int32_t*>(ws) : nullptr;
    if (groups) {
      const int64_t cols = bits ? 0 : table_cols(L, page_size);
      bi::shared_source_kernel<<<(unsigned)B, 256, 0, st>>>(a, source, cols, (int)pieces.per_page, (int)pieces.per_split);
      const int rc = launch_status(what);
      if (rc) return rc;
    }
    char* after = static_cast<char*>(ws) + source_n;
    ws_bytes -= source_n;
    if (!bits) {
      if (!groups)
        return bi_attn_scored(q, k, v, block_table, table_stride, page_size, num_pages, kv_lens, out, B, Hq, Hkv, Tq, L, D,
                              strides, causal, scale, &none, dtype, ws, ws_bytes, stream);
      const int64_t st9[9] = {strides[0], strides[1], strides[2], pieces.k, strides[4], strides[5], pieces.v, strides[7], strides[8]};
      return bi_attn_scored(q, k, v, source, table_cols(L, page_size), std::min<int64_t>(page_size, bi::kSplit), pieces.count,
                            kv_lens, out, B, Hq, Hkv, Tq, L, D, st9, causal, scale, &none, dtype, after, ws_bytes, stream);
    }
    const int64_t nb = dense_slice(B, Hkv, L, D, dtype), one = Hkv * L * D;
    const int64_t dense_st[9] = {strides[0], strides[1], strides[2], one, L * D, D, one, L * D, D};
    char* kd = after;
    char* vd = kd + nb * one * es;
    char* rest = vd + nb * one * es;                      // (a multiple of 16 bytes: D is one of 32)
    for (int64_t b0 = 0; b0 < B; b0 += nb) {
      const int64_t n = std::min(nb, B - b0);
      int rc = read_quantized(k, k_groups, v, v_groups, qs, block_table + b0 * table_stride, table_stride, page_size,
                              num_pages, kv_lens ? kv_lens + b0 : nullptr, source ? source + 2 * b0 : nullptr, block_table,
                              kd, vd, n, Hkv, L, D, bits, group_size, 0, dtype, stream);
      if (rc) return rc;
      rc = bi_attn_scored(static_cast<const char*>(q) + b0 * strides[0] * es, kd, vd, nullptr, 0, 0, 0,
                          kv_lens ? kv_lens + b0 : nullptr, static_cast<char*>(out) + b0 * Hq * Tq * D * es, n, Hq, Hkv, Tq,
                          L, D, dense_st, causal, scale, &none, dtype, rest, ws_bytes - 2 * nb * one * es, stream);
      if (rc) return rc;
    }
    return BI_OK;
  }

  const int64_t nsplit = (L + bi::kSplit - 1) / bi::kSplit, rows1 = Tq * (Hq / Hkv), n = B * Hq * Tq * nsplit;
  a.q = q; a.k = k; a.v = v; a.kg = k_groups; a.vg = v_groups;
  a.out = out;
  a.q_sb = strides[0]; a.q_sh = strides[1]; a.q_st = strides[2];
  a.k_sp = strides[3]; a.k_sh = strides[4]; a.k_sl = strides[5];
  a.v_sp = strides[6]; a.v_sh = strides[7]; a.v_sl = strides[8];
  a.kg_sp = a.kg_sh = a.kg_sl = a.vg_sp = a.vg_sh = a.vg_sl = 0;
  a.gshift = 5;
  if (bits) {
    a.kg_sp = strides[9]; a.kg_sh = strides[10]; a.kg_sl = strides[11];
    a.vg_sp = strides[12]; a.vg_sh = strides[13]; a.vg_sl = strides[14];
    a.gshift = group_size == 32 ? 5 : group_size == 64 ? 6 : 7;
  }
  auto reach = [&](int i) { return (num_pages - 1) * strides[i] + (Hkv - 1) * strides[i + 1] + (page_size - 1) * strides[i + 2] + D; };
  a.near = bits && reach(3) < ((int64_t)1 << 32) && reach(6) < ((int64_t)1 << 32);
  a.hkv_inv = bi::inverse(Hkv);
  a.rows1_inv = bi::inverse(rows1);
  a.g_inv = bi::inverse(Hq / Hkv);
  a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.Tq = (int)Tq; a.nsplit = (int)nsplit;
  a.causal = causal ? 1 : 0;
  a.scale_log2 = scale * bi::kLog2e;
  const int64_t up = (n + 3) / 4 * 4;
  a.pm = static_cast<float*>(ws);
  a.pl = a.pm + up;
  a.pacc = a.pl + up;
  a.plan = reinterpret_cast<int32_t*>(static_cast<char*>(ws) + partial_bytes(B, Hq, Tq, L, D));
  auto launch = [&](auto t) -> int {
    typedef decltype(t) T;
    switch (D) {
      case 32: return bi::launch_pages<T, 32>(a, bits, st);
      case 64: return bi::launch_pages<T, 64>(a, bits, st);
      case 96: return bi::launch_pages<T, 96>(a, bits, st);
      case 128: return bi::launch_pages<T, 128>(a, bits, st);
      case 192: return bi::launch_pages<T, 192>(a, bits, st);
      default: return bi::launch_pages<T, 256>(a, bits, st);
    }
  };
  if (dtype == BI_BF16) return launch(bi::bf16());
  if (dtype == BI_F16) return launch(bi::f16());
  return launch(float());
}
