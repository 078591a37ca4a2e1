// bi_paged.hip — what fills a paged K/V cache: pages and slots of a step's new
// tokens (bi_paged_slots), and the rotary embedding of queries and keys with
// the write of keys and values into the pages (bi_rope_paged_cache).
#include <algorithm>

#include "bi_common.h"

namespace bi {

// ---------------------------------------------------------------------------
// Pages and slots. Request b holds len_b tokens and gets new_b more, pages of
// P = 2^shift tokens:
//   have_b = ceil(len_b / P), want_b = ceil((len_b + new_b) / P),
//   need_b = want_b - have_b, or 0 for a request that cannot fit;
//   its new pages are free[first_b + j], j < need_b, first_b = cursor + the
//   needs of the requests before it.
// A request whose pages end behind the free list or do not fit the table, or
// that brings more than T tokens, is refused: its length stays and its rows get
// slot -1. Needs add up in whole
// numbers, so the plan is the same however the work is split.
//
// Bound by latency: a decode step of 64 requests moves 3 KB. So one launch,
// with no pass between workgroups: each workgroup adds up the needs of all
// requests before its own (8 bytes a request from the cache; at 4,096 requests
// the last of 16 workgroups reads 32 KB). 64 requests of one token 3.4 us, 256 of
// up to 2,048 (6.6 MB of slots and positions) 7.3.
// ---------------------------------------------------------------------------
struct SlotArgs {
  const int32_t *lens, *news, *free_pages, *cursor;
  int32_t *table, *positions, *out_lens, *out_cursor;
  int64_t* slots;
  int64_t table_stride, num_free, cap;      // cap: tokens that a table row holds
  int B, T, shift, max_pages, per_block, rows_y;
};

struct Request {
  int len, n, have;
  int64_t need;      // pages it asks of the free list
  bool fits;         // its pages fit the table, its tokens the T rows
};

__device__ __forceinline__ Request request_of(const SlotArgs& a, int b) {
  Request r;
  r.len = (int)min((int64_t)max(a.lens[b], 0), a.cap);
  r.n = max(a.news[b], 0);
  const int64_t mask = ((int64_t)1 << a.shift) - 1;
  r.have = (int)((r.len + mask) >> a.shift);
  const int64_t want = ((int64_t)r.len + r.n + mask) >> a.shift;
  r.fits = want <= a.max_pages && r.n <= a.T;
  r.need = r.fits ? want - r.have : 0;
  return r;
}

constexpr int kSlotThreads = 256;

__global__ __launch_bounds__(kSlotThreads) void paged_slots_kernel(SlotArgs a) {
  __shared__ int64_t wave_sum[kSlotThreads / kWave];
  __shared__ int64_t first_s[kSlotThreads];            // first free-list index of each request of the group
  __shared__ int len_s[kSlotThreads], n_s[kSlotThreads], have_s[kSlotThreads];
  const int t = threadIdx.x, wave = t / kWave, lane = t % kWave;
  const int b0 = (int)blockIdx.x * a.per_block;
  const int nb = min(a.per_block, a.B - b0);           // requests of this group (0 for an empty batch)
  const int64_t start = a.cursor ? min((int64_t)max(a.cursor[0], 0), a.num_free) : 0;

  // Needs of every request before the group.
  int64_t before = 0;
  for (int b = t; b < b0; b += kSlotThreads) before += request_of(a, b).need;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) before += __shfl_xor((long long)before, off, kWave);
  if (lane == 0) wave_sum[wave] = before;
  __syncthreads();
  before = start;
#pragma unroll
  for (int w = 0; w < kSlotThreads / kWave; ++w) before += wave_sum[w];
  __syncthreads();                                     // wave_sum is used again

  // The group's own: one thread per request, an inclusive scan of the needs.
  Request r{0, 0, 0, 0, true};
  if (t < nb) r = request_of(a, b0 + t);
  int64_t incl = r.need;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const int64_t up = __shfl_up((long long)incl, off, kWave);
    if (lane >= off) incl += up;
  }
  if (lane == kWave - 1) wave_sum[wave] = incl;
  __syncthreads();
  incl += before;
#pragma unroll
  for (int w = 0; w < kSlotThreads / kWave - 1; ++w)
    if (w < wave) incl += wave_sum[w];
  const bool ok = r.fits && (r.need == 0 || incl <= a.num_free);
  len_s[t] = r.len;
  n_s[t] = ok ? r.n : 0;
  have_s[t] = r.have;
  first_s[t] = incl - r.need;
  // Admitted requests that take pages come before every refused one that asks
  // for some, so the new cursor is the largest end that is still in the list;
  // the group in which the ends pass the list's end (else the last) knows it.
  int64_t reach = t < nb && r.need > 0 && ok ? incl : before;
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) reach = max(reach, (int64_t)__shfl_xor((long long)reach, off, kWave));
  __syncthreads();                                     // wave_sum read, the group's requests visible
  int64_t total = before;
#pragma unroll
  for (int w = 0; w < kSlotThreads / kWave; ++w) total += wave_sum[w];
  __syncthreads();
  if (lane == 0) wave_sum[wave] = reach;
  __syncthreads();
  if (blockIdx.y == 0) {
    if (t == 0 && before <= a.num_free && (total > a.num_free || b0 + a.per_block >= a.B)) {
#pragma unroll
      for (int w = 0; w < kSlotThreads / kWave; ++w) reach = max(reach, wave_sum[w]);
      a.out_cursor[0] = (int)reach;
    }
    if (t < nb) a.out_lens[b0 + t] = r.len + n_s[t];
    // New table entries: 256 / per_block threads for each request.
    const int share = kSlotThreads / a.per_block, g = t / share;
    if (g < nb && n_s[g] > 0) {
      const int64_t mask = ((int64_t)1 << a.shift) - 1;
      const int need = (int)(((int64_t)len_s[g] + n_s[g] + mask) >> a.shift) - have_s[g];
      for (int j = t % share; j < need; j += share)
        a.table[(int64_t)(b0 + g) * a.table_stride + have_s[g] + j] = a.free_pages[first_s[g] + j];
    }
  }
  // Slots and positions of the group's T rows each (the workgroup's share of
  // them): the new tokens are the last rows, as the causal attention counts.
  const int row0 = (int)blockIdx.y * a.rows_y, rows = min(a.rows_y, a.T - row0);
  for (int i = t; i < nb * rows; i += kSlotThreads) {
    const int g = nb == 1 ? 0 : i / rows, row = row0 + (nb == 1 ? i : i - g * rows);
    const int back = a.T - n_s[g];                     // padding rows
    int64_t slot = -1;
    int pos = 0;
    if (row >= back) {
      pos = len_s[g] + row - back;
      const int pg = pos >> a.shift;
      const int page = pg < have_s[g] ? a.table[(int64_t)(b0 + g) * a.table_stride + pg]
                                      : a.free_pages[first_s[g] + pg - have_s[g]];
      if (page >= 0) slot = ((int64_t)page << a.shift) + (pos & ((1 << a.shift) - 1));
    }
    const int64_t at = (int64_t)(b0 + g) * a.T + row;
    a.slots[at] = slot;
    a.positions[at] = pos;
  }
}

// ---------------------------------------------------------------------------
// RoPE and the write into the pages. A token's position may have up to four
// axes (time, height, width of an image or video token): the rotated pairs of
// dims are cut into one section per axis, and column d of the tables is read at
// the position of d's axis. With the halves x1, x2 of a head's first 2 R dims
//   y1 = T(x1 cos - x2 sin), y2 = T(x2 cos + x1 sin)
// in fp32 and rounded once; dims from 2 R on, and values, are copied. Each
// output element depends on its own inputs only.
//
// Bound by HBM bytes for prompts and by the launch for a decode step. One
// thread takes 8 + 8 elements of `HG` heads of one token and reads its pieces
// of cos and sin once for them. Tokens run inside heads, so that a wave writes
// runs of rows of one head's queries and pages: 4 x 2048 tokens, 32 / 8 heads of
// 128, three axes, bf16 44.5 -> 42.3 us (heads inside tokens before; 4.4 TB/s of
// the 4.8 that a large copy reaches).
// ---------------------------------------------------------------------------
struct RopePagedArgs {
  const void *q, *k, *v, *cos, *sin;
  const int32_t* positions;                            // [axes, B * T]
  const int64_t* slots;                                // [B * T]
  void *qo, *kp, *vp;
  int64_t q_row, k_row, v_row;                         // elements between tokens
  int64_t kp_sp, kp_sh, kp_sl, vp_sp, vp_sh, vp_sl;    // page, head, row of the pools
  int64_t num_slots;
  int B, T, Hq, Hkv, D, half, table_rows, axes, shift;
  int end[4];                                          // pairs of dims up to each axis's end
};

template <typename T, typename TAB, int HG>
__global__ __launch_bounds__(256) void rope_paged_kernel(RopePagedArgs a) {
  const unsigned cph = (unsigned)a.D / 16, heads = (unsigned)a.Hq + 2 * a.Hkv;
  const unsigned groups = (heads + HG - 1) / HG;
  const unsigned id = blockIdx.x * 256u + threadIdx.x;
  const unsigned c = id % cph, rest = id / cph;
  const unsigned t = rest % (unsigned)a.T, rest2 = rest / (unsigned)a.T;
  const unsigned h0 = rest2 % groups * HG, b = rest2 / groups;
  if (b >= (unsigned)a.B) return;
  const unsigned bt = b * (unsigned)a.T + t;
  const int rc = a.half / 8;                           // chunks of rotated pairs
  const bool turn = (int)c < rc;
  const int d1 = turn ? 8 * (int)c : 2 * a.half + 16 * ((int)c - rc);
  const int d2 = turn ? a.half + 8 * (int)c : d1 + 8;
  const int64_t slot = a.slots[bt];
  const bool write = slot >= 0 && slot < a.num_slots;
  const int64_t page = write ? slot >> a.shift : 0, row = write ? slot & (((int64_t)1 << a.shift) - 1) : 0;

  float x1[HG][8], x2[HG][8];
#pragma unroll
  for (int g = 0; g < HG; ++g) {
    const int h = (int)h0 + g;
    if (h >= (int)heads || (h >= a.Hq && !write)) continue;
    const T* src = h < a.Hq ? static_cast<const T*>(a.q) + (int64_t)bt * a.q_row + (int64_t)h * a.D
                   : h < a.Hq + a.Hkv
                       ? static_cast<const T*>(a.k) + (int64_t)bt * a.k_row + (int64_t)(h - a.Hq) * a.D
                       : static_cast<const T*>(a.v) + (int64_t)bt * a.v_row + (int64_t)(h - a.Hq - a.Hkv) * a.D;
    load8<T>(src + d1, x1[g]);
    load8<T>(src + d2, x2[g]);
  }
  float co[8], si[8];
  if (turn) {
    const int64_t n = (int64_t)a.B * a.T;
    auto table_row = [&](int axis) {
      return (int64_t)min(max(a.positions[axis * n + bt], 0), a.table_rows - 1) * a.half;
    };
    auto axis_of = [&](int d) {
      int x = 0;
      while (x + 1 < a.axes && d >= a.end[x]) ++x;
      return x;
    };
    const int ax = axis_of(d1);
    if (d1 + 8 <= a.end[ax]) {
      const int64_t r = table_row(ax) + d1;
      load8<TAB>(static_cast<const TAB*>(a.cos) + r, co);
      load8<TAB>(static_cast<const TAB*>(a.sin) + r, si);
    } else {                                           // a section ends inside the chunk
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int64_t r = table_row(axis_of(d1 + e)) + d1 + e;
        co[e] = to_f32(static_cast<const TAB*>(a.cos)[r]);
        si[e] = to_f32(static_cast<const TAB*>(a.sin)[r]);
      }
    }
  }
#pragma unroll
  for (int g = 0; g < HG; ++g) {
    const int h = (int)h0 + g;
    if (h >= (int)heads || (h >= a.Hq && !write)) continue;
    if (turn && h < a.Hq + a.Hkv) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y1 = __builtin_fmaf(x1[g][e], co[e], -(x2[g][e] * si[e]));
        const float y2 = __builtin_fmaf(x2[g][e], co[e], x1[g][e] * si[e]);
        x1[g][e] = y1;
        x2[g][e] = y2;
      }
    }
    T* dst = h < a.Hq ? static_cast<T*>(a.qo) + (((int64_t)b * a.Hq + h) * a.T + t) * a.D
             : h < a.Hq + a.Hkv
                 ? static_cast<T*>(a.kp) + page * a.kp_sp + (int64_t)(h - a.Hq) * a.kp_sh + row * a.kp_sl
                 : static_cast<T*>(a.vp) + page * a.vp_sp + (int64_t)(h - a.Hq - a.Hkv) * a.vp_sh + row * a.vp_sl;
    store8<T>(dst + d1, x1[g]);
    store8<T>(dst + d2, x2[g]);
  }
}

template <typename T, typename TAB>
static void launch_rope_paged(const RopePagedArgs& a, hipStream_t st) {
  // Two heads a thread once that leaves 2^17 threads: its pieces of cos and sin
  // serve both, and twice the loads are in flight. 8 x 1024 tokens of 14 / 2 heads
  // of 64, fp16: 10.8 -> 9.8 us, 4 x 1000 of 8 / 8 of 128, fp32: 27.4 -> 23.3; four
  // heads no faster; 64 tokens of 32 / 8: 3.7 -> 4.1, so fewer keep one.
  const int64_t per_head = (int64_t)a.B * a.T * (a.D / 16);
  const int heads = a.Hq + 2 * a.Hkv;
  if (per_head * heads >= (1 << 18))
    rope_paged_kernel<T, TAB, 2><<<(unsigned)((per_head * ((heads + 1) / 2) + 255) / 256), 256, 0, st>>>(a);
  else
    rope_paged_kernel<T, TAB, 1><<<(unsigned)((per_head * heads + 255) / 256), 256, 0, st>>>(a);
}

// log2 of a power of two in [1, 2^24], or -1.
static int page_shift_of(int64_t page_size) {
  if (page_size <= 0 || page_size > ((int64_t)1 << 24) || (page_size & (page_size - 1))) return -1;
  int s = 0;
  while (((int64_t)1 << s) < page_size) ++s;
  return s;
}

}  // namespace bi

extern "C" int bi_paged_slots(const int32_t* kv_lens, const int32_t* new_lens, int32_t* block_table,
                              int64_t table_stride, int64_t max_pages, const int32_t* free_pages, int64_t num_free,
                              const int32_t* cursor, int64_t* slots, int32_t* positions, int32_t* out_lens,
                              int32_t* out_cursor, int64_t B, int64_t T, int64_t page_size, void* stream) {
  using namespace bi_host;
  const char* what = "bi_paged_slots";
  const int shift = bi::page_shift_of(page_size);
  if (shift < 0)
    return fail(BI_E_INVALID_ARG, "%s: page size %lld must be a power of two in [1, 2^24]", what, (long long)page_size);
  if (B < 0 || T <= 0 || max_pages <= 0 || num_free < 0 || table_stride < max_pages)
    return fail(BI_E_INVALID_ARG, "%s: bad shape B=%lld T=%lld max_pages=%lld table_stride=%lld num_free=%lld", what,
                (long long)B, (long long)T, (long long)max_pages, (long long)table_stride, (long long)num_free);
  // (positions are 32-bit: a table row's tokens and a step's new ones)
  if (B > ((int64_t)1 << 20) || T > ((int64_t)1 << 24) || max_pages > 0x7fffffffLL || num_free > 0x7fffffffLL ||
      max_pages > (0x7fffffffLL - T) / page_size)
    return fail(BI_E_UNSUPPORTED, "%s: shape too large", what);
  if ((B > 0 && (!kv_lens || !new_lens || !block_table || !slots || !positions || !out_lens)) || !out_cursor ||
      (num_free > 0 && !free_pages))
    return fail(BI_E_INVALID_ARG, "%s: null pointer argument", what);
  if ((B > 0 && (out_lens == kv_lens || out_lens == new_lens)) || out_cursor == cursor)
    return fail(BI_E_INVALID_ARG, "%s: outputs must not be the inputs (every workgroup reads all of them)", what);
  bi::SlotArgs a;
  a.lens = kv_lens; a.news = new_lens; a.free_pages = free_pages; a.cursor = cursor;
  a.table = block_table; a.positions = positions; a.out_lens = out_lens; a.out_cursor = out_cursor; a.slots = slots;
  a.table_stride = table_stride; a.num_free = num_free; a.cap = max_pages * page_size;
  a.B = (int)B; a.T = (int)T; a.shift = shift; a.max_pages = (int)max_pages;
  // Requests of a workgroup: about 1024 rows, a power of two, and no more than
  // 1024 groups in all; a request of more rows is cut along them.
  int per = 1;
  while (per < bi::kSlotThreads && ((int64_t)per * T < 1024 || (B + per - 1) / per > 1024)) per *= 2;
  a.per_block = per;
  a.rows_y = per == 1 ? (int)std::min<int64_t>(T, 2048) : (int)T;
  dim3 grid((unsigned)std::max<int64_t>(1, (B + per - 1) / per), (unsigned)((T + a.rows_y - 1) / a.rows_y));
  bi::paged_slots_kernel<<<grid, bi::kSlotThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  return launch_status(what);
}

extern "C" int bi_rope_paged_cache(const void* q, int64_t q_row, const void* k, int64_t k_row, const void* v,
                                   int64_t v_row, const void* cos, const void* sin, int64_t table_rows,
                                   int table_dtype, const int32_t* positions, const int64_t* sections, int64_t axes,
                                   const int64_t* slots, void* q_out, void* k_pages, void* v_pages, int64_t num_pages,
                                   int64_t page_size, int64_t B, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                   const int64_t* strides, int dtype, void* stream) {
  using namespace bi_host;
  const char* what = "bi_rope_paged_cache";
  const int shift = bi::page_shift_of(page_size);
  if (shift < 0)
    return fail(BI_E_INVALID_ARG, "%s: page size %lld must be a power of two in [1, 2^24]", what, (long long)page_size);
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || D % 16 || table_rows <= 0 || num_pages <= 0 || !strides ||
      !sections)
    return fail(BI_E_INVALID_ARG, "%s: bad shape B=%lld T=%lld Hq=%lld Hkv=%lld D=%lld table_rows=%lld num_pages=%lld",
                what, (long long)B, (long long)T, (long long)Hq, (long long)Hkv, (long long)D, (long long)table_rows,
                (long long)num_pages);
  if (axes < 1 || axes > 4)
    return fail(BI_E_UNSUPPORTED, "%s: %lld position axes (1 to 4)", what, (long long)axes);
  if ((dtype != BI_BF16 && dtype != BI_F16 && dtype != BI_F32) || (table_dtype != dtype && table_dtype != BI_F32))
    return fail(BI_E_UNSUPPORTED, "%s: dtype %d with tables of dtype %d (the same, or fp32)", what, dtype, table_dtype);
  if (B > 0x7fffffffLL || T > 0x7fffffffLL || Hq > 65536 || Hkv > 65536 || D > 65536 || table_rows > 0x7fffffffLL ||
      num_pages > 0x7fffffffLL || B * T > ((int64_t)1 << 31) - 1 ||
      B * T * (Hq + 2 * Hkv) * (D / 16) > ((int64_t)1 << 32) - 256)  // threads
    return fail(BI_E_UNSUPPORTED, "%s: shape too large", what);
  bi::RopePagedArgs a;
  int64_t half = 0;
  for (int i = 0; i < 4; ++i) {
    if (i < axes) {
      if (sections[i] < 0 || sections[i] > D / 2)
        return fail(BI_E_INVALID_ARG, "%s: section %d of %lld pairs of dims", what, i, (long long)sections[i]);
      half += sections[i];
    }
    a.end[i] = (int)std::min<int64_t>(half, D);
  }
  if (half <= 0 || half > D / 2 || half % 8)
    return fail(BI_E_INVALID_ARG, "%s: sections of %lld pairs of dims; need a multiple of 8, at most D / 2 = %lld", what,
                (long long)half, (long long)(D / 2));
  if (B == 0 || T == 0) return BI_OK;
  const int64_t unit = 16 / (int64_t)dtype_size(dtype);
  if (k_pages && k_pages == v_pages) return fail(BI_E_INVALID_ARG, "%s: one pool for keys and values", what);
  bool ok = q && k && v && cos && sin && positions && slots && q_out && k_pages && v_pages && q_row >= Hq * D &&
            k_row >= Hkv * D && v_row >= Hkv * D && q_row % unit == 0 && k_row % unit == 0 && v_row % unit == 0;
  for (const void* p : {q, k, v, cos, sin, (const void*)q_out, (const void*)k_pages, (const void*)v_pages})
    ok = ok && aligned16(p);
  for (int i = 0; i < 6; ++i) ok = ok && strides[i] >= 0 && strides[i] % unit == 0;
  if (!ok)
    return fail(BI_E_INVALID_ARG, "%s: null or misaligned operand (16-byte aligned rows, rows of at least H * D)", what);
  a.q = q; a.k = k; a.v = v; a.cos = cos; a.sin = sin; a.positions = positions; a.slots = slots;
  a.qo = q_out; a.kp = k_pages; a.vp = v_pages; a.q_row = q_row; a.k_row = k_row; a.v_row = v_row;
  a.kp_sp = strides[0]; a.kp_sh = strides[1]; a.kp_sl = strides[2];
  a.vp_sp = strides[3]; a.vp_sh = strides[4]; a.vp_sl = strides[5];
  a.num_slots = num_pages * page_size;
  a.B = (int)B; a.T = (int)T; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.D = (int)D; a.half = (int)half;
  a.table_rows = (int)table_rows; a.axes = (int)axes; a.shift = shift;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool wide = table_dtype == BI_F32;
  if (dtype == BI_BF16) wide ? bi::launch_rope_paged<bi::bf16, float>(a, st) : bi::launch_rope_paged<bi::bf16, bi::bf16>(a, st);
  else if (dtype == BI_F16) wide ? bi::launch_rope_paged<bi::f16, float>(a, st) : bi::launch_rope_paged<bi::f16, bi::f16>(a, st);
  else bi::launch_rope_paged<float, float>(a, st);
  return launch_status(what);
}
