// bi_qcache.hip — a paged K/V cache in 8 or 4 bits: the rotary embedding of queries
// and keys with the quantized write of keys and values into the pages
// (bi_rope_quantized_cache), and the reading of whole sequences back
// (bi_read_quantized_cache). Rows and groups: bi_qcache.h.
#include <algorithm>

#include "bi_qcache.h"

namespace bi {

// ---------------------------------------------------------------------------
// The write. Queries as in bi_rope_paged_cache: y1 = T(x1 cos - x2 sin), y2 = T(x2
// cos + x1 sin) in fp32, rounded once. Keys the same, then, as values, per group of
// g values of a row
//   bias = min, scale = T((max - min) / (2^bits - 1)), or 1 where that is 0,
//   code = round((y - bias) / scale), to even, clamped to [0, 2^bits - 1],
// in fp32 with IEEE quotients: the framework's quantizer on the rows that
// bi_rope_paged_cache writes. A group with an infinity or a NaN gets NaN for both.
//
// Bound by HBM bytes for prompts and by the launch for a decode step: 8192 tokens of 32 / 8
// heads of 128 in bf16 to 8 bits move 184 MB in 40 us, 4.6 TB/s (50 us with a division
// for each value and index, and a thread for one head of Q), in fp32 80 us. One thread
// takes 16 values of a row; a key's thread also reads the pairs that its values turn
// with (the row is in the cache then), so that it holds 16 neighbours and a group is
// 2, 4 or 8 neighbouring lanes. Rows are whole numbers of groups, so no group
// straddles a wave. Threads of queries take two runs of 8 that turn together, of two
// heads, which turn alike.
// ---------------------------------------------------------------------------
struct RopeQuantArgs {
  const void *q, *k, *v, *cos, *sin;
  const int32_t* positions;                            // [axes, B * T]
  const int64_t* slots;                                // [B * T]
  void* qo;
  char *kc, *vc;                                       // codes
  void *kg, *vg;                                       // (scale, bias) pairs
  int64_t q_row, k_row, v_row;
  int64_t kc_sp, kc_sh, kc_sl, kg_sp, kg_sh, kg_sl;    // page, head, row: bytes of codes, elements of pairs
  int64_t vc_sp, vc_sh, vc_sl, vg_sp, vg_sh, vg_sl;
  int64_t num_slots;
  int B, T, Hq, Hkv, D, half, table_rows, axes, shift, gshift;
  unsigned cph, cph_inv, t_inv, hq_inv, hkv_inv;       // pieces of 16 dims per head; 2^32 / cph, T, heads (pairs of q's) and 2 Hkv
  unsigned q_blocks;                                   // workgroups of queries; the others take keys and values
  int end[4];                                          // pairs of dims up to each axis's end
};

// x / d from inv = 2^32 / d rounded down (2^32 - 1 for 1).
__device__ __forceinline__ unsigned quotient(unsigned x, unsigned d, unsigned inv) {
  const unsigned q = __umulhi(x, inv);                 // or one less
  return x - q * d >= d ? q + 1 : q;
}

// cos and sin of pairs d .. d + 7 of token bt.
template <typename TAB>
__device__ __forceinline__ void table8(const RopeQuantArgs& a, unsigned bt, int d, float (&co)[8], float (&si)[8]) {
  const int64_t n = (int64_t)a.B * a.T;
  auto row = [&](int axis) {
    return (int64_t)min(max(a.positions[axis * n + bt], 0), a.table_rows - 1) * a.half;
  };
  auto axis_of = [&](int e) {
    int x = 0;
    while (x + 1 < a.axes && e >= a.end[x]) ++x;
    return x;
  };
  const int ax = axis_of(d);
  if (d + 8 <= a.end[ax]) {
    const int64_t r = row(ax) + d;
    load8<TAB>(static_cast<const TAB*>(a.cos) + r, co);
    load8<TAB>(static_cast<const TAB*>(a.sin) + r, si);
  } else {                                             // a section ends inside the run
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t r = row(axis_of(d + e)) + d + e;
      co[e] = to_f32(static_cast<const TAB*>(a.cos)[r]);
      si[e] = to_f32(static_cast<const TAB*>(a.sin)[r]);
    }
  }
}

template <typename T, typename TAB, int BITS>
__global__ __launch_bounds__(256) void rope_quant_kernel(RopeQuantArgs a) {
  const unsigned cph = a.cph;
  if (blockIdx.x < a.q_blocks) {
    const unsigned id = blockIdx.x * 256u + threadIdx.x, hn = ((unsigned)a.Hq + 1) / 2;
    const unsigned rest = quotient(id, cph, a.cph_inv), c = id - rest * cph;
    const unsigned rest2 = quotient(rest, (unsigned)a.T, a.t_inv), t = rest - rest2 * (unsigned)a.T;
    const unsigned b = quotient(rest2, hn, a.hq_inv), h0 = 2 * (rest2 - b * hn);
    if (b >= (unsigned)a.B) return;
    const int heads = min(2, a.Hq - (int)h0);
    const unsigned bt = b * (unsigned)a.T + t;
    const int rc = a.half / 8;
    const bool turn = (int)c < rc;
    const int d1 = turn ? 8 * (int)c : 2 * a.half + 16 * ((int)c - rc);
    const int d2 = turn ? a.half + 8 * (int)c : d1 + 8;
    const T* src = static_cast<const T*>(a.q) + (int64_t)bt * a.q_row + (int64_t)h0 * a.D;
    float x1[2][8], x2[2][8], co[8], si[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h >= heads) continue;
      load8<T>(src + h * a.D + d1, x1[h]);
      load8<T>(src + h * a.D + d2, x2[h]);
    }
    if (turn) table8<TAB>(a, bt, d1, co, si);
    T* dst = static_cast<T*>(a.qo) + (((int64_t)b * a.Hq + h0) * a.T + t) * a.D;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h >= heads) continue;
      if (turn) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y1 = __builtin_fmaf(x1[h][e], co[e], -(x2[h][e] * si[e]));
          const float y2 = __builtin_fmaf(x2[h][e], co[e], x1[h][e] * si[e]);
          x1[h][e] = y1;
          x2[h][e] = y2;
        }
      }
      store8<T>(dst + (int64_t)h * a.T * a.D + d1, x1[h]);
      store8<T>(dst + (int64_t)h * a.T * a.D + d2, x2[h]);
    }
    return;
  }
  const unsigned id = (blockIdx.x - a.q_blocks) * 256u + threadIdx.x;
  const unsigned rest = quotient(id, cph, a.cph_inv), c = id - rest * cph;
  const unsigned rest2 = quotient(rest, (unsigned)a.T, a.t_inv), t = rest - rest2 * (unsigned)a.T;
  const unsigned b = quotient(rest2, 2u * a.Hkv, a.hkv_inv), hv = rest2 - b * (2u * a.Hkv);
  // (Threads past the end and of padding rows stay for the lanes that share their wave.)
  const bool live = b < (unsigned)a.B;
  const bool key = hv < (unsigned)a.Hkv;
  const int h = (int)(key ? hv : hv - a.Hkv);
  const unsigned bt = live ? b * (unsigned)a.T + t : 0;
  const int64_t slot = live ? a.slots[bt] : -1;
  const bool write = slot >= 0 && slot < a.num_slots;
  float x[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
  if (write) {
    const T* src = key ? static_cast<const T*>(a.k) + (int64_t)bt * a.k_row + (int64_t)h * a.D
                       : static_cast<const T*>(a.v) + (int64_t)bt * a.v_row + (int64_t)h * a.D;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int d = 16 * (int)c + 8 * i;
      load8<T>(src + d, x[i]);
      if (key && d < 2 * a.half) {
        const bool low = d < a.half;
        float p[8], co[8], si[8];
        load8<T>(src + (low ? d + a.half : d - a.half), p);
        table8<TAB>(a, bt, low ? d : d - a.half, co, si);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float ps = p[e] * si[e];
          x[i][e] = to_f32(to_store<T>(__builtin_fmaf(x[i][e], co[e], low ? -ps : ps)));
        }
      }
    }
  }
  float lo = INFINITY, hi = -INFINITY, odd = 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo = fminf(lo, x[i][e]);
      hi = fmaxf(hi, x[i][e]);
      odd = fmaxf(odd, fabsf(x[i][e]) < INFINITY ? 0.0f : 1.0f);   // (fminf and fmaxf pass a NaN by)
    }
  const int lanes = (1 << a.gshift) / 16;              // 2, 4 or 8
  for (int off = 1; off < lanes; off <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, off, kWave));
    hi = fmaxf(hi, __shfl_xor(hi, off, kWave));
    odd = fmaxf(odd, __shfl_xor(odd, off, kWave));
  }
  if (!write) return;
  constexpr float kTop = (float)((1 << BITS) - 1);
  // (a range past fp32's: the difference of the quotients)
  const float range = hi - lo;
  float scale = to_f32(to_store<T>(range < INFINITY ? range / kTop : hi / kTop - lo / kTop));
  if (!(scale > 0.0f)) scale = 1.0f;
  // The last code is left out where its value, which the rounded scale may put past
  // the largest one, would overflow: finite values read back finite.
  const float most = fabsf(to_f32(to_store<T>(__builtin_fmaf(kTop, scale, lo)))) < INFINITY ? kTop : kTop - 1.0f;
  const int64_t page = slot >> a.shift, row = slot & (((int64_t)1 << a.shift) - 1);
  char* codes = key ? a.kc + page * a.kc_sp + h * a.kc_sh + row * a.kc_sl : a.vc + page * a.vc_sp + h * a.vc_sh + row * a.vc_sl;
  T* pairs = key ? static_cast<T*>(a.kg) + page * a.kg_sp + h * a.kg_sh + row * a.kg_sl
                 : static_cast<T*>(a.vg) + page * a.vg_sp + h * a.vg_sh + row * a.vg_sl;
  uint32_t w[BITS / 2];
  auto encode = [&](auto divide) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < BITS / 2; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = __builtin_rintf(divide(x[i][e] - lo));
        const uint32_t code = (uint32_t)fminf(fmaxf(y, 0.0f), most);
        const int at = (8 * i + e) * BITS;
        w[at / 32] |= code << (at % 32);
      }
  };
  // The IEEE quotient of n by the group's scale s without a division each: from r, the
  // rounded 1 / s, q = n r is off by less than 2 units in its last place, n - q s is exact,
  // and q + r (n - q s) lies within 2^-23 units of n / s before it is rounded. A
  // quotient by a scale of 11 bits or fewer is 2^-13 units at least from where its rounding
  // turns; by one of 24 bits that step gives a neighbour of n / s, and from such a q a second
  // one the rounded quotient (Markstein 1990). Of a q below 1/4, code 0 in any case, the
  // remainder may be no normal number; scales from 2^-80 on keep it exact above.
  if (scale >= 0x1p-80f && range < INFINITY) {
    const float r = 1.0f / scale;
    encode([&](float n) {
      float q = n * r;
#pragma unroll
      for (int i = 0; i < (sizeof(T) == 2 ? 1 : 2); ++i) q = __builtin_fmaf(__builtin_fmaf(-q, scale, n), r, q);
      return q;
    });
  } else {
    encode([&](float n) { return n / scale; });
  }
  if constexpr (BITS == 8) *reinterpret_cast<u32x4*>(codes + 16 * c) = u32x4{w[0], w[1], w[2], w[3]};
  else *reinterpret_cast<u32x2*>(codes + 8 * c) = u32x2{w[0], w[1]};
  if (c % (unsigned)lanes == 0) {
    T* p = pairs + 2 * (16 * (int)c >> a.gshift);
    const T s = odd != 0.0f ? to_store<T>(NAN) : to_store<T>(scale), z = odd != 0.0f ? to_store<T>(NAN) : to_store<T>(lo);
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint32_t*>(p) = (uint32_t)__builtin_bit_cast(uint16_t, s) | (uint32_t)__builtin_bit_cast(uint16_t, z) << 16;
    } else {
      *reinterpret_cast<u32x2*>(p) = u32x2{__builtin_bit_cast(uint32_t, s), __builtin_bit_cast(uint32_t, z)};
    }
  }
}

// ---------------------------------------------------------------------------
// The reading back: [B, Hkv, L, D] of T from the pages of every sequence, rows from
// its length on as zeros (FILL) or left as they are. Bound by HBM bytes, mostly those
// written: 16 sequences of up to 8192 tokens, 8 heads of 128 from 8 bits to bf16, in
// 138 us near the rate of a copy (133); to fp32 in 349 (240). One thread takes 16 codes of a row of K or V.
// `source` (null: none): of each sequence the one in whose pages its first keys lie
// (a row of `all`) and how many do.
// ---------------------------------------------------------------------------
struct ReadQuantArgs {
  const char *kc, *vc;
  const void *kg, *vg;
  const int32_t *table, *kv_lens, *source, *all;
  void *ko, *vo;
  int64_t kc_sp, kc_sh, kc_sl, kg_sp, kg_sh, kg_sl, vc_sp, vc_sh, vc_sl, vg_sp, vg_sh, vg_sl, table_stride;
  int Hkv, L, D, shift, gshift, num_pages, fill;
};

template <typename T, int BITS>
__global__ __launch_bounds__(256) void read_quant_kernel(ReadQuantArgs a) {
  // grid: (runs of 256 pieces of one head's rows, kv heads x {K, V}, sequences)
  const unsigned ppr = (unsigned)a.D / 16;
  const unsigned id = blockIdx.x * 256u + threadIdx.x;
  const unsigned pos = id / ppr, c = id % ppr;
  if (pos >= (unsigned)a.L) return;
  const int b = blockIdx.z, h = (int)(blockIdx.y % (unsigned)a.Hkv);
  const bool key = blockIdx.y < (unsigned)a.Hkv;
  const int len = a.kv_lens ? min(max(a.kv_lens[b], 0), a.L) : a.L;
  T* dst = static_cast<T*>(key ? a.ko : a.vo) + (((int64_t)b * a.Hkv + h) * a.L + pos) * a.D + 16 * c;
  typename Frag<T>::type y[2];
  if ((int)pos < len) {
    const bool shared = a.source && (int)pos < a.source[2 * b + 1];
    const int32_t* of = shared ? a.all + a.source[2 * b] * a.table_stride : a.table + b * a.table_stride;
    const int64_t page = min(max(of[pos >> a.shift], 0), a.num_pages - 1);
    const int64_t row = pos & ((1u << a.shift) - 1);
    const char* codes = key ? a.kc + page * a.kc_sp + h * a.kc_sh + row * a.kc_sl : a.vc + page * a.vc_sp + h * a.vc_sh + row * a.vc_sl;
    const T* pairs = key ? static_cast<const T*>(a.kg) + page * a.kg_sp + h * a.kg_sh + row * a.kg_sl
                         : static_cast<const T*>(a.vg) + page * a.vg_sp + h * a.vg_sh + row * a.vg_sl;
    const Codes16<BITS> w = load_codes16<BITS>(codes + 2 * BITS * c);
    const Pair<T> g = load_pair(pairs + 2 * (16 * (int)c >> a.gshift));
#pragma unroll
    for (int i = 0; i < 2; ++i) y[i] = dequant_frag<T, BITS>(w.half(i), g);
  } else {
    if (!a.fill) return;
    y[0] = y[1] = frag_zero<typename Frag<T>::type>();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<u32x4*>(dst + 8 * i) = __builtin_bit_cast(u32x4, y[i]);
    } else {
      *reinterpret_cast<f32x4*>(dst + 8 * i) = y[i].lo;
      *reinterpret_cast<f32x4*>(dst + 8 * i + 4) = y[i].hi;
    }
  }
}

}  // namespace bi

namespace {

// log2 of a power of two in [1, 2^24], or -1.
int shift_of(int64_t n) {
  if (n <= 0 || n > ((int64_t)1 << 24) || (n & (n - 1))) return -1;
  int s = 0;
  while (((int64_t)1 << s) < n) ++s;
  return s;
}

}  // namespace

namespace bi_host {

// Codes and groups of a quantized pool: bits, group size and head dim; base pointers
// and (page, head, row) strides of codes (bytes, multiples of 16) and pairs (elements, even).
int check_quant(const char* what, int64_t D, int64_t bits, int64_t group_size, const void* const* pointers, int n,
                const int64_t* strides, int dtype) {
  if (bits != 4 && bits != 8) return fail(BI_E_UNSUPPORTED, "%s: %lld bits (4 or 8)", what, (long long)bits);
  if (group_size != 32 && group_size != 64 && group_size != 128)
    return fail(BI_E_UNSUPPORTED, "%s: groups of %lld (32, 64 or 128)", what, (long long)group_size);
  if (D <= 0 || D % group_size)
    return fail(BI_E_INVALID_ARG, "%s: head dim %lld is no whole number of groups of %lld", what, (long long)D,
                (long long)group_size);
  if (dtype != BI_BF16 && dtype != BI_F16 && dtype != BI_F32)
    return fail(BI_E_UNSUPPORTED, "%s: unknown dtype %d", what, dtype);
  if (!strides) return fail(BI_E_INVALID_ARG, "%s: null pointer argument", what);
  bool ok = true;
  for (int i = 0; i < n; ++i) ok = ok && pointers[i] && aligned16(pointers[i]);
  for (int i = 0; i < 12; ++i) ok = ok && strides[i] >= 0 && strides[i] % (i % 6 < 3 ? 16 : 2) == 0;
  if (!ok)
    return fail(BI_E_INVALID_ARG, "%s: null or misaligned pool (16-byte aligned codes, whole pairs)", what);
  return BI_OK;
}

}  // namespace bi_host

extern "C" int bi_rope_quantized_cache(const void* q, int64_t q_row, const void* k, int64_t k_row, const void* v,
                                       int64_t v_row, const void* cos, const void* sin, int64_t table_rows,
                                       int table_dtype, const int32_t* positions, const int64_t* sections, int64_t axes,
                                       const int64_t* slots, void* q_out, void* k_codes, void* k_groups, void* v_codes,
                                       void* v_groups, int64_t num_pages, int64_t page_size, int64_t B, int64_t T,
                                       int64_t Hq, int64_t Hkv, int64_t D, int bits, int64_t group_size,
                                       const int64_t* strides, int dtype, void* stream) {
  using namespace bi_host;
  const char* what = "bi_rope_quantized_cache";
  const int shift = shift_of(page_size);
  if (shift < 0)
    return fail(BI_E_INVALID_ARG, "%s: page size %lld must be a power of two in [1, 2^24]", what, (long long)page_size);
  if (B < 0 || T < 0 || Hq <= 0 || Hkv <= 0 || D <= 0 || table_rows <= 0 || num_pages <= 0 || !sections)
    return fail(BI_E_INVALID_ARG, "%s: bad shape B=%lld T=%lld Hq=%lld Hkv=%lld D=%lld table_rows=%lld num_pages=%lld",
                what, (long long)B, (long long)T, (long long)Hq, (long long)Hkv, (long long)D, (long long)table_rows,
                (long long)num_pages);
  if (axes < 1 || axes > 4)
    return fail(BI_E_UNSUPPORTED, "%s: %lld position axes (1 to 4)", what, (long long)axes);
  const void* pools[4] = {k_codes, k_groups, v_codes, v_groups};
  int rc = check_quant(what, D, bits, group_size, pools, B == 0 || T == 0 ? 0 : 4, strides, dtype);
  if (rc) return rc;
  if (table_dtype != dtype && table_dtype != BI_F32)
    return fail(BI_E_UNSUPPORTED, "%s: dtype %d with tables of dtype %d (the same, or fp32)", what, dtype, table_dtype);
  if (B > 0x7fffffffLL || T > 0x7fffffffLL || Hq > 65536 || Hkv > 65536 || D > 65536 || table_rows > 0x7fffffffLL ||
      num_pages > 0x7fffffffLL || B * T > ((int64_t)1 << 31) - 1 ||
      B * T * (Hq + 1 + 2 * Hkv) * (D / 16) > ((int64_t)1 << 32) - 1024)  // threads
    return fail(BI_E_UNSUPPORTED, "%s: shape too large", what);
  bi::RopeQuantArgs a;
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
  if (k_codes == v_codes || k_groups == v_groups)
    return fail(BI_E_INVALID_ARG, "%s: one pool for keys and values", what);
  bool ok = positions && slots && q_row >= Hq * D && k_row >= Hkv * D && v_row >= Hkv * D && q_row % unit == 0 &&
            k_row % unit == 0 && v_row % unit == 0;
  for (const void* p : {q, k, v, cos, sin, (const void*)q_out}) ok = ok && p && aligned16(p);
  if (!ok)
    return fail(BI_E_INVALID_ARG, "%s: null or misaligned operand (16-byte aligned rows, rows of at least H * D)", what);
  a.q = q; a.k = k; a.v = v; a.cos = cos; a.sin = sin; a.positions = positions; a.slots = slots; a.qo = q_out;
  a.kc = static_cast<char*>(k_codes); a.vc = static_cast<char*>(v_codes); a.kg = k_groups; a.vg = v_groups;
  a.q_row = q_row; a.k_row = k_row; a.v_row = v_row;
  a.kc_sp = strides[0]; a.kc_sh = strides[1]; a.kc_sl = strides[2];
  a.kg_sp = strides[3]; a.kg_sh = strides[4]; a.kg_sl = strides[5];
  a.vc_sp = strides[6]; a.vc_sh = strides[7]; a.vc_sl = strides[8];
  a.vg_sp = strides[9]; a.vg_sh = strides[10]; a.vg_sl = strides[11];
  a.num_slots = num_pages * page_size;
  a.B = (int)B; a.T = (int)T; a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.D = (int)D; a.half = (int)half;
  a.table_rows = (int)table_rows; a.axes = (int)axes; a.shift = shift; a.gshift = shift_of(group_size);
  const int64_t per_head = B * T * (D / 16);
  auto inverse = [](int64_t d) { return d == 1 ? 0xffffffffu : (unsigned)(((int64_t)1 << 32) / d); };
  a.cph = (unsigned)(D / 16);
  a.cph_inv = inverse(D / 16);
  a.t_inv = inverse(T);
  a.hq_inv = inverse((Hq + 1) / 2);
  a.hkv_inv = inverse(2 * Hkv);
  a.q_blocks = (unsigned)((per_head * ((Hq + 1) / 2) + 255) / 256);
  const unsigned grid = a.q_blocks + (unsigned)((per_head * 2 * Hkv + 255) / 256);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto launch = [&](auto t, auto tab) {
    typedef decltype(t) TT;
    typedef decltype(tab) TAB;
    if (bits == 8) bi::rope_quant_kernel<TT, TAB, 8><<<grid, 256, 0, st>>>(a);
    else bi::rope_quant_kernel<TT, TAB, 4><<<grid, 256, 0, st>>>(a);
  };
  const bool wide = table_dtype == BI_F32;
  if (dtype == BI_BF16) wide ? launch(bi::bf16(), float()) : launch(bi::bf16(), bi::bf16());
  else if (dtype == BI_F16) wide ? launch(bi::f16(), float()) : launch(bi::f16(), bi::f16());
  else launch(float(), float());
  return launch_status(what);
}

namespace bi_host {

// bi_read_quantized_cache with ReadQuantArgs' source.
int read_quantized(const void* k_codes, const void* k_groups, const void* v_codes, const void* v_groups,
                   const int64_t* strides, const int32_t* block_table, int64_t table_stride, int64_t page_size,
                   int64_t num_pages, const int32_t* kv_lens, const int32_t* source, const int32_t* all, void* k_out,
                   void* v_out, int64_t B, int64_t Hkv, int64_t L, int64_t D, int bits, int64_t group_size, int fill,
                   int dtype, void* stream) {
  const char* what = "bi_read_quantized_cache";
  const int shift = shift_of(page_size);
  if (shift < 0)
    return fail(BI_E_INVALID_ARG, "%s: page size %lld must be a power of two in [1, 2^24]", what, (long long)page_size);
  if (B < 0 || Hkv <= 0 || L < 0 || D <= 0)
    return fail(BI_E_INVALID_ARG, "%s: bad shape B=%lld Hkv=%lld L=%lld D=%lld", what, (long long)B, (long long)Hkv,
                (long long)L, (long long)D);
  const void* pools[4] = {k_codes, k_groups, v_codes, v_groups};
  const bool none = B == 0 || L == 0;
  int rc = check_quant(what, D, bits, group_size, pools, none ? 0 : 4, strides, dtype);
  if (rc) return rc;
  if (none) return BI_OK;
  if (num_pages <= 0 || num_pages > 0x7fffffffLL || table_stride < (L + page_size - 1) / page_size)
    return fail(BI_E_INVALID_ARG, "%s: num_pages %lld, table stride %lld for %lld keys", what, (long long)num_pages,
                (long long)table_stride, (long long)L);
  if (!block_table || !k_out || !v_out || !aligned16(k_out) || !aligned16(v_out))
    return fail(BI_E_INVALID_ARG, "%s: null or misaligned operand", what);
  if (B > 65535 || Hkv > 32767 || D > 65536 || L > 0x7fffffffLL || L * (D / 16) > ((int64_t)1 << 31) ||
      (L * (D / 16) + 255) / 256 * 2 * Hkv * B > ((int64_t)1 << 24) - 1)
    return fail(BI_E_UNSUPPORTED, "%s: shape too large", what);
  bi::ReadQuantArgs a;
  a.kc = static_cast<const char*>(k_codes); a.vc = static_cast<const char*>(v_codes); a.kg = k_groups; a.vg = v_groups;
  a.table = block_table; a.kv_lens = kv_lens; a.source = source; a.all = all; a.ko = k_out; a.vo = v_out; a.table_stride = table_stride;
  a.kc_sp = strides[0]; a.kc_sh = strides[1]; a.kc_sl = strides[2];
  a.kg_sp = strides[3]; a.kg_sh = strides[4]; a.kg_sl = strides[5];
  a.vc_sp = strides[6]; a.vc_sh = strides[7]; a.vc_sl = strides[8];
  a.vg_sp = strides[9]; a.vg_sh = strides[10]; a.vg_sl = strides[11];
  a.Hkv = (int)Hkv; a.L = (int)L; a.D = (int)D; a.shift = shift; a.gshift = shift_of(group_size);
  a.num_pages = (int)num_pages; a.fill = fill ? 1 : 0;
  const dim3 grid((unsigned)((L * (D / 16) + 255) / 256), (unsigned)(2 * Hkv), (unsigned)B);
  hipStream_t st = static_cast<hipStream_t>(stream);
  auto launch = [&](auto t) {
    typedef decltype(t) TT;
    if (bits == 8) bi::read_quant_kernel<TT, 8><<<grid, 256, 0, st>>>(a);
    else bi::read_quant_kernel<TT, 4><<<grid, 256, 0, st>>>(a);
  };
  if (dtype == BI_BF16) launch(bi::bf16());
  else if (dtype == BI_F16) launch(bi::f16());
  else launch(float());
  return launch_status(what);
}

}  // namespace bi_host

extern "C" int bi_read_quantized_cache(const void* k_codes, const void* k_groups, const void* v_codes,
                                       const void* v_groups, const int64_t* strides, const int32_t* block_table,
                                       int64_t table_stride, int64_t page_size, int64_t num_pages,
                                       const int32_t* kv_lens, void* k_out, void* v_out, int64_t B, int64_t Hkv,
                                       int64_t L, int64_t D, int bits, int64_t group_size, int fill, int dtype,
                                       void* stream) {
  return bi_host::read_quantized(k_codes, k_groups, v_codes, v_groups, strides, block_table, table_stride, page_size,
                                 num_pages, kv_lens, nullptr, nullptr, k_out, v_out, B, Hkv, L, D, bits, group_size, fill,
                                 dtype, stream);
}
