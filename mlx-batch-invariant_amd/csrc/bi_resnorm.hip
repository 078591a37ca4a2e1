// bi_resnorm.hip — the norms around a block in one pass: what a block adds to
// the residual stream, normed, gated and scaled, and the next block's input.
//
//   u = x * inv(x) * w_post      (w_post may be null: ones; POST = false: u = x)
//   y = res + u * gate * scale   (gate may be null: ones)       -> T(y)
//   h = y * inv(y) * w_pre       (PRE = false: no h)            -> T(h)
//   inv(z) = 1 / sqrtf(sum z^2 / D + eps)
//
// in fp32, left to right, y kept unrounded for h, each output rounded once.
// The sums follow rms_norm's order (bi_rmsnorm.hip): thread t of 256 owns the
// 8-element chunks t, t + 256, ..., a wave folds by the xor butterfly, the wave
// sums are added left to right: D alone fixes it.
#include <algorithm>

#include "bi_common.h"

namespace bi {

constexpr int kResThreads = 256;

struct ResNormArgs {
  const void *x, *res, *gate, *w_post, *w_pre;
  void *y, *h;
  int64_t x_row, res_row, gate_row, gate_group;   // gate row r / gate_group
  int64_t first, rows;                            // rows first .. rows - 1 (of this launch)
  int D;
  float eps, scale;
};

// How a row's 8-element chunks are read and written: rows of whole 16-byte
// pieces; rows at any element (an odd D, a slice), whose chunks are still one
// access each (the hardware takes any address; the last chunk may be short and
// goes element by element); rows longer than the registers hold, element by element.
enum RowForm { kAligned, kAnywhere, kElements };

template <typename T>
struct Any16 { uint32_t w[4]; } __attribute__((packed, aligned(alignof(T))));

// Eight elements from index `base`, zeros past D.
template <typename T, RowForm FORM>
__device__ __forceinline__ void row_load(const T* p, int base, int D, float* out) {
  if constexpr (FORM == kAligned) {
    load8<T>(p + base, out);
    return;
  }
  if (FORM == kAnywhere && base + 8 <= D) {
    T e[8];
    *reinterpret_cast<Any16<T>*>(e) = *reinterpret_cast<const Any16<T>*>(p + base);
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<Any16<T>*>(e + 4) = *reinterpret_cast<const Any16<T>*>(p + base + 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = to_f32(e[i]);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) out[e] = base + e < D ? to_f32(p[base + e]) : 0.0f;
}
template <typename T, RowForm FORM>
__device__ __forceinline__ void row_store(T* p, int base, int D, const float* in) {
  if constexpr (FORM == kAligned) {
    store8<T>(p + base, in);
    return;
  }
  if (FORM == kAnywhere && base + 8 <= D) {
    T e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = to_store<T>(in[i]);
    *reinterpret_cast<Any16<T>*>(p + base) = *reinterpret_cast<const Any16<T>*>(e);
    if constexpr (sizeof(T) == 4)
      *reinterpret_cast<Any16<T>*>(p + base + 4) = *reinterpret_cast<const Any16<T>*>(e + 4);
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (base + e < D) p[base + e] = to_store<T>(in[e]);
}

// Sum over the WPR waves of a row in rms_norm's order (waves it does not have
// would add 0 there); every thread gets it. The barrier before the write lets a
// second sum use the same words.
template <int WPR>
__device__ __forceinline__ float row_sum(float ss, float* wave_sums) {
  ss = wave_sum_butterfly(ss);
  if constexpr (WPR == 1) return ss;
  const int wave = threadIdx.x / kWave, first = wave / WPR * WPR;
  __syncthreads();
  if (threadIdx.x % kWave == 0) wave_sums[wave] = ss;
  __syncthreads();
  float total = wave_sums[first];
#pragma unroll
  for (int i = 1; i < WPR; ++i) total = total + wave_sums[first + i];
  return total;
}

// Rows of up to NC * 512 * WPR elements, kept in registers between the sums, WPR
// waves each: 4 / WPR rows in a workgroup. Bound by HBM: one read of x, residual and
// gate, one write of y and h. 16384 rows of 4096 with a gate, bf16: 105 us, 5.1 TB/s;
// rows of 4097 (kAnywhere; a third chunk, in which one thread has work) 177 us, 425
// element by element.
template <typename T, int NC, RowForm FORM, bool POST, bool PRE, int WPR>
__global__ __launch_bounds__(kResThreads) void res_norm_kernel(ResNormArgs a) {
  static_assert(WPR == 4 || NC == 1, "res_norm_kernel: a row's chunks are its threads'");
  __shared__ float wave_sums[kResThreads / kWave];
  constexpr int kRowThreads = WPR * kWave;
  const int t = threadIdx.x % kRowThreads;
  const int64_t row0 = a.first + (int64_t)blockIdx.x * (kResThreads / kRowThreads) + threadIdx.x / kRowThreads;
  const bool live = row0 < a.rows;
  const int64_t row = live ? row0 : a.rows - 1;        // (a workgroup's spare rows repeat the last and store nothing)
  const T* x = static_cast<const T*>(a.x) + row * a.x_row;
  const T* res = static_cast<const T*>(a.res) + row * a.res_row;
  const T* gate = a.gate ? static_cast<const T*>(a.gate) + row / a.gate_group * a.gate_row : nullptr;
  const T* w1 = static_cast<const T*>(a.w_post);
  const T* w2 = static_cast<const T*>(a.w_pre);
  const int D = a.D, nchunks = (D + 7) / 8;
  float u[NC][8], y[NC][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int chunk = t + c * kRowThreads;
    if (chunk < nchunks) {
      row_load<T, FORM>(x, 8 * chunk, D, u[c]);
      row_load<T, FORM>(res, 8 * chunk, D, y[c]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) u[c][e] = y[c][e] = 0.0f;
    }
  }
  if constexpr (POST) {
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(u[c][e], u[c][e], ss);
    const float inv = 1.0f / sqrtf(row_sum<WPR>(ss, wave_sums) / (float)D + a.eps);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int chunk = t + c * kRowThreads;
      float w[8];
      if (w1 && chunk < nchunks) row_load<T, FORM>(w1, 8 * chunk, D, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[c][e] = w1 && chunk < nchunks ? (u[c][e] * inv) * w[e] : u[c][e] * inv;
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int chunk = t + c * kRowThreads;
    if (chunk < nchunks) {
      if (gate) {
        float g[8];
        row_load<T, FORM>(gate, 8 * chunk, D, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[c][e] = u[c][e] * g[e];
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[c][e] = y[c][e] + u[c][e] * a.scale;
        if (FORM == kAligned || 8 * chunk + e < D) ss = __builtin_fmaf(y[c][e], y[c][e], ss);
      }
      if (live) row_store<T, FORM>(static_cast<T*>(a.y) + row * D, 8 * chunk, D, y[c]);
    }
  }
  if constexpr (PRE) {
    const float inv = 1.0f / sqrtf(row_sum<WPR>(ss, wave_sums) / (float)D + a.eps);
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int chunk = t + c * kRowThreads;
      if (chunk < nchunks) {
        float w[8];
        if (w2) row_load<T, FORM>(w2, 8 * chunk, D, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[c][e] = w2 ? (y[c][e] * inv) * w[e] : y[c][e] * inv;
        if (live) row_store<T, FORM>(static_cast<T*>(a.h) + row * D, 8 * chunk, D, y[c]);
      }
    }
  }
}

// Longer rows: the same order, x, res and gate read again for each pass, element by
// element: 4096 rows of 9000 / 16384 with a gate for each, bf16: 376 / 687 us, 1.0 TB/s
// of one pass's bytes (rows of 8192, kept in registers: 77 us, 4.4).
template <typename T, bool POST, bool PRE>
__global__ __launch_bounds__(kResThreads) void res_norm_kernel_long(ResNormArgs a) {
  __shared__ float wave_sums[kResThreads / kWave];
  const int64_t row = a.first + blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_row;
  const T* res = static_cast<const T*>(a.res) + row * a.res_row;
  const T* gate = a.gate ? static_cast<const T*>(a.gate) + row / a.gate_group * a.gate_row : nullptr;
  const T* w1 = static_cast<const T*>(a.w_post);
  const T* w2 = static_cast<const T*>(a.w_pre);
  const int D = a.D, nchunks = (D + 7) / 8;
  float inv1 = 1.0f;
  if constexpr (POST) {
    float ss = 0.0f;
    for (int chunk = threadIdx.x; chunk < nchunks; chunk += kResThreads) {
      float u[8];
      row_load<T, kElements>(x, 8 * chunk, D, u);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(u[e], u[e], ss);
    }
    inv1 = 1.0f / sqrtf(row_sum<kResThreads / kWave>(ss, wave_sums) / (float)D + a.eps);
  }
  auto stream = [&](int chunk, float* y) {            // the chunk's y, unrounded
    float u[8], w[8];
    row_load<T, kElements>(x, 8 * chunk, D, u);
    row_load<T, kElements>(res, 8 * chunk, D, y);
    if (POST) {
      if (w1) row_load<T, kElements>(w1, 8 * chunk, D, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = w1 ? (u[e] * inv1) * w[e] : u[e] * inv1;
    }
    if (gate) {
      row_load<T, kElements>(gate, 8 * chunk, D, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = u[e] * w[e];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = y[e] + u[e] * a.scale;
  };
  float ss = 0.0f;
  for (int chunk = threadIdx.x; chunk < nchunks; chunk += kResThreads) {
    float y[8];
    stream(chunk, y);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (8 * chunk + e < D) ss = __builtin_fmaf(y[e], y[e], ss);
    if constexpr (!PRE) row_store<T, kElements>(static_cast<T*>(a.y) + row * D, 8 * chunk, D, y);
  }
  if constexpr (PRE) {
    const float inv = 1.0f / sqrtf(row_sum<kResThreads / kWave>(ss, wave_sums) / (float)D + a.eps);
    for (int chunk = threadIdx.x; chunk < nchunks; chunk += kResThreads) {
      float y[8], w[8];
      stream(chunk, y);
      row_store<T, kElements>(static_cast<T*>(a.y) + row * D, 8 * chunk, D, y);
      if (w2) row_load<T, kElements>(w2, 8 * chunk, D, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = w2 ? (y[e] * inv) * w[e] : y[e] * inv;
      row_store<T, kElements>(static_cast<T*>(a.h) + row * D, 8 * chunk, D, y);
    }
  }
}

template <typename T, bool POST, bool PRE>
static void launch_res_norm(const ResNormArgs& a, bool vec, hipStream_t st) {
  const int64_t rows = a.rows - a.first;
  const int nchunks = (a.D + 7) / 8;
#define BI_RES(NC, WPR)                                                                                 \
  do {                                                                                                  \
    const unsigned grid = (unsigned)((rows + 4 / WPR - 1) / (4 / WPR));                                 \
    if (vec) res_norm_kernel<T, NC, kAligned, POST, PRE, WPR><<<grid, kResThreads, 0, st>>>(a);         \
    else res_norm_kernel<T, NC, kAnywhere, POST, PRE, WPR><<<grid, kResThreads, 0, st>>>(a);            \
  } while (0)
  // A wave or two for rows that fill no more: all of its lanes have work, and rows
  // of one wave meet no barrier. 16384 rows of 896, bf16: 31.7 us with four waves a
  // row, 26.2 with two.
  if (nchunks <= kWave) BI_RES(1, 1);
  else if (nchunks <= 2 * kWave) BI_RES(1, 2);
  else if (nchunks <= kResThreads) BI_RES(1, 4);
  else if (nchunks <= 2 * kResThreads) BI_RES(2, 4);
  else if (nchunks <= 3 * kResThreads) BI_RES(3, 4);
  else if (nchunks <= 4 * kResThreads) BI_RES(4, 4);
  else res_norm_kernel_long<T, POST, PRE><<<(unsigned)rows, kResThreads, 0, st>>>(a);
#undef BI_RES
}

template <typename T>
static void launch_res_norm_t(ResNormArgs a, bool post, bool pre, bool vec, hipStream_t st) {
  // A launch holds fewer than 2^32 threads: more rows take several.
  constexpr int64_t kMost = (int64_t)1 << 23;
  const int64_t rows = a.rows;
  for (; a.first < rows; a.first += kMost) {
    a.rows = std::min(rows, a.first + kMost);
    if (post && pre) launch_res_norm<T, true, true>(a, vec, st);
    else if (post) launch_res_norm<T, true, false>(a, vec, st);
    else launch_res_norm<T, false, true>(a, vec, st);
  }
}

}  // namespace bi

extern "C" int bi_residual_rms_norm(const void* x, int64_t x_row_stride, const void* res, int64_t res_row_stride,
                                    const void* gate, int64_t gate_row_stride, int64_t gate_group, const void* w_post,
                                    const void* w_pre, void* y, void* h, int64_t rows, int64_t D, float eps,
                                    float scale, int post, int pre, int dtype, void* stream) {
  using namespace bi_host;
  const char* what = "bi_residual_rms_norm";
  if (rows < 0 || D <= 0 || D > (int64_t)1 << 30)
    return fail(BI_E_INVALID_ARG, "%s: bad shape rows=%lld D=%lld", what, (long long)rows, (long long)D);
  if (rows > 0x7fffffffLL)
    return fail(BI_E_UNSUPPORTED, "%s: rows=%lld (fewer than 2^31)", what, (long long)rows);
  if (dtype != BI_BF16 && dtype != BI_F16 && dtype != BI_F32)
    return fail(BI_E_UNSUPPORTED, "%s: unknown dtype %d", what, dtype);
  if (!post && !pre) return fail(BI_E_INVALID_ARG, "%s: neither norm asked for", what);
  if (rows == 0) return BI_OK;
  if (!x || !res || !y || (pre && !h)) return fail(BI_E_INVALID_ARG, "%s: null pointer argument", what);
  if (x_row_stride < D || res_row_stride < D || (gate && (gate_row_stride < 0 || gate_group <= 0)))
    return fail(BI_E_INVALID_ARG, "%s: row strides %lld, %lld < D %lld, or gate rows of stride %lld for %lld rows each",
                what, (long long)x_row_stride, (long long)res_row_stride, (long long)D, (long long)gate_row_stride,
                (long long)gate_group);
  bi::ResNormArgs a{x, res, gate, post ? w_post : nullptr, pre ? w_pre : nullptr, y, h, x_row_stride, res_row_stride,
                    gate ? gate_row_stride : 0, gate ? gate_group : 1, 0, rows, (int)D, eps, scale};
  bool vec = D % 8 == 0 && a.x_row % 8 == 0 && a.res_row % 8 == 0 && a.gate_row % 8 == 0;
  for (const void* p : {x, res, gate, a.w_post, a.w_pre, (const void*)y, (const void*)h}) vec = vec && aligned16(p);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == BI_BF16) bi::launch_res_norm_t<bi::bf16>(a, post, pre, vec, st);
  else if (dtype == BI_F16) bi::launch_res_norm_t<bi::f16>(a, post, pre, vec, st);
  else bi::launch_res_norm_t<float>(a, post, pre, vec, st);
  return launch_status(what);
}
