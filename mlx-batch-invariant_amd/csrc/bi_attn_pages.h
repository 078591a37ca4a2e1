// bi_attn_pages.h — attention of few rows over paged caches: pages of 8- or 4-bit
// codes, and batches whose sequences share a prefix that is read once.
//
// The order of operations is that of bi_attn_common.h: an output's bits are those
// of the plain kernels over the same keys (codes: over the values that they stand
// for, T(fma(code, scale, bias))), whichever rows share a workgroup.
//
// A segment is a run of splits with the rows that see them: the whole 256-key
// splits of a group's shared prefix with the rows of every sequence of the group,
// or a sequence's other splits with its own rows. Rows of a segment are
// (sequence, token, head of the kv head), heads inside tokens inside sequences.
#pragma once

#include "bi_attn_mfma.h"
#include "bi_attn_pages_api.h"
#include "bi_qcache.h"

namespace bi {

// x / d for x >= 0 from inv = inverse(d).
__device__ __forceinline__ int quotient(int x, int d, unsigned inv) {
  const int q = (int)__umulhi((unsigned)x, inv);          // or one less
  return x - q * d >= d ? q + 1 : q;
}

// The length of a wave-uniform sequence, by a scalar load: waiting for it does not wait
// for the vector loads in flight, which return in order.
__device__ __forceinline__ int pages_len_uniform(const PagesArgs& a, int b) {
  if (!a.kv_lens) return a.L;
  return min(max(load_uniform_i32(a.kv_lens + __builtin_amdgcn_readfirstlane(b)), 0), a.L);
}

typedef int i32x4_t __attribute__((ext_vector_type(4)));

// The item that the workgroup takes in a round, of the 8 XCDs (which workgroups reach
// in turn) each a run of neighbours: the chunks of one split, and the heads of one
// page, share its cache. The last round is dealt to all XCDs too. -1: none is left.
__device__ __forceinline__ int dealt(int round, int items) {
  const int grid = (int)gridDim.x, base = round * grid, n = min(items - base, grid);
  const int run = (n + 7) / 8, i = (int)(blockIdx.x / 8), at = (int)(blockIdx.x % 8) * run + i;
  return i < run && at < n ? base + at : -1;
}

// The operands of a P.V step in LDS, the two halves of a lane `half` pieces apart.
template <typename T>
__device__ __forceinline__ void store_pfrag(u32x4* p, int half, const PFrag<T>& pf) {
  if constexpr (sizeof(T) == 2) {
    p[0] = __builtin_bit_cast(u32x4, pf.hi);
    p[half] = __builtin_bit_cast(u32x4, pf.lo);
  } else {
    p[0] = __builtin_bit_cast(u32x4, pf.f.lo);
    p[half] = __builtin_bit_cast(u32x4, pf.f.hi);
  }
}
template <typename T>
__device__ __forceinline__ PFrag<T> load_pfrag(const u32x4* p, int half) {
  PFrag<T> pf;
  if constexpr (sizeof(T) == 2) {
    pf.hi = __builtin_bit_cast(typename Frag<T>::type, p[0]);
    pf.lo = __builtin_bit_cast(typename Frag<T>::type, p[half]);
  } else {
    pf.f.lo = __builtin_bit_cast(f32x4, p[0]);
    pf.f.hi = __builtin_bit_cast(f32x4, p[half]);
  }
  return pf;
}

// ---------------------------------------------------------------------------
// The plan of a call: segments (groups, then sequences) with the first item of each,
// and how many 16-row chunks an item takes. Of each segment kPlanWords words: first
// item, first sequence, sequences, first split, splits.
// Groups are the runs starts[n] .. starts[n + 1] of sequences (clamped, each from
// the last one's end on); one of fewer than two sequences shares nothing. The
// shared splits are whole and lie within the first sequence's own keys. (shared_source_kernel
// finds one sequence's group by the same rule.)
// Every workgroup of attn_pages plans a call of up to kPlanFused segments for itself, in
// LDS (a launch of its own takes 7 us); of more, one workgroup does it in front of them.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kPlanMostChunks = 32;
constexpr int kPlanCached = 2048;        // segments whose first items a workgroup keeps in LDS

// By a workgroup of NT threads; `seg` in LDS or in memory, `part` in LDS. (All counts
// stay below 2^31: the caller's items at one chunk each do.)
template <int NT>
__device__ __forceinline__ void plan_segments(const PagesArgs& a, int32_t* seg, int* part, int& items, int& per) {
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int rows1 = a.Tq * (a.Hq / a.Hkv);                // rows of one sequence and kv head
  // Sequences: all splits their own to begin with (the first word: the length).
  for (int b = tid; b < a.B; b += NT) {
    int32_t* s = seg + (int64_t)(a.groups + b) * kPlanWords;
    const int len = pages_len(a, b);
    s[0] = len;
    s[1] = b;
    s[2] = 1;
    s[3] = 0;
    s[4] = max((len + kSplit - 1) / kSplit, a.nsplit == 1 ? 1 : 0);   // (one split: its items write the results)
  }
  // Groups, NT at a time; ends of earlier ones bound a start from below.
  int ends = 0;
  for (int n0 = 0; n0 == 0 || n0 < a.groups; n0 += NT) {
    const int n = n0 + tid;
    int lo = n < a.groups ? plan_start(a, n) : 0;
    const int hi = n < a.groups ? plan_start(a, n + 1) : 0;
    const int want = n < a.groups && a.slens ? min(max(a.slens[n], 0), a.L) : a.shared_len;
    int run = max(lo, hi);                                // the running maximum of all starts
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int up = __shfl_up(run, off, kWave);
      if (lane >= off) run = max(run, up);
    }
    if (lane == kWave - 1) part[wave] = run;
    __syncthreads();
    int before = ends;
    for (int w = 0; w < NT / kWave; ++w) {
      if (w < wave) before = max(before, part[w]);
      ends = max(ends, part[w]);
    }
    const int up = __shfl_up(run, 1, kWave);
    if (lane > 0) before = max(before, up);
    lo = max(lo, before);
    if (n < a.groups) {
      int32_t* s = seg + (int64_t)n * kPlanWords;
      s[1] = lo;
      s[2] = max(hi - lo, 0);
      s[3] = 0;
      s[4] = hi - lo > 1 ? min(want, (int)seg[(int64_t)(a.groups + lo) * kPlanWords]) / kSplit : 0;
    }
    __syncthreads();
  }
  // Their sequences' own splits begin behind the shared ones.
  for (int n = wave; n < a.groups; n += NT / kWave) {
    const int32_t* s = seg + (int64_t)n * kPlanWords;
    const int lo = s[1], size = s[2], splits = s[4];
    if (splits == 0) continue;
    for (int b = lo + lane; b < lo + size; b += kWave) {
      int32_t* t = seg + (int64_t)(a.groups + b) * kPlanWords;
      t[3] = splits;
      t[4] = max(t[4] - splits, 0);
    }
  }
  __syncthreads();
  const int nseg = a.groups + a.B;
  auto chunks_of = [&](const int32_t* s) { return (s[2] * rows1 + 15) / 16; };
  int units = 0;
  for (int i = tid; i < nseg; i += NT) {
    const int32_t* s = seg + (int64_t)i * kPlanWords;
    units += s[4] * chunks_of(s);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) units += __shfl_xor(units, off, kWave);
  if (lane == 0) part[wave] = units;
  __syncthreads();
  units = 0;
  for (int w = 0; w < NT / kWave; ++w) units += part[w];
  per = min(max(units * a.Hkv / a.slots, 1), kPlanMostChunks);
  // First items: an exclusive scan.
  items = 0;
  for (int i0 = 0; i0 < nseg; i0 += NT) {
    const int i = i0 + tid;
    int32_t* s = seg + (int64_t)min(i, nseg - 1) * kPlanWords;
    const int own = i < nseg ? s[4] * ((chunks_of(s) + per - 1) / per) * a.Hkv : 0;
    int incl = own;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int up = __shfl_up(incl, off, kWave);
      if (lane >= off) incl += up;
    }
    __syncthreads();
    if (lane == kWave - 1) part[wave] = incl;
    __syncthreads();
    int first = items + incl - own;
    for (int w = 0; w < NT / kWave; ++w) {
      if (w < wave) first += part[w];
      items += part[w];
    }
    if (i < nseg) s[0] = first;
  }
  __syncthreads();
}

// plan: [0] items in all, [1] chunks an item, [2 ...] the segments.
static __global__ __launch_bounds__(kPlanThreads) void pages_plan_kernel(PagesArgs a) {
  __shared__ int part[kPlanThreads / kWave];
  int items, per;
  plan_segments<kPlanThreads>(a, a.plan + 2, part, items, per);
  if (threadIdx.x == 0) {
    a.plan[0] = items;
    a.plan[1] = per;
  }
}

// The codes of K row r that lane (r, qq) needs as score operands, dims 32 st + 8 qq .. + 7
// of every step st, are pieces of 8 or 4 bytes. A lane reads 16 bytes instead, the
// row's four lanes 64 in a run: two steps of 8 bits (lane qq half of step qq / 2) or four
// of 4 (lane qq step qq), and they hand each other their pieces by swaps of 16-lane rows.
__device__ __forceinline__ void swap32(uint32_t& x, uint32_t& y) {   // x's upper 32 lanes for y's lower 32
  const auto p = __builtin_amdgcn_permlane32_swap(x, y, false, false);
  x = p[0];
  y = p[1];
}
__device__ __forceinline__ void swap16(uint32_t& x, uint32_t& y) {   // x's odd rows for y's even rows
  const auto p = __builtin_amdgcn_permlane16_swap(x, y, false, false);
  x = p[0];
  y = p[1];
}
template <int KS, int BITS>
struct KRow {
  static constexpr int kW = BITS / 4;                     // words of a piece
  static constexpr int kFour = BITS == 4 ? KS / 4 * 4 : 0;   // steps read four at a time; the others in twos, the last alone
  uint32_t w[KS][kW];
  __device__ __forceinline__ void load(const char* base, uint32_t off, int qq) {   // (a wave-uniform base takes the offset as it is)
    if constexpr (kFour > 0) {
      const char* p = base + (off + (uint32_t)(16 * qq));
#pragma unroll
      for (int st = 0; st < kFour; st += 4) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(p + 4 * BITS * st);
#pragma unroll
        for (int i = 0; i < 4; ++i) w[st + i][0] = x[i];
      }
    }
    if constexpr (KS - kFour >= 2) {
      const char* p = base + (off + (uint32_t)(2 * BITS * qq));
#pragma unroll
      for (int st = kFour; st + 2 <= KS; st += 2) {
        if constexpr (BITS == 8) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(p + 4 * BITS * st);
#pragma unroll
          for (int i = 0; i < 4; ++i) w[st + i / 2][i % 2] = x[i];
        } else {
          const u32x2 x = *reinterpret_cast<const u32x2*>(p + 4 * BITS * st);
          w[st][0] = x[0];
          w[st + 1][0] = x[1];
        }
      }
    }
    if constexpr (KS % 2 == 1) {
      const Codes8<BITS> c = load_codes8<BITS>(base + (off + (uint32_t)(BITS * qq)) + 4 * BITS * (KS - 1));
#pragma unroll
      for (int i = 0; i < kW; ++i) w[KS - 1][i] = c.w[i];
    }
  }
  __device__ __forceinline__ void arrange() {
#pragma unroll
    for (int st = 0; st < kFour; st += 4) {
      swap32(w[st][0], w[st + 2][0]);
      swap32(w[st + 1][0], w[st + 3][0]);
      swap16(w[st][0], w[st + 1][0]);
      swap16(w[st + 2][0], w[st + 3][0]);
    }
#pragma unroll
    for (int st = kFour; st + 2 <= KS; st += 2)
#pragma unroll
      for (int i = 0; i < kW; ++i) {
        swap16(w[st][i], w[st + 1][i]);
        swap32(w[st][i], w[st + 1][i]);
      }
  }
  __device__ __forceinline__ Codes8<BITS> codes(int st) const {
    Codes8<BITS> c;
#pragma unroll
    for (int i = 0; i < kW; ++i) c.w[i] = w[st][i];
    return c;
  }
};

// ---------------------------------------------------------------------------
// One 256-thread workgroup per item (segment, split, kv head, run of 16-row
// chunks), a resident grid over all items. Wave w's keys are 64 w .. 64 w + 63 of the
// split, lane l's page that of key 64 w + l. K of those keys stays in the wave's
// registers and V of the split in LDS (codes: dequantized once), so that a chunk of
// rows costs its Q^T, its products and the exchange of maxima and weights. Wave w takes
// the dims 16 dt, dt = NJ w .. NJ w + NJ - 1, of P.V. (fp32 rows of more than 128 dims: V
// in two slices, copied for every chunk.) BITS 0: rows of T; 8 or 4: codes.
// Bound by a chunk's chain where many rows share a prefix: it takes a CU about 1.3 us, 48
// products a wave (as long as 0.35 us) among some 330 vector instructions and two
// exchanges. 64 sequences behind 8192 keys, up to 512 of their own: 54 us, in which a SIMD
// issues in 46% of its cycles (vector instructions in 31%), the matrix unit is busy in
// 11%, and a wave waits for half of its time. By latency and bytes where they share
// little. 64 sequences of 32 / 8 heads of 128 in bf16 behind 8192 keys, 256 of their own:
// 63 us with the merge, where every sequence reading its own keys takes 323; without
// the shared keys 24. Codes that nobody shares take longer here than in attn_codes: 64
// sequences of up to 8192 keys of their own 269 us in 8 bits and 242 in 4 instead of
// 150 and 98.
// Of a second half of the grid that takes its items from the last on, loads beside the
// others' products, nothing came (57 -> 59 us), nor of waiting for the next rows in front
// of the stores.
// ---------------------------------------------------------------------------
template <typename T, int D>
constexpr int pages_v_slices() {
  return (kSplit * D * (int)sizeof(T) + (128 << 10) - 1) >> 17;
}
// Workgroups per CU that the registers are held to: two where LDS has room for them. (64
// dims fit three anyway, and held to them are slower, 43 instead of 41 us for 64
// sequences behind 8192 keys; 32 dims gain, 32 instead of 34.5.) Within that only fp32 of
// 256 dims spills, 36 to 52 registers; scalars, 38 to 156 of them, go to the lanes of
// vector registers.
template <typename T, int D>
constexpr int pages_min_blocks() {
  return sizeof(T) == 4 || D > 128 ? 1 : D > 32 ? 2 : 3;
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(256, (pages_min_blocks<T, D>())) void attn_pages(PagesArgs a) {
  typedef typename Frag<T>::type F;
  constexpr int NVP = pages_v_slices<T, D>();
  constexpr int DV = D / NVP;
  typedef KVTile<T, DV> KV;
  constexpr int KT = 4, KS = D / 32;
  constexpr int NDTV = DV / 16, NJ = (NDTV + 3) / 4;
  constexpr int CPW = KV::copies(kSplit) / 4;
  constexpr int kPBytes = 8 * 2 * kWave * 16;             // P.V operands of every 32-key step
  constexpr int kVBytes = kSplit * KV::kRowBytes;
  // Rows of 256 bytes: V fills 64 KB, and with the weights behind it two workgroups
  // would not fit a CU. Its last two steps go to registers and the weights over them.
  constexpr int KEEP = NVP == 1 && kVBytes == (64 << 10) ? 2 : 0;
  constexpr int kPAt = kVBytes - KEEP * 32 * KV::kRowBytes;
  static_assert(DV % 32 == 0 && CPW >= 1 && kPBytes >= KEEP * 32 * KV::kRowBytes, "attn_pages: V slice tiling");
  __shared__ __attribute__((aligned(1024))) char Vs[kPAt + kPBytes];
  __shared__ __attribute__((aligned(16))) float mx[16][4];   // a row's maximum in each wave's keys
  __shared__ __attribute__((aligned(16))) int row_s[16], lim_s[16];
  extern __shared__ int seg_s[];                          // the plan's segments, or their first items
  u32x4* const Ps = reinterpret_cast<u32x4*>(Vs + kPAt);

  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane % 16, qq = lane / 16;
  const int G = a.Hq / a.Hkv, rows1 = a.Tq * G;
  const bool direct = a.nsplit == 1;
  const int page_mask = (1 << a.page_shift) - 1;
  const int dt0 = min(NJ * wave, NDTV - NJ < 0 ? 0 : NDTV - 1);   // this wave's first dim tile (a wave without one repeats the last)

  const int nseg = a.groups + a.B;
  const bool fused = nseg <= kPlanFused;
  const int32_t* seg = a.plan + 2;
  int items, per;
  if (fused) {
    plan_segments<256>(a, seg_s, row_s, items, per);
    items = __builtin_amdgcn_readfirstlane(items);
    per = __builtin_amdgcn_readfirstlane(per);
  } else {
    items = a.plan[0];
    per = a.plan[1];
    if (nseg <= kPlanCached) {
      for (int i = tid; i < nseg; i += 256) seg_s[i] = seg[(int64_t)i * kPlanWords];
      __syncthreads();
    }
  }
  struct Item { int seq0, nseq, split, hk, chunk0, chunks, n_act; };   // n_act < 0: no more items
  auto locate = [&](int item) -> Item {
    if (item < 0) return Item{0, 0, 0, 0, 0, 0, -1};
    // the last segment that starts at or before the item (ones without items share a start with the next)
    int at = 0;
    if (nseg <= kPlanCached) {
      const int words = fused ? kPlanWords : 1;
      for (int i = lane; i < nseg; i += kWave) at += __popcll(__ballot(seg_s[i * words] <= item));   // (starts rise)
      at = __builtin_amdgcn_readfirstlane(at) - 1;
    } else {
      for (int step = 1 << (31 - __builtin_clz(nseg)); step > 0; step >>= 1)
        if (at + step < nseg && load_uniform_i32(uniform_ptr(seg + (int64_t)(at + step) * kPlanWords)) <= item) at += step;
    }
    int w[4];
    if (fused) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = __builtin_amdgcn_readfirstlane(seg_s[at * kPlanWords + i]);
    } else {
      const int32_t* sg = uniform_ptr(seg + (int64_t)at * kPlanWords);
      load_uniform4_i32(sg, sg + 1, sg + 2, sg + 3, w);
    }
    Item it;
    it.seq0 = w[1];
    it.nseq = w[2];
    const int all = (it.nseq * rows1 + 15) / 16, runs = (all + per - 1) / per, each = (all + runs - 1) / runs;   // (even runs)
    const int local = item - w[0], x = local / runs, y = quotient(x, a.Hkv, a.hkv_inv);
    it.chunk0 = (local - x * runs) * each;
    it.chunks = min(each, all - it.chunk0);
    it.hk = x - y * a.Hkv;
    it.split = w[3] + y;
    it.n_act = min(kSplit, pages_len_uniform(a, it.seq0) - it.split * kSplit);
    return it;
  };
  auto page_of = [&](const Item& it) {
    if (it.n_act <= 0) return 0;
    const int pos = it.split * kSplit + min(tid, it.n_act - 1);
    return a.table[(int64_t)it.seq0 * a.table_stride + (pos >> a.page_shift)];
  };

  Item it = locate(dealt(0, items));
  int page = page_of(it);
  for (int round = 1; it.n_act >= 0; ++round) {
    const int seq0 = it.seq0, hk = it.hk, split = it.split, chunk0 = it.chunk0, chunks = it.chunks, n_act = it.n_act;
    const int nrows = it.nseq * rows1, j0 = split * kSplit;   // rows of the segment
    // Row p of the segment: (sequence, head, token).
    auto row_of = [&](int p, int& b, int& h, int& t) {
      const int x = quotient(p, rows1, a.rows1_inv);
      b = seq0 + x;
      p -= x * rows1;
      t = quotient(p, G, a.g_inv);
      h = hk * G + p - t * G;
    };
    if (n_act == 0) {                                     // (direct, an empty sequence) no keys: zeros in this item's rows
      const int rows0 = 16 * chunk0, n = min(16 * chunks, nrows - rows0) * D;   // (at most kPlanMostChunks chunks)
      for (int i = tid; i < n; i += 256) {
        int b, h, t;
        row_of(rows0 + i / D, b, h, t);
        static_cast<T*>(a.out)[(((int64_t)b * a.Hq + h) * a.Tq + t) * D + i % D] = (T)0.0f;
      }
      it = locate(dealt(round, items));
      page = page_of(it);
      continue;
    }

    // A chunk's rows: this lane's Q^T, its index among the outputs (-1: none), and how
    // many keys of the split it may see.
    struct Rows { F qf[KS]; int row, lim; };
    auto request_rows = [&](int chunk, Rows& x) __attribute__((always_inline)) {
      const int p = 16 * chunk + r;
      int b, h, t;
      row_of(min(p, nrows - 1), b, h, t);
      // (strides of Q below 2^32: one product each)
      const T* qrow = static_cast<const T*>(a.q) + ((uint64_t)(uint32_t)b * (uint32_t)a.q_sb + (uint64_t)(uint32_t)h * (uint32_t)a.q_sh +
                                                    (uint64_t)(uint32_t)t * (uint32_t)a.q_st);
#pragma unroll
      for (int st = 0; st < KS; ++st) x.qf[st] = frag_load(qrow + 32 * st + 8 * qq);   // (columns without a row are never stored)
      const int len = pages_len(a, b);
      x.row = p < nrows ? (b * a.Hq + h) * a.Tq + t : -1;
      x.lim = p < nrows ? (a.causal ? len - a.Tq + t + 1 : len) - j0 : 0;
    };
    // This lane's key; the others' offsets come by lane exchanges.
    const int64_t my_page = clamp_page(page, a.num_pages);
    const int64_t my_row = (j0 + min(tid, n_act - 1)) & page_mask;
    const int64_t k_off = my_page * a.k_sp + my_row * a.k_sl, v_off = my_page * a.v_sp + my_row * a.v_sl;
    auto off_of = [&](int64_t off, int l) {
      return (int64_t)((uint64_t)(uint32_t)__shfl((int)(uint32_t)off, l, kWave) |
                       (uint64_t)(uint32_t)__shfl((int)(uint32_t)((uint64_t)off >> 32), l, kWave) << 32);
    };
    const char* kb = uniform_ptr(static_cast<const char*>(a.k) + hk * a.k_sh * (BITS ? 1 : (int)sizeof(T)));
    const char* vb = uniform_ptr(static_cast<const char*>(a.v) + hk * a.v_sh * (BITS ? 1 : (int)sizeof(T)));
    // V of the wave's 64 keys to LDS, codes as the values they stand for.
    auto copy_v = [&](int vp) __attribute__((always_inline)) {
      int l = lane;
      asm volatile("" : "+v"(l));                         // (offsets within tiles are not kept over the items)
      if constexpr (BITS == 0) {
#pragma unroll
        for (int c = 0; c < CPW; ++c) {
          const int f = 64 * c + l, row = f / KV::kCPR, slot = f - row * KV::kCPR;   // of the wave's rows
          const T* vr = reinterpret_cast<const T*>(vb) + off_of(v_off, row) + vp * DV;
          copy_to_lds16(vr + (slot ^ KV::template key<true>(64 * wave + row)) * (16 / (int)sizeof(T)), Vs + 1024 * (wave * CPW + c));
          if (c % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // (a few addresses at a time)
        }
      } else {
        constexpr int PPR = DV / 16;                      // pieces of 16 codes per row
        const int64_t vg_off = my_page * a.vg_sp + my_row * a.vg_sl;
#pragma unroll
        for (int i = 0; i < PPR; ++i) {
          const int f = l + 64 * i, row = f / PPR, dv = (f - row * PPR) * 16, d = dv + vp * DV;
          const Codes16<BITS> c = load_codes16<BITS>(vb + off_of(v_off, row) + d / 8 * BITS);
          const Pair<T> g = load_pair(static_cast<const T*>(a.vg) + hk * a.vg_sh + off_of(vg_off, row) + 2 * (d >> a.gshift));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const F x = dequant_frag<T, BITS>(c.half(h), g);
            if constexpr (sizeof(T) == 2) {
              *reinterpret_cast<u32x4*>(Vs + KV::template off<true>(64 * wave + row, dv / 8 + h)) = __builtin_bit_cast(u32x4, x);
            } else {
              *reinterpret_cast<f32x4*>(Vs + KV::template off<true>(64 * wave + row, dv / 4 + 2 * h)) = x.lo;
              *reinterpret_cast<f32x4*>(Vs + KV::template off<true>(64 * wave + row, dv / 4 + 2 * h + 1)) = x.hi;
            }
          }
        }
      }
    };
    F vf[KEEP ? KEEP : 1][NJ];
    if constexpr (NVP == 1) copy_v(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    Rows rows;
    request_rows(chunk0, rows);
    F kf[KT][KS];
    if constexpr (BITS == 0) {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const T* kr = reinterpret_cast<const T*>(kb) + off_of(k_off, 16 * t + r) + 8 * qq;
#pragma unroll
        for (int st = 0; st < KS; ++st) kf[t][st] = frag_load(kr + 32 * st);
      }
    } else {
      const int64_t kg_off = my_page * a.kg_sp + my_row * a.kg_sl;
      KRow<KS, BITS> kc[KT];
      Pair<T> g[KT][KS];
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        kc[t].load(kb + off_of(k_off, 16 * t + r), 0u, qq);
        const T* kg = static_cast<const T*>(a.kg) + hk * a.kg_sh + off_of(kg_off, 16 * t + r);
#pragma unroll
        for (int st = 0; st < KS; ++st) g[t][st] = load_pair(kg + 2 * (32 * st >> a.gshift));
      }
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        kc[t].arrange();
#pragma unroll
        for (int st = 0; st < KS; ++st) kf[t][st] = dequant_frag<T, BITS>(kc[t].codes(st), g[t][st]);
      }
    }
    asm volatile("" ::: "memory");

    it = locate(dealt(round, items));                   // the next item's pages
    page = page_of(it);
    if constexpr (KEEP > 0) {
      stage_barrier<0>();                                 // V landed
#pragma unroll
      for (int k = 0; k < KEEP; ++k)
#pragma unroll
        for (int j = 0; j < NJ; ++j) vf[k][j] = KV::vfrag(Vs, 32 * (8 - KEEP + k), min(dt0 + j, NDTV - 1), lane);
      stage_barrier<63>();                                // read by everyone
    }

    bool landed = false;
    for (int c = 0; c < chunks; ++c) {
      const int row = rows.row, lim = rows.lim;
      if (!direct && !__ballot(lim > 0)) {                // no partials: the merge reads none (the same in every wave)
        if (c + 1 < chunks) request_rows(chunk0 + c + 1, rows);
        continue;
      }
      float s[KT][4];
      float m = -INFINITY;
      auto scores = [&](auto masked) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < KT; ++t) {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < KS; ++st) acc = mfma_step(kf[t][st], rows.qf[st], acc);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const bool seen = !decltype(masked)::value || 64 * wave + 16 * t + 4 * qq + i < lim;
            s[t][i] = seen ? acc[i] * a.scale_log2 : -INFINITY;
            m = fmaxf(m, s[t][i]);
          }
        }
      };
      if (__ballot(row >= 0 && lim < kSplit)) scores(std::true_type());
      else scores(std::false_type());
      if (c + 1 < chunks) request_rows(chunk0 + c + 1, rows);
      m = quarter_max(m);
      if (qq == 0) mx[r][wave] = m;
      if (tid < 16) {
        row_s[tid] = row;
        lim_s[tid] = lim;
      }
      stage_barrier<63>();
      const f32x4 m4 = *reinterpret_cast<const f32x4*>(mx[r]);
      const i32x4_t arow = *reinterpret_cast<const i32x4_t*>(row_s + 4 * qq);   // the rows of the accumulators, 4 qq + i
      const i32x4_t alim = *reinterpret_cast<const i32x4_t*>(lim_s + 4 * qq);
      m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
      const float msub = m == -INFINITY ? 0.0f : m;       // no visible key: weights 0, not NaN
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float p8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p8[e] = __builtin_amdgcn_exp2f(s[2 * h + e / 4][e % 4] - msub);
        store_pfrag<T>(Ps + (2 * wave + h) * 2 * kWave + lane, kWave, make_pfrag<T>(p8));
      }
      if (!direct && wave == 0 && qq == 0 && lim > 0) a.pm[(int64_t)row * a.nsplit + split] = m;
      const int sum_wave = c & 3;                         // which wave adds up the weights
      f32x4 lsum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int vp = 0; vp < NVP; ++vp) {
        if constexpr (NVP > 1) {
          __syncthreads();                                // every wave is done with the last slice
          copy_v(vp);
          stage_barrier<0>();
        } else if (KEEP == 0 && !landed) {
          landed = true;
          stage_barrier<0>();                             // weights visible, V landed
        } else {
          stage_barrier<63>();
        }
        f32x4 acc[NJ];
        int vl = lane;
        asm volatile("" : "+v"(vl));
        // P.V of this wave's dim tiles; `clean` takes infinities and NaN of V as 0.
        // One wave also adds up the weights, a chain beside the others'.
        auto weigh = [&](bool clean, auto sum) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < kSplit / 32; ++ks) {
            const PFrag<T> pf = load_pfrag<T>(Ps + ks * 2 * kWave + lane, kWave);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              F v = ks < 8 - KEEP ? KV::vfrag(Vs, 32 * ks, min(dt0 + j, NDTV - 1), vl) : vf[ks < 8 - KEEP ? 0 : ks - 8 + KEEP][j];
              if (clean) v = finite_frag(v);
              acc[j] = pv_step<T>(pf, v, acc[j]);
            }
            if constexpr (decltype(sum)::value) lsum = pv_step<T>(pf, ones_frag<T>(), lsum);
            if (ks % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // (or every step's reads are gathered in front, and spill)
          }
        };
        if (vp == 0 && (wave == sum_wave || direct)) weigh(false, std::true_type());
        else weigh(false, std::false_type());
        // A hidden key's weight 0 times an infinity or NaN of its V row is NaN: such a
        // wave weighs again without them and notes the ones its rows see (kSeenTag), which
        // it looks for in the pages.
        float size = 0.0f;                                // (an infinite sum of finite ones costs time only)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) size += fabsf(acc[j][i]);
        if (__ballot(!(size < INFINITY))) {
          weigh(true, std::false_type());
          int dim0 = vp * DV + 16 * dt0 + r;
          asm volatile("" : "+v"(dim0));
          for (int key = 0; key < n_act; ++key) {
            const int pos = j0 + key;
            const int64_t pg = clamp_page(a.table[(int64_t)seq0 * a.table_stride + (pos >> a.page_shift)], a.num_pages);
            const int64_t prow = pos & page_mask;
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              const int dim = min(dim0 + 16 * j, D - 16 + r);
              float x;
              if constexpr (BITS == 0) {
                x = to_f32(reinterpret_cast<const T*>(vb)[pg * a.v_sp + prow * a.v_sl + dim]);
              } else {
                const uint32_t code = (uint8_t)vb[pg * a.v_sp + prow * a.v_sl + dim * BITS / 8];
                const Pair<T> g = load_pair(static_cast<const T*>(a.vg) + hk * a.vg_sh + pg * a.vg_sp + prow * a.vg_sl + 2 * (dim >> a.gshift));
                x = to_f32(to_store<T>(__builtin_fmaf((float)(BITS == 8 ? code : code >> 4 * (dim & 1) & 15u), g.s, g.b)));
              }
              if (fabsf(x) < INFINITY) continue;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key < alim[i]) acc[j][i] = note_seen(acc[j][i], x);
            }
          }
        }
        const uint32_t dim = (uint32_t)(vp * DV + 16 * NJ * wave + r);
        if (direct) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            T* o = static_cast<T*>(a.out) + ((uint64_t)(uint32_t)arow[i] * (uint32_t)D + dim);
            if (arow[i] >= 0)
#pragma unroll
              for (int j = 0; j < NJ; ++j)
                if (NDTV % 4 == 0 || NJ * wave + j < NDTV) o[16 * j] = to_store<T>(only_split(acc[j][i], lsum[i]));
          }
        } else {                                          // (a row's partials: fewer than 2^32 elements)
          const uint32_t row_n = (uint32_t)a.nsplit * (uint32_t)D, at = (uint32_t)split * (uint32_t)D + dim;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float* o = a.pacc + ((uint64_t)(uint32_t)arow[i] * row_n + at);
            if (alim[i] > 0)
#pragma unroll
              for (int j = 0; j < NJ; ++j)
                if (NDTV % 4 == 0 || NJ * wave + j < NDTV) o[16 * j] = acc[j][i];
          }
        }
      }
      if (!direct && wave == sum_wave && r == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (alim[i] > 0) a.pl[(int64_t)arow[i] * a.nsplit + split] = lsum[i];
      }
    }
    stage_barrier<63>();                                  // every wave is done with LDS
  }
}

// ---------------------------------------------------------------------------
// Codes, at most 16 rows a sequence and kv head (a decode step, a few draft tokens):
// the codes of V stay codes in LDS. One 256-thread workgroup per item (sequence,
// split, kv head), neighbouring items on one XCD. Wave w's keys are 64 w .. 64 w + 63
// of the split, lane l's page that of key 64 w + l (read an item ahead), so that a
// wave finds all its rows by lane exchanges; it scores them with K dequantized in
// registers. For P.V wave w takes the dims 16 dt, dt = NJ w .. NJ w + NJ - 1: a
// transposing LDS read gives a lane the codes of 8 keys (4 bits: 16) of one dim, and
// each is dequantized once, with its key's pair from LDS.
// Bound by bytes and latency at 8 bits (a SIMD issues in 66% of its cycles, vector
// instructions in 48%), by issue at 4 (89% and 63%: an fma, half a rounding pair and some
// cutting for every value, most of a step's instructions): 64 sequences of up to 8192
// keys, 32 / 8 heads of 128: 150 us for 8 bits in bf16 (572 MB; a copy takes 112), 98 for 4
// bits in fp16 (303 MB, 59); cards differ, up to 163 and 111. fp32, 8 bits: 251 (606 MB, 119).
// Nothing that follows from the lane alone is kept over the items: at 128 registers it
// goes to scratch memory, and reading it back waits for every copy in flight (110 instead
// of 98 us). What is left there, 8 to 12 bytes a lane, is used in rare paths; scalars, 53
// to 120, go to the lanes of vector registers.
// Codes converted before they go to LDS took 500 and 459, the next item's codes
// requested an item ahead, with two workgroups a CU for the registers, 176 and 136.
// ---------------------------------------------------------------------------
// The tile of V's codes: row r, 16-byte chunk c in slot c ^ key(r) where a row holds a
// power of two of them, so that the rows of a transposing read (32 keys, one chunk)
// fall in distinct banks.
template <int D, int BITS>
struct CodeTile {
  static constexpr int kRowBytes = D * BITS / 8;
  static constexpr int kCPR = kRowBytes / 16;
  static constexpr bool kSwz = (kCPR & (kCPR - 1)) == 0;
  static __device__ __forceinline__ int key(int r) {
    const int x = (r & 7) | (r >> 4 & 1) << 3;
    return !kSwz ? 0 : kCPR == 16 ? x : kCPR == 8 ? x >> 1 : kCPR == 4 ? x >> 2 : kCPR == 2 ? x >> 3 : 0;
  }
  static __device__ __forceinline__ int off(int r, int c) { return r * kRowBytes + ((c ^ key(r)) << 4); }
};

typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2_t lds_i32x2;
// (restrict: see lds_read_tr16)
__device__ __forceinline__ i32x2_t lds_read_tr8(lds_i32x2* __restrict p) { return __builtin_amdgcn_ds_read_tr8_b64_v2i32(p); }
__device__ __forceinline__ i32x2_t lds_read_tr4(lds_i32x2* __restrict p) { return __builtin_amdgcn_ds_read_tr4_b64_v2i32(p); }

// N words of memory that is 4-byte aligned.
template <int N>
__device__ __forceinline__ void load_words(const void* p, uint32_t* w) {
  typedef uint32_t v4 __attribute__((ext_vector_type(4), aligned(4)));
  typedef uint32_t v2 __attribute__((ext_vector_type(2), aligned(4)));
  int i = 0;
#pragma unroll
  for (; i + 4 <= N; i += 4) {
    const v4 x = *reinterpret_cast<const v4*>(static_cast<const char*>(p) + 4 * i);
#pragma unroll
    for (int e = 0; e < 4; ++e) w[i + e] = x[e];
  }
  if constexpr (N % 4 >= 2) {
    const v2 x = *reinterpret_cast<const v2*>(static_cast<const char*>(p) + 4 * i);
    w[i] = x[0];
    w[i + 1] = x[1];
    i += 2;
  }
  if constexpr (N % 2 == 1) w[i] = *reinterpret_cast<const uint32_t*>(static_cast<const char*>(p) + 4 * i);
}

// Rows whose weights a workgroup keeps in LDS (4, 8 or 16).
__host__ __device__ inline int codes_rows(int rows1) { return rows1 <= 4 ? 4 : rows1 <= 8 ? 8 : 16; }

// Workgroups per CU that the registers are held to.
template <typename T, int D, int BITS>
constexpr int codes_min_blocks() {
  return sizeof(T) == 2 && D <= 128 ? (BITS == 4 ? 4 : 3) : 1;
}

template <typename T, int D, int BITS, int GS>
__global__ __launch_bounds__(256, (codes_min_blocks<T, D, BITS>())) void attn_codes(PagesArgs a) {
  typedef typename Frag<T>::type F;
  typedef CodeTile<D, BITS> CT;
  constexpr int KT = 4, KS = D / 32, NDT = D / 16, NJ = (NDT + 3) / 4;
  constexpr int NCOPY = kSplit * CT::kCPR / 64 / 4;       // V copy instructions of a wave
  constexpr int PW = sizeof(T) == 2 ? 1 : 2;              // words of a pair
  constexpr int NG = D / GS;                              // groups of a row
  // Pairs that a wave's dim tiles need: one where they share a group (two tiles from
  // an even one on, four of 64 dims), else one for each or for two of them.
  constexpr int NS = NJ == 3 ? 3 : NJ == 4 && GS == 32 ? 2 : 1;
  __shared__ __attribute__((aligned(1024))) char Vs[kSplit * CT::kRowBytes];
  __shared__ __attribute__((aligned(16))) float vsc[NG][kSplit], vbi[NG][kSplit];   // V's scales (times the codes' factors) and biases
  // (a wave's scales may be too large for that: fp16's are finite times 2^24)
  constexpr bool BIG = BITS == 4 && !std::is_same<T, f16>::value;
  __shared__ int big_s[4];
  __shared__ float mx[4][16];
  extern __shared__ u32x4 Ps[];                           // [step][half][lane row][row of the sequence]

  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane % 16, qq = lane / 16;
  const int G = a.Hq / a.Hkv, rows1 = a.Tq * G;
  // Row p of the sequence is column 4 (p % 4) + p / 4 of the scores, so that up to four
  // rows are the first register of the accumulators' four lane rows.
  const int my_p = r / 4 + r % 4 * 4;
  const int ni = (rows1 + 3) / 4;                         // registers that hold rows
  const int rc = codes_rows(rows1);                       // rows that Ps holds; lanes without one read another's
  const int ps = qq * rc + (my_p & (rc - 1));
  const bool direct = a.nsplit == 1;
  const int page_mask = (1 << a.page_shift) - 1;

  // Item -> (sequence, split, kv head), found from the lengths 64 sequences at a time;
  // a workgroup's items rise.
  int c64 = -1, lo = 0, hi = 0, incl = 0;
  struct Item { int b, split, hk, n_act; };               // n_act < 0: no more items
  auto items_of = [&](int b) { return b < a.B ? (direct ? 1 : (pages_len(a, b) + kSplit - 1) / kSplit) * a.Hkv : 0; };
  auto scan = [&] {
    int l = lane;
    asm volatile("" : "+v"(l));                         // (its addresses are not kept over the items)
    ++c64;
    incl = items_of(64 * c64 + l);
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int up = __shfl_up(incl, off, kWave);
      if (lane >= off) incl += up;
    }
    lo = hi;
    hi = lo + __builtin_amdgcn_readlane(incl, 63);
  };
  scan();
  int items = hi;                                         // of all sequences
  if (a.B > 64) {
    int sum = 0;
    for (int b = tid; b < a.B; b += 256) sum += items_of(b);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, kWave);
    int* part = reinterpret_cast<int*>(&mx[0][0]);
    if (lane == 0) part[wave] = sum;
    __syncthreads();
    items = __builtin_amdgcn_readfirstlane(part[0] + part[1] + part[2] + part[3]);
    __syncthreads();
  }
  auto locate = [&](int item) -> Item {
    while (item >= hi && 64 * (c64 + 1) < a.B) scan();
    if (item < 0) return Item{0, 0, 0, -1};
    const int i = __popcll(__ballot(lo + incl <= item));
    const int local = item - lo - (i ? __builtin_amdgcn_readlane(incl, max(i - 1, 0)) : 0);
    Item it;
    it.b = 64 * c64 + i;
    it.split = quotient(local, a.Hkv, a.hkv_inv);
    it.hk = local - it.split * a.Hkv;
    it.n_act = min(kSplit, pages_len_uniform(a, it.b) - it.split * kSplit);
    return it;
  };
  const int full = items / (int)gridDim.x * (int)gridDim.x;   // items of the rounds that every workgroup has one of
  const int last = dealt(items / (int)gridDim.x, items);
  auto next = [&](int item) { return item + (int)gridDim.x < full ? item + (int)gridDim.x : item < full ? last : -1; };
  auto page_of = [&](const Item& it) {
    if (it.n_act <= 0) return 0;
    const int pos = it.split * kSplit + min(tid, it.n_act - 1);
    return a.table[(int64_t)it.b * a.table_stride + (pos >> a.page_shift)];
  };

  // (token, head) p of sequence b, heads inside tokens.
  auto out_row = [&](int b, int hk, int p) {
    const int x = quotient(p, G, a.g_inv);
    return (b * a.Hq + hk * G + p - x * G) * a.Tq + x;
  };
  auto off_of = [&](uint64_t off, int l) {
    return (uint64_t)(uint32_t)__shfl((int)(uint32_t)off, l, kWave) |
           (uint64_t)(uint32_t)__shfl((int)(uint32_t)(off >> 32), l, kWave) << 32;
  };
  int item = full ? dealt(0, items) : last;
  Item it = locate(item);
  int page = page_of(it);
  for (; it.n_act >= 0;) {
    const int b = it.b, hk = it.hk, j0 = it.split * kSplit, n_act = it.n_act, split = it.split;
    if (n_act == 0) {                                     // (direct, an empty sequence) no keys: zeros
      for (int i = tid; i < rows1 * D; i += 256)
        static_cast<T*>(a.out)[(int64_t)out_row(b, hk, i / D) * D + i % D] = (T)0.0f;
      item = next(item);
      it = locate(item);
      page = page_of(it);
      continue;
    }
    const int total = pages_len_uniform(a, b);

    // Memory requests: pairs of this lane's key, Q^T, K, V. A lane finds its own key's
    // rows; the others' come by lane exchanges.
    const uint32_t my_page = (uint32_t)clamp_page(page, a.num_pages);
    const uint32_t my_row = (j0 + min(tid, n_act - 1)) & page_mask;
    auto row_off = [&](int64_t sp, int64_t sl) { return (uint64_t)my_page * (uint32_t)sp + (uint64_t)my_row * (uint32_t)sl; };
    uint32_t kp[NG][PW], vp[NG][PW];
    load_words<NG * PW>(static_cast<const T*>(a.kg) + hk * a.kg_sh + row_off(a.kg_sp, a.kg_sl), &kp[0][0]);
    load_words<NG * PW>(static_cast<const T*>(a.vg) + hk * a.vg_sh + row_off(a.vg_sp, a.vg_sl), &vp[0][0]);
    F qf[KS];
    {
      int p = min(my_p, rows1 - 1);
      asm volatile("" : "+v"(p));                         // (what follows from lanes alone is not kept over the items: registers)
      const int x = quotient(p, G, a.g_inv);
      const T* qrow = static_cast<const T*>(a.q) + ((uint64_t)(uint32_t)b * (uint32_t)a.q_sb + (uint64_t)(uint32_t)(hk * G + p - x * G) * (uint32_t)a.q_sh +
                                                    (uint64_t)(uint32_t)x * (uint32_t)a.q_st);
#pragma unroll
      for (int st = 0; st < KS; ++st) qf[st] = my_p < rows1 ? frag_load(qrow + 32 * st + 8 * qq) : frag_zero<F>();
    }
    KRow<KS, BITS> kc[KT];
    const char* kb = uniform_ptr(static_cast<const char*>(a.k) + hk * a.k_sh);
    const char* vb = uniform_ptr(static_cast<const char*>(a.v) + hk * a.v_sh);
    // (offsets within tiles are taken from the lane anew for every item: kept over the
    // items they hold registers)
    int l = lane;
    asm volatile("" : "+v"(l));
    auto v_piece = [&](int c, int& row) {                 // of the wave's copy c: its row and 16-byte piece
      if constexpr (CT::kSwz) {                           // (the wave's first row is a multiple of 64, so the keys agree)
        constexpr int kRPC = 64 / CT::kCPR;               // rows of a copy
        row = l / CT::kCPR + kRPC * c;
        return (l % CT::kCPR) ^ CT::key(l / CT::kCPR) ^ (kRPC >= 32 ? 0 : CT::key(kRPC * c & (kRPC >= 8 ? 16 : 23)));
      } else {
        row = (64 * c + l) / CT::kCPR;
        return 64 * c + l - row * CT::kCPR;
      }
    };
    if (a.near) {                                         // pools below 4 GiB: 32-bit offsets
      const uint32_t k_off = my_page * (uint32_t)a.k_sp + my_row * (uint32_t)a.k_sl;
      const uint32_t v_off = my_page * (uint32_t)a.v_sp + my_row * (uint32_t)a.v_sl;
#pragma unroll
      for (int t = 0; t < KT; ++t) kc[t].load(kb, (uint32_t)__shfl((int)k_off, 16 * t + r, kWave), qq);
      asm volatile("" ::: "memory");
#pragma unroll
      for (int c = 0; c < NCOPY; ++c) {
        int row;
        const int piece = v_piece(c, row);
        copy_to_lds16(vb + ((uint32_t)__shfl((int)v_off, row, kWave) + (uint32_t)(piece << 4)), Vs + 1024 * (wave * NCOPY + c));
      }
    } else {
      const uint64_t k_off = row_off(a.k_sp, a.k_sl), v_off = row_off(a.v_sp, a.v_sl);
#pragma unroll
      for (int t = 0; t < KT; ++t) kc[t].load(kb + off_of(k_off, 16 * t + r), 0u, qq);
      asm volatile("" ::: "memory");
#pragma unroll
      for (int c = 0; c < NCOPY; ++c) {
        int row;
        const int piece = v_piece(c, row);
        copy_to_lds16(vb + off_of(v_off, row) + (piece << 4), Vs + 1024 * (wave * NCOPY + c));
      }
    }
    asm volatile("" ::: "memory");
    item = next(item);
    it = locate(item);                   // the next item's pages
    page = page_of(it);

    // V's pairs to LDS. (A wave that holds a scale of 2^100 or more converts its codes.)
    bool k_big = false, v_big = false;
    if constexpr (BIG) {
      float ks = 0.0f, vs = 0.0f;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        ks = fmaxf(ks, fabsf(unpack_pair<T>(kp[g]).s));
        vs = fmaxf(vs, fabsf(unpack_pair<T>(vp[g]).s));
      }
      k_big = __ballot(ks >= 0x1p100f) != 0;
      v_big = __ballot(vs >= 0x1p100f) != 0;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const Pair<T> x = unpack_pair<T>(vp[g]);
      vsc[g][tid] = x.s * (v_big ? 1.0f : code_factor<BITS>(tid));   // (a step's element e is key e of 4 from a multiple of 4 on)
      vbi[g][tid] = x.b;
    }
    if (BIG && lane == 0) big_s[wave] = v_big;
    int lim = 0, row = -1;
    if (my_p < rows1) {
      int p = my_p;
      asm volatile("" : "+v"(p));
      lim = (a.causal ? total - a.Tq + quotient(p, G, a.g_inv) + 1 : total) - j0;
      row = out_row(b, hk, p);
    }
    float s[KT][4];
    float m = -INFINITY;
    auto scores = [&](auto masked, auto big) __attribute__((always_inline)) {
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
        Pair<T> g[NG];
#pragma unroll
        for (int i = 0; i < NG; ++i) {
          uint32_t u[PW];
#pragma unroll
          for (int w = 0; w < PW; ++w) u[w] = (uint32_t)__shfl((int)kp[i][w], 16 * t + r, kWave);
          g[i] = unpack_pair<T>(u);
        }
        kc[t].arrange();
#pragma unroll
        for (int st = 0; st < KS; ++st) {
          const Pair<T> p = g[32 * st / GS];
          F k;
          if constexpr (decltype(big)::value) {
            k = dequant_frag<T, BITS>(kc[t].codes(st), p);
          } else {
            float sc[8], bi[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              sc[e] = p.s * code_factor<BITS>(e);
              bi[e] = p.b;
            }
            k = dequant_scaled8<T, BITS>(kc[t].codes(st), sc, bi);
          }
          acc = mfma_step(k, qf[st], acc);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool seen = !decltype(masked)::value || 64 * wave + 16 * t + 4 * qq + i < lim;
          s[t][i] = seen ? acc[i] * a.scale_log2 : -INFINITY;
          m = fmaxf(m, s[t][i]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // (columns without a row may hold anything)
    if (k_big) scores(std::true_type(), std::true_type());
    else if (__ballot(my_p < rows1 && lim < kSplit)) scores(std::true_type(), std::false_type());
    else scores(std::false_type(), std::false_type());
    m = quarter_max(m);
    // (an address read back from scratch memory here would wait for V's copies)
    int ln = lane;
    asm volatile("" : "+v"(ln));
    if (ln < 16) mx[wave][ln] = m;
    stage_barrier<63>();                                  // (V's copies may still be in flight)
    m = fmaxf(fmaxf(mx[0][ln % 16], mx[1][ln % 16]), fmaxf(mx[2][ln % 16], mx[3][ln % 16]));
    const float msub = m == -INFINITY ? 0.0f : m;         // no visible key: weights 0, not NaN
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float p8[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) p8[e] = __builtin_amdgcn_exp2f(s[2 * h + e / 4][e % 4] - msub);
      if (my_p < rc) store_pfrag<T>(Ps + (2 * wave + h) * 8 * rc + ps, 4 * rc, make_pfrag<T>(p8));
    }
    if (!direct && wave == 0 && qq == 0 && lim > 0) a.pm[(int64_t)row * a.nsplit + split] = m;
    int arow[4], alim[4];                                 // the rows of the accumulators, 4 qq + i
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      arow[i] = -1;
      alim[i] = 0;
      if (i < ni) {
        arow[i] = __shfl(row, 4 * qq + i, kWave);
        alim[i] = __shfl(lim, 4 * qq + i, kWave);
      }
    }
    stage_barrier<0>();                                   // V landed, weights and pairs visible

    f32x4 acc[NJ], lsum = {0.f, 0.f, 0.f, 0.f};
    // P.V of this wave's dim tiles; `clean` takes infinities and NaN of V as 0.
    // The reads of a step are requested a step ahead, codes two steps.
    struct Step {
      PFrag<T> pf;
      float s[NS][8], b[NS][8];
    };
    auto read_step = [&](Step& x, int ks) __attribute__((always_inline)) {
      x.pf = load_pfrag<T>(Ps + ks * 8 * rc + ps, 4 * rc);
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const int g = min((NJ * wave + (NJ == 3 ? 1 : 2) * i) * 16 / GS, NG - 1);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 s4 = *reinterpret_cast<const f32x4*>(&vsc[g][32 * ks + 16 * h + 4 * qq]);
          const f32x4 b4 = *reinterpret_cast<const f32x4*>(&vbi[g][32 * ks + 16 * h + 4 * qq]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x.s[i][4 * h + e] = s4[e];
            x.b[i][4 * h + e] = b4[e];
          }
        }
      }
    };
    // Byte of this lane's part of the first keys' codes of each dim tile; 32 (64) keys
    // further the key repeats.
    int at[NJ];
    {
      int lr = r;
      asm volatile("" : "+v"(lr));                     // (not kept over the items)
      const int key = BITS == 8 ? 4 * qq + (lr >> 1 & 3) + (lr >> 1 & 4) * 4 : 32 * (lr >> 3) + 4 * qq + (lr & 3) + (lr & 4) * 4;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int dt = min(NJ * wave + j, NDT - 1);
        at[j] = BITS == 8 ? CT::off(key, dt) + 8 * (lr & 1) : CT::off(key, dt >> 1) + 8 * (dt & 1);
      }
    }
    auto read_codes = [&](Codes8<BITS> (&c)[2][NJ], int k2) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if constexpr (BITS == 8) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const i32x2_t w = lds_read_tr8((lds_i32x2*)(Vs + at[j] + (64 * k2 + 32 * h) * CT::kRowBytes));
            c[h][j].w[0] = (uint32_t)w[0];
            c[h][j].w[BITS / 4 - 1] = (uint32_t)w[1];
          }
        } else {
          const i32x2_t w = lds_read_tr4((lds_i32x2*)(Vs + at[j] + 64 * k2 * CT::kRowBytes));
          c[0][j].w[0] = (uint32_t)w[0];
          c[1][j].w[0] = (uint32_t)w[1];
        }
      }
    };
    auto step_of = [&](const Step& x, const Codes8<BITS> (&c)[NJ], bool clean, auto big) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int i = NS == 1 ? 0 : j / (NJ == 3 ? 1 : 2);
        F v;
        if constexpr (decltype(big)::value) v = dequant_frag8<T, BITS>(c[j], x.s[i], x.b[i]);
        else v = dequant_scaled8<T, BITS>(c[j], x.s[i], x.b[i]);
        if (clean) v = finite_frag(v);
        acc[j] = pv_step<T>(x.pf, v, acc[j]);             // (a wave without a tile computes the last one, unused)
      }
    };
    // The scale of a key as its pair has it, from LDS.
    auto plain = [&](float sc, int key) { return BIG && big_s[key / 64] ? sc : sc * (1.0f / code_factor<BITS>(key)); };
    auto weigh = [&](bool clean) __attribute__((always_inline)) {   // (rare ones, in little code)
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
      for (int k2 = 0; k2 < kSplit / 64; ++k2) {
        Codes8<BITS> vc[2][NJ];
        Step x;
        read_codes(vc, k2);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          read_step(x, 2 * k2 + h);
#pragma unroll
          for (int i = 0; i < NS; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) x.s[i][e] = plain(x.s[i][e], 64 * k2 + e);
          step_of(x, vc[h], clean, std::true_type());
        }
      }
    };
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (BIG && __builtin_amdgcn_readfirstlane(big_s[0] | big_s[1] | big_s[2] | big_s[3])) {
      weigh(false);
    } else {
      Step st[2];
      Codes8<BITS> vc[2][2][NJ];
      read_codes(vc[0], 0);
      read_step(st[0], 0);
#pragma unroll
      for (int ks = 0; ks < kSplit / 32; ++ks) {
        if (ks % 2 == 0 && ks + 2 < kSplit / 32) read_codes(vc[(ks / 2 + 1) % 2], ks / 2 + 1);
        if (ks + 1 < kSplit / 32) read_step(st[(ks + 1) % 2], ks + 1);
        step_of(st[ks % 2], vc[ks / 2 % 2][ks % 2], false, std::false_type());
        __builtin_amdgcn_sched_barrier(0);                // (or every step's reads are gathered in front, and spill)
      }
    }
    const int sum_wave = NDT < 4 * NJ ? 3 : 0;            // (the wave with the fewest dims adds up the weights)
    if (wave == sum_wave || direct) {
#pragma unroll
      for (int ks = 0; ks < kSplit / 32; ++ks) lsum = pv_step<T>(load_pfrag<T>(Ps + ks * 8 * rc + ps, 4 * rc), ones_frag<T>(), lsum);
    }
    // A hidden key's weight 0 times an infinity or NaN of its V row is NaN: such a
    // wave weighs again without them and notes the ones its rows see (kSeenTag).
    bool finite = true;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) finite = finite && (NJ * wave + j >= NDT || fabsf(acc[j][i]) < INFINITY);
    if (__ballot(!finite)) {
      weigh(true);
      for (int key = 0; key < n_act; ++key) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (NJ * wave + j >= NDT) continue;
          const int dim = 16 * (NJ * wave + j) + r, byte = dim * BITS / 8;
          const uint32_t c = (uint8_t)Vs[CT::off(key, byte >> 4) + (byte & 15)];
          const float code = (float)(BITS == 8 ? c : c >> 4 * (dim & 1) & 15u);
          const float x = to_f32(to_store<T>(__builtin_fmaf(code, plain(vsc[dim / GS][key], key), vbi[dim / GS][key])));
          if (fabsf(x) < INFINITY) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (key < alim[i]) acc[j][i] = note_seen(acc[j][i], x);
        }
      }
    }
    int rr = r;
    asm volatile("" : "+v"(rr));                          // (addresses are not kept over the items)
    const uint32_t dim = (uint32_t)(16 * NJ * wave + rr);
    if (direct) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= ni) continue;
        T* o = static_cast<T*>(a.out) + ((uint64_t)(uint32_t)arow[i] * (uint32_t)D + dim);
        if (arow[i] >= 0)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            if (NDT % 4 == 0 || NJ * wave + j < NDT) o[16 * j] = to_store<T>(only_split(acc[j][i], lsum[i]));
      }
    } else {                                              // (a row's partials: fewer than 2^32 elements)
      const uint32_t row_n = (uint32_t)a.nsplit * (uint32_t)D, at = (uint32_t)split * (uint32_t)D + dim;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (i >= ni) continue;
        float* o = a.pacc + ((uint64_t)(uint32_t)arow[i] * row_n + at);
        if (alim[i] > 0)
#pragma unroll
          for (int j = 0; j < NJ; ++j)
            if (NDT % 4 == 0 || NJ * wave + j < NDT) o[16 * j] = acc[j][i];
      }
    }
    if (!direct && wave == sum_wave && r == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < ni && alim[i] > 0) a.pl[(int64_t)arow[i] * a.nsplit + split] = lsum[i];
    }
    stage_barrier<63>();                                  // every wave is done with Vs, Ps and the pairs
  }
}

// Merges the splits of every row, left to right, and divides. A row's lanes are whole
// 16-lane rows of one wave, kE dims a lane; the partials of 16 splits are requested
// together (decode has few rows: a row's time is its round trips). Lane j of each 16 takes
// split j's maximum and sum: running maxima are a scan, so every split's two factors
// come from all lanes at once, and each one's turn is a product and an fma a dim.
// Bound by round trips: 2048 rows of 34 splits of 128 dims, 35 MB, 8.8 us (13.0 with the
// factors worked out by every lane).
// A split in which the row sees no score above -inf (l = 0 at m = -inf) is passed over.
template <int D>
struct MergeRow {
  static constexpr int kE = D > 128 ? 4 : 2;
  static constexpr int kLanes = D / kE <= 16 ? 16 : D / kE <= 32 ? 32 : 64;
};
// x of lane J of the lane's row of 16.
template <int J>
__device__ __forceinline__ float row_lane(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x150 + J, 0xf, 0xf, false));
}
template <int N, int J = 0, class F>
__device__ __forceinline__ void in_turn(const F& f) {
  if constexpr (J < N) {
    f(std::integral_constant<int, J>());
    in_turn<N, J + 1>(f);
  }
}
// The maximum of lanes 0 .. j of the row of 16, in lane j.
__device__ __forceinline__ float row_scan_max(float x) {
  auto up = [](float x, auto by) {                        // (-inf from before the row)
    return fmaxf(x, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp((int)0xff800000, __builtin_bit_cast(int, x),
                                                                           0x110 + decltype(by)::value, 0xf, 0xf, false)));
  };
  x = up(x, std::integral_constant<int, 1>());
  x = up(x, std::integral_constant<int, 2>());
  x = up(x, std::integral_constant<int, 4>());
  return up(x, std::integral_constant<int, 8>());
}

template <typename T, int D>
__global__ __launch_bounds__(256) void attn_pages_merge(PagesArgs a) {
  constexpr int kE = MergeRow<D>::kE, kLanes = MergeRow<D>::kLanes, kDeep = 16;
  typedef float fE __attribute__((ext_vector_type(kE)));
  const int row0 = (int)(blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes), rows = a.B * a.Hq * a.Tq;   // (b, head, token), the output's order
  int row = min(row0, rows - 1);                          // (lanes without work follow the last)
  if (kLanes == kWave) row = __builtin_amdgcn_readfirstlane(row);
  const int d0 = threadIdx.x % kLanes * kE, d = min(d0, D - kE), j16 = threadIdx.x % 16;
  const int bh = row / a.Tq, t = row - bh * a.Tq;
  const int len = pages_len(a, bh / a.Hq);
  const int seen = a.causal ? len - a.Tq + t + 1 : len;
  int ns = seen > 0 ? (seen + kSplit - 1) / kSplit : 0;
  if (kLanes == kWave) ns = __builtin_amdgcn_readfirstlane(ns);
  float M = -INFINITY, Ls = 0.0f, A[kE];
  uint32_t kinds[kE];
#pragma unroll
  for (int e = 0; e < kE; ++e) A[e] = 0.0f, kinds[e] = 0;
  const float *pm = a.pm + (int64_t)row * a.nsplit, *pl = a.pl + (int64_t)row * a.nsplit;
  const float* pacc = a.pacc + (int64_t)row * a.nsplit * D + d;
  auto batch = [&](int i0, auto all) __attribute__((always_inline)) {
    const int i = min(i0 + j16, ns - 1);
    const float m = pm[i], l = pl[i];
    fE pa[kDeep];
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      pa[j] = *reinterpret_cast<const fE*>(pacc + (int64_t)(decltype(all)::value ? i0 + j : min(i0 + j, ns - 1)) * D);
    const bool live = i0 + j16 < ns && (m > -INFINITY || l != 0.0f);
    const float Mi = fmaxf(M, row_scan_max(live ? m : -INFINITY));            // after split i
    const float Mb = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, M), __builtin_bit_cast(int, Mi), 0x111, 0xf, 0xf, false));   // before it
    const float c_old = live ? __builtin_amdgcn_exp2f(Mb - Mi) : 1.0f, c_new = __builtin_amdgcn_exp2f(m - Mi);
    const float lc = live ? l * c_new : -0.0f;            // (x 1 + -0 is x)
    const float on = live ? 1.0f : 0.0f;
    M = row_lane<15>(Mi);
    float odd = 0.0f;
    auto turn = [&](auto jc, auto every) __attribute__((always_inline)) {
      constexpr int j = decltype(jc)::value;
      const float co = row_lane<j>(c_old), cn = row_lane<j>(c_new);
      const bool in = decltype(every)::value || row_lane<j>(on) != 0.0f;
      Ls = __builtin_fmaf(Ls, co, row_lane<j>(lc));
#pragma unroll
      for (int e = 0; e < kE; ++e) {
        A[e] = __builtin_fmaf(A[e], co, in ? pa[j][e] * cn : -0.0f);
        odd += pa[j][e];                                  // (the last split several times: no matter)
      }
    };
    if (decltype(all)::value && !__ballot(!live)) in_turn<kDeep>([&](auto j) __attribute__((always_inline)) { turn(j, std::true_type()); });
    else in_turn<kDeep>([&](auto j) __attribute__((always_inline)) { turn(j, std::false_type()); });
    if (odd != odd) {                                     // a NaN among them
#pragma unroll
      for (int j = 0; j < kDeep; ++j)
#pragma unroll
        for (int e = 0; e < kE; ++e) kinds[e] |= seen_kinds(pa[j][e]);
    }
  };
  int i0 = 0;
  for (; i0 + kDeep <= ns; i0 += kDeep) batch(i0, std::true_type());
  if (i0 < ns) batch(i0, std::false_type());
  if (row0 >= rows || d0 >= D) return;
  T* o = static_cast<T*>(a.out) + (int64_t)row * D + d;
#pragma unroll
  for (int e = 0; e < kE; ++e)
    o[e] = to_store<T>(kinds[e] ? seen_value(kinds[e], Ls) : Ls != 0.0f ? A[e] / Ls : 0.0f);
}

}  // namespace bi
