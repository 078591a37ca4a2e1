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

__device__ __forceinline__ int pages_len(const PagesArgs& a, int b) {
  return a.kv_lens ? min(max(a.kv_lens[b], 0), a.L) : a.L;
}

// ---------------------------------------------------------------------------
// The plan of a call with shared prefixes: segments (groups, then sequences) with
// the first item of each, and how many 16-row chunks an item takes. One workgroup.
// plan: [0] items in all, [1] chunks of 16 rows an item, [2 ...] for each segment
// (first item, first sequence, sequences, first split, splits).
// Groups are the runs starts[n] .. starts[n + 1] of sequences (clamped, each from
// the last one's end on); one of fewer than two sequences shares nothing. The
// shared splits are whole and lie within the first sequence's own keys.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kPlanRounds = 4;           // items a workgroup of the resident grid gets, at least, where chunks allow
constexpr int kPlanMostChunks = 32;

__device__ __forceinline__ int plan_start(const PagesArgs& a, int n) {
  return a.starts ? min(max(a.starts[n], 0), a.B) : n ? a.B : 0;
}

static __global__ __launch_bounds__(kPlanThreads) void pages_plan_kernel(PagesArgs a, int slots) {
  __shared__ int64_t part[kPlanThreads / kWave];
  __shared__ int64_t total_s;
  __shared__ int carry_s;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  int32_t* seg = a.plan + 2;
  const int rows1 = a.Tq * (a.Hq / a.Hkv);                // rows of one sequence and kv head
  // Sequences: all splits their own to begin with.
  for (int b = tid; b < a.B; b += kPlanThreads) {
    int32_t* s = seg + (int64_t)(a.groups + b) * kPlanWords;
    s[1] = b;
    s[2] = 1;
    s[3] = 0;
    s[4] = max((pages_len(a, b) + kSplit - 1) / kSplit, a.nsplit == 1 ? 1 : 0);   // (one split: its items write the results)
  }
  if (tid == 0) carry_s = 0;
  __syncthreads();
  // Groups, 1024 at a time; ends of earlier ones bound a start from below.
  for (int n0 = 0; n0 < a.groups; n0 += kPlanThreads) {
    const int n = n0 + tid;
    int lo = n < a.groups ? plan_start(a, n) : 0, hi = n < a.groups ? plan_start(a, n + 1) : 0;
    // running maximum of every start up to this one's end
    int run = max(lo, hi);
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int up = __shfl_up(run, off, kWave);
      if (lane >= off) run = max(run, up);
    }
    if (lane == kWave - 1) part[wave] = run;
    __syncthreads();
    int before = carry_s;
    for (int w = 0; w < wave; ++w) before = max(before, (int)part[w]);
    const int up = __shfl_up(run, 1, kWave);
    if (lane > 0) before = max(before, up);
    lo = max(lo, before);                                 // (before: all ends of the groups in front)
    __syncthreads();
    if (tid == kPlanThreads - 1) carry_s = max(before, run);
    if (n < a.groups) {
      int splits = 0;
      if (hi - lo > 1 && a.nsplit > 1) {
        const int want = a.slens ? min(max(a.slens[n], 0), a.L) : a.shared_len;
        splits = min(want, pages_len(a, lo)) / kSplit;
      }
      int32_t* s = seg + (int64_t)n * kPlanWords;
      s[1] = lo;
      s[2] = max(hi - lo, 0);
      s[3] = 0;
      s[4] = splits;
    }
    __syncthreads();
  }
  // Their sequences' own splits begin behind the shared ones.
  for (int n = wave; n < a.groups; n += kPlanThreads / kWave) {
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
  auto chunks_of = [&](const int32_t* s) { return (int64_t)(((int64_t)s[2] * rows1 + 15) / 16); };
  auto sum = [&](int64_t x) -> int64_t {                  // over the workgroup
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor((long long)x, off, kWave);
    __syncthreads();
    if (lane == 0) part[wave] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < kPlanThreads / kWave; ++w) x += part[w];
    return x;
  };
  int64_t units = 0;
  for (int i = tid; i < nseg; i += kPlanThreads) {
    const int32_t* s = seg + (int64_t)i * kPlanWords;
    units += s[4] * chunks_of(s);
  }
  units = sum(units) * a.Hkv;
  const int per = (int)min(max(units / ((int64_t)slots * kPlanRounds), (int64_t)1), (int64_t)kPlanMostChunks);
  // First items: an exclusive scan, 1024 segments at a time.
  int64_t base = 0;
  for (int i0 = 0; i0 < nseg; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int32_t* s = seg + (int64_t)min(i, nseg - 1) * kPlanWords;
    const int64_t items = i < nseg ? s[4] * ((chunks_of(s) + per - 1) / per) * a.Hkv : 0;
    int64_t incl = items;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
      const int64_t up = __shfl_up((long long)incl, off, kWave);
      if (lane >= off) incl += up;
    }
    __syncthreads();
    if (lane == kWave - 1) part[wave] = incl;
    __syncthreads();
    int64_t first = base;
    for (int w = 0; w < wave; ++w) first += part[w];
    if (i < nseg) s[0] = (int32_t)(first + incl - items);
    for (int w = 0; w < kPlanThreads / kWave; ++w) base += part[w];
  }
  if (tid == 0) {
    a.plan[0] = (int32_t)base;
    a.plan[1] = per;
  }
}

// ---------------------------------------------------------------------------
// One 256-thread workgroup per item (segment, split, kv head, run of 16-row
// chunks), a resident grid over all items. Wave w scores keys 64 w .. 64 w + 63
// of the split (K in registers, dequantized there), the maxima are exchanged
// through LDS, each wave leaves its keys' weights there as the operands of the
// P.V steps, and wave w computes the dims 16 dt, dt = NJ w .. NJ w + NJ - 1, from
// the split's V in LDS. BITS 0: rows of T; 8 or 4: codes. MULTI: items of several
// chunks, from the plan; else one chunk of at most 16 rows a sequence, and each
// workgroup finds its items from the lengths.
// ---------------------------------------------------------------------------
template <typename T, int D>
constexpr int pages_v_slices() {
  return (kSplit * D * (int)sizeof(T) + (128 << 10) - 1) >> 17;
}

template <typename T, int D, int BITS, bool MULTI>
__global__ __launch_bounds__(256) void attn_pages(PagesArgs a) {
  typedef typename Frag<T>::type F;
  constexpr int NVP = pages_v_slices<T, D>();
  constexpr int DV = D / NVP;
  typedef KVTile<T, DV> KV;
  constexpr int KT = 4, KS = D / 32;
  constexpr int NDTV = DV / 16, NJ = (NDTV + 3) / 4;
  constexpr int CPW = KV::copies(kSplit) / 4;
  static_assert(DV % 32 == 0 && CPW >= 1, "attn_pages: V slice tiling");
  __shared__ __attribute__((aligned(1024))) char Vs[kSplit * KV::kRowBytes];
  __shared__ u32x4 Ps[8][2][kWave];                       // P.V operands of every 32-key step
  __shared__ float mx[4][16];
  __shared__ int pg[kSplit];                              // page of each key of the split

  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane % 16, qq = lane / 16;
  const int G = a.Hq / a.Hkv, rows1 = a.Tq * G;
  const bool direct = a.nsplit == 1;
  const int page_mask = (1 << a.page_shift) - 1;
  // Neighbouring items on one XCD (workgroups reach the 8 of them in turn): the
  // chunks of one split, and the heads of one page, share its cache.
  const int w0 = (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8);

  int per = 1, items = 0;
  int c64 = -1, lo = 0, hi = 0, incl = 0;                 // MULTI: segments 64 c64 .., else sequences
  const int nseg = MULTI ? a.groups + a.B : a.B;
  if constexpr (MULTI) {
    items = a.plan[0];
    per = a.plan[1];
  }
  for (int item = w0;; item += (int)gridDim.x) {
    int seq0, nseq, split, hk, chunk0;
    if constexpr (MULTI) {
      if (item >= items) break;
      // the last segment that starts at or before the item (ones without items share a start with the next)
      const int32_t* seg = a.plan + 2;
      int at = 0;
      for (int step = 1 << (31 - __builtin_clz(nseg)); step > 0; step >>= 1)
        if (at + step < nseg && seg[(int64_t)(at + step) * kPlanWords] <= item) at += step;
      at = __builtin_amdgcn_readfirstlane(at);
      const int32_t* s = seg + (int64_t)at * kPlanWords;
      seq0 = s[1];
      nseq = s[2];
      const int runs = (int)(((int64_t)nseq * rows1 + 16 * per - 1) / (16 * per));
      int local = item - s[0];
      const int x = local / runs;
      chunk0 = (local - x * runs) * per;
      hk = x % a.Hkv;
      split = s[3] + x / a.Hkv;
    } else {
      while (item >= hi && 64 * (c64 + 1) < nseg) {
        ++c64;
        const int b = 64 * c64 + lane;
        incl = b < nseg ? (direct ? 1 : (pages_len(a, b) + kSplit - 1) / kSplit) * a.Hkv : 0;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
          const int up = __shfl_up(incl, off, kWave);
          if (lane >= off) incl += up;
        }
        lo = hi;
        hi = lo + __builtin_amdgcn_readlane(incl, 63);
      }
      if (item >= hi) break;
      const int i = __popcll(__ballot(lo + incl <= item));
      seq0 = 64 * c64 + i;
      nseq = 1;
      chunk0 = 0;
      const int local = item - lo - (i ? __builtin_amdgcn_readlane(incl, max(i - 1, 0)) : 0);
      hk = local % a.Hkv;
      split = local / a.Hkv;
    }
    seq0 = __builtin_amdgcn_readfirstlane(seq0);
    hk = __builtin_amdgcn_readfirstlane(hk);
    split = __builtin_amdgcn_readfirstlane(split);
    const int nrows = nseq * rows1;                       // of the segment
    const int j0 = split * kSplit;
    const int len0 = __builtin_amdgcn_readfirstlane(pages_len(a, seq0));
    const int n_act = min(kSplit, len0 - j0);
    // Row p of the segment: its index among the outputs, the keys of the split that it may see.
    auto row_of = [&](int p, int& b, int& h, int& t) {
      b = seq0;
      if (MULTI) {
        const int x = p / rows1;
        b += x;
        p -= x * rows1;
      }
      t = p / G;
      h = hk * G + p - t * G;
    };
    if (n_act <= 0) {                                     // (direct, an empty sequence) no keys: zeros
      for (int i = tid; i < nrows * D; i += 256) {
        int b, h, t;
        row_of(i / D, b, h, t);
        static_cast<T*>(a.out)[(((int64_t)b * a.Hq + h) * a.Tq + t) * D + i % D] = (T)0.0f;
      }
      continue;
    }

    {                                                     // pages of the split's keys
      const int pos = j0 + min(tid, n_act - 1);
      pg[tid] = clamp_page(a.table[(int64_t)seq0 * a.table_stride + (pos >> a.page_shift)], a.num_pages);
    }
    __syncthreads();

    auto q_frags = [&](int chunk, F (&qf)[KS]) {
      const int p = 16 * chunk + r;
      int b, h, t;
      row_of(min(p, nrows - 1), b, h, t);
      const T* qrow = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)h * a.q_sh + (int64_t)t * a.q_st;
#pragma unroll
      for (int st = 0; st < KS; ++st) qf[st] = p < nrows ? frag_load(qrow + 32 * st + 8 * qq) : frag_zero<F>();
    };
    F qf[KS];
    q_frags(chunk0, qf);
    F kf[KT][KS];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int key = min(64 * wave + 16 * t + r, n_act - 1);
      const int64_t page = pg[key];
      const int row = (j0 + key) & page_mask;
      if constexpr (BITS == 0) {
        const T* kr = static_cast<const T*>(a.k) + page * a.k_sp + hk * a.k_sh + row * a.k_sl + 8 * qq;
#pragma unroll
        for (int st = 0; st < KS; ++st) kf[t][st] = frag_load(kr + 32 * st);
      } else {
        const char* kr = static_cast<const char*>(a.k) + page * a.k_sp + hk * a.k_sh + row * a.k_sl + qq * BITS;
        const T* kg = static_cast<const T*>(a.kg) + page * a.kg_sp + hk * a.kg_sh + row * a.kg_sl;
#pragma unroll
        for (int st = 0; st < KS; ++st)
          kf[t][st] = dequant_frag<T, BITS>(load_codes8<BITS>(kr + 4 * BITS * st), load_pair(kg + 2 * (32 * st >> a.gshift)));
      }
    }
    auto copy_v = [&](int vp) __attribute__((always_inline)) {
      if constexpr (BITS == 0) {
        auto vrow = [&](int key) {
          return static_cast<const T*>(a.v) + (int64_t)pg[key] * a.v_sp + hk * a.v_sh +
                 (int64_t)((j0 + key) & page_mask) * a.v_sl + vp * DV;
        };
#pragma unroll
        for (int c = 0; c < CPW; ++c) KV::template copy<true>(Vs, wave * CPW + c, vrow, n_act, lane);
      } else {
        constexpr int PPR = DV / 16;                      // pieces of 16 codes per row
#pragma unroll
        for (int i = 0; i < PPR; ++i) {
          const int f = tid + 256 * i, key = f / PPR, d = (f - key * PPR) * 16 + vp * DV;
          const int at = min(key, n_act - 1);
          const int64_t page = pg[at];
          const int row = (j0 + at) & page_mask;
          const char* vr = static_cast<const char*>(a.v) + page * a.v_sp + hk * a.v_sh + row * a.v_sl + d / 8 * BITS;
          const T* vg = static_cast<const T*>(a.vg) + page * a.vg_sp + hk * a.vg_sh + row * a.vg_sl;
          const Codes16<BITS> c = load_codes16<BITS>(vr);
          const Pair<T> g = load_pair(vg + 2 * (d >> a.gshift));
          const int dv = d - vp * DV;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const F x = dequant_frag<T, BITS>(c.half(h), g);
            if constexpr (sizeof(T) == 2) {
              *reinterpret_cast<u32x4*>(Vs + KV::template off<true>(key, dv / 8 + h)) = __builtin_bit_cast(u32x4, x);
            } else {
              *reinterpret_cast<f32x4*>(Vs + KV::template off<true>(key, dv / 4 + 2 * h)) = x.lo;
              *reinterpret_cast<f32x4*>(Vs + KV::template off<true>(key, dv / 4 + 2 * h + 1)) = x.hi;
            }
          }
        }
      }
    };
    if constexpr (NVP == 1) copy_v(0);

    const int chunks = MULTI ? min(per, (nrows - 16 * chunk0 + 15) / 16) : 1;
    for (int c = 0; c < chunks; ++c) {
      const int chunk = chunk0 + c;
      // This lane's row of the scores.
      int lim = 0, row = -1;
      {
        const int p = 16 * chunk + r;
        if (p < nrows) {
          int b, h, t;
          row_of(p, b, h, t);
          const int len = MULTI ? pages_len(a, b) : len0;
          lim = (a.causal ? len - a.Tq + t + 1 : len) - j0;
          row = (b * a.Hq + h) * a.Tq + t;
        }
      }
      const bool any = __ballot(lim > 0) != 0;            // (the same in every wave)
      if (!any && !direct) {
        if (MULTI && c + 1 < chunks) q_frags(chunk + 1, qf);
        continue;
      }
      float s[KT][4];
      float m = -INFINITY;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < KS; ++st) acc = mfma_step(kf[t][st], qf[st], acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[t][i] = 64 * wave + 16 * t + 4 * qq + i < lim ? acc[i] * a.scale_log2 : -INFINITY;
          m = fmaxf(m, s[t][i]);
        }
      }
      if (MULTI && c + 1 < chunks) q_frags(chunk + 1, qf);
      m = quarter_max(m);
      if (qq == 0) mx[wave][r] = m;
      __syncthreads();
      m = fmaxf(fmaxf(mx[0][r], mx[1][r]), fmaxf(mx[2][r], mx[3][r]));
      const float msub = m == -INFINITY ? 0.0f : m;       // no visible key: weights 0, not NaN
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float p8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) p8[e] = __builtin_amdgcn_exp2f(s[2 * h + e / 4][e % 4] - msub);
        const PFrag<T> pf = make_pfrag<T>(p8);
        if constexpr (sizeof(T) == 2) {
          Ps[2 * wave + h][0][lane] = __builtin_bit_cast(u32x4, pf.hi);
          Ps[2 * wave + h][1][lane] = __builtin_bit_cast(u32x4, pf.lo);
        } else {
          Ps[2 * wave + h][0][lane] = __builtin_bit_cast(u32x4, pf.f.lo);
          Ps[2 * wave + h][1][lane] = __builtin_bit_cast(u32x4, pf.f.hi);
        }
      }
      if (!direct && wave == 0 && qq == 0 && lim > 0) a.pm[(int64_t)row * a.nsplit + split] = m;
      int arow[4], alim[4];                               // the rows of the accumulators, 4 qq + i
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        arow[i] = __shfl(row, 4 * qq + i, kWave);
        alim[i] = __shfl(lim, 4 * qq + i, kWave);
      }
      auto p_frag = [&](int ks) {
        PFrag<T> pf;
        const u32x4 x0 = Ps[ks][0][lane], x1 = Ps[ks][1][lane];
        if constexpr (sizeof(T) == 2) {
          pf.hi = __builtin_bit_cast(F, x0);
          pf.lo = __builtin_bit_cast(F, x1);
        } else {
          pf.f.lo = __builtin_bit_cast(f32x4, x0);
          pf.f.hi = __builtin_bit_cast(f32x4, x1);
        }
        return pf;
      };
      const int sum_wave = c & 3;                         // which wave adds up the weights
      f32x4 lsum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int vp = 0; vp < NVP; ++vp) {
        if constexpr (NVP > 1) {
          __syncthreads();                                // every wave is done with the last slice
          copy_v(vp);
        }
        stage_barrier<0>();                               // V landed, weights visible
        f32x4 acc[NJ];
        // P.V of this wave's dim tiles; `clean` takes infinities and NaN of V as 0.
        auto weigh = [&](bool clean, bool sum) __attribute__((always_inline)) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
          for (int ks = 0; ks < kSplit / 32; ++ks) {
            const PFrag<T> pf = p_frag(ks);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              if (NJ * wave + j >= NDTV) continue;
              F v = KV::vfrag(Vs, 32 * ks, NJ * wave + j, lane);
              if (clean) v = finite_frag(v);
              acc[j] = pv_step<T>(pf, v, acc[j]);
            }
            if (sum) lsum = pv_step<T>(pf, ones_frag<T>(), lsum);
          }
        };
        weigh(false, vp == 0 && (wave == sum_wave || direct));
        // A hidden key's weight 0 times an infinity or NaN of its V row is NaN: such a
        // wave weighs again without them and notes the ones its rows see (kSeenTag).
        bool finite = true;
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) finite = finite && (NJ * wave + j >= NDTV || fabsf(acc[j][i]) < INFINITY);
        if (__ballot(!finite)) {
          weigh(true, false);
          for (int key = 0; key < n_act; ++key) {
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              if (NJ * wave + j >= NDTV) continue;
              const int dim = 16 * (NJ * wave + j) + r;
              constexpr int kPer = 16 / (int)sizeof(T);
              const float x = to_f32(reinterpret_cast<const T*>(Vs + KV::template off<true>(key, dim / kPer))[dim % kPer]);
              if (fabsf(x) < INFINITY) continue;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key < alim[i]) acc[j][i] = note_seen(acc[j][i], x);
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (NJ * wave + j >= NDTV) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = vp * DV + 16 * (NJ * wave + j) + r;
            if (direct) {
              if (arow[i] >= 0) static_cast<T*>(a.out)[(int64_t)arow[i] * D + d] = to_store<T>(only_split(acc[j][i], lsum[i]));
            } else if (alim[i] > 0) {
              a.pacc[((int64_t)arow[i] * a.nsplit + split) * D + d] = acc[j][i];
            }
          }
        }
      }
      if (!direct && wave == sum_wave && r == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (alim[i] > 0) a.pl[(int64_t)arow[i] * a.nsplit + split] = lsum[i];
      }
    }
    __syncthreads();                                      // every wave is done with Vs, pg before the next item's
  }
}

// Merges the splits of every row, left to right, and divides: one thread per four
// dims of a row. A split in which the row sees no score above -inf (l = 0 at m =
// -inf) is passed over.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_pages_merge(PagesArgs a) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = id / (D / 4);                       // (b, head, token), the output's order
  if (row >= (int64_t)a.B * a.Hq * a.Tq) return;
  const int d = (int)(id % (D / 4)) * 4;
  const int t = (int)(row % a.Tq), b = (int)(row / a.Tq / a.Hq);
  const int len = pages_len(a, b);
  const int seen = a.causal ? len - a.Tq + t + 1 : len;
  const int ns = seen > 0 ? (seen + kSplit - 1) / kSplit : 0;
  float M = -INFINITY, Ls = 0.0f, A[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t kinds[4] = {0, 0, 0, 0};
  const int64_t p0 = row * a.nsplit;
  for (int i0 = 0; i0 < ns; i0 += 4) {                    // four splits' partials requested together
    float pm[4], pl[4];
    f32x4 pa[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t p = p0 + min(i0 + j, ns - 1);
      pm[j] = a.pm[p];
      pl[j] = a.pl[p];
      pa[j] = *reinterpret_cast<const f32x4*>(a.pacc + p * D + d);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (i0 + j < ns && (pm[j] > -INFINITY || pl[j] != 0.0f)) {
        const float acc[4] = {pa[j][0], pa[j][1], pa[j][2], pa[j][3]};
        merge_split<4>(M, Ls, A, pm[j], pl[j], acc);
      }
    }
    const f32x4 any = (pa[0] + pa[1]) + (pa[2] + pa[3]);  // (the last split several times: no matter)
    const float odd = (any[0] + any[1]) + (any[2] + any[3]);
    if (odd != odd) {                                     // a NaN among them
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) kinds[e] |= seen_kinds(pa[j][e]);
    }
  }
  T* o = static_cast<T*>(a.out) + row * D + d;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    o[e] = to_store<T>(kinds[e] ? seen_value(kinds[e], Ls) : Ls != 0.0f ? A[e] / Ls : 0.0f);
}

}  // namespace bi
