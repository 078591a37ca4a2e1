// bi_attn_mod.h — prefill attention whose scores are capped by a tanh or get a
// distance bias, under a document mask or a prefix mask (ScoreMod,
// bi_attn_common.h). Layouts, tiles and the order of every sum are those of
// attn_prefill_mfma (bi_attn_mfma.h): with nothing to change a score or a mask
// the results are its bits, and a token's are those of the decode kernel. It is
// a text of its own so that the plain kernel's registers stay as they are. 4 x 2048
// tokens, causal, 32 / 8 heads of 128, bf16, capped: 300 us, 457 TFLOP/s (the plain
// kernel 257); vector instructions, some 20 a score, issue in 60% of the SIMDs'
// cycles, the MFMAs are busy in 31%.
//
// Registers: D = 128 takes all 256 in 16 bits, and spills 6 or 7 with a distance bias
// or with a cap above 128 (which runs there: 395 us where smaller caps take 300).
// fp32 spills 36 to 77 at D = 192 (4 x 1024 tokens, 32 / 8 heads, capped 790 us; the
// plain kernel, which spills none, 795) and 554 to 609 at D = 256 (16 / 8 heads: 1294 us;
// the plain kernel, which spills 80 to 103, 740). 16 bits at D = 256, one workgroup a
// CU: 4 x 2048 tokens, 16 / 8 heads, capped 354 us, 389 TFLOP/s (plain 281).
//
//   scores     s = cap tanh(dot scale / cap) - slope |pos_q - key| in log2 units
//              (mod_score). Compiled in, since a branch at every score would
//              stop the pipelined body's MFMAs.
//   prefix     a row's key limit is max(pos_q + 1, prefix): limits still grow
//              with the token, so nothing else changes.
//   documents  the split's document numbers come to LDS with its first K chunk;
//              the splits in front of and behind all whose range of numbers meets
//              the workgroup's are skipped, and one with a single number, the
//              workgroup's own, runs unmasked; the first one's chunks in front of the
//              documents are skipped too. Any numbers are right; sorted ones
//              (documents packed one after another) skip all they can.
//   masked V   a hidden key's weight 0 times an infinity or NaN in its V row
//              would be NaN. Such rows are as good as never there, so the kernel
//              looks at its sums instead: if one is not finite, the workgroup
//              runs again with every split masked, clears such elements in LDS
//              and notes in `poison` which rows see one in which dim, and its
//              kind (kSeenTag's low bits); those get it back at the end.
#pragma once

#include "bi_attn_mfma.h"

namespace bi {

// Keys [0, n) that a (token, head) row may see; a document mask comes on top.
// Grows with the row, so a tile's last row has its largest limit.
template <class Args>
__device__ __forceinline__ int mod_nkeys(const Args& a, const int32_t* docs, int len, int prefix, int G, int npairs,
                                         int pair) {
  if (pair >= npairs) return 0;
  const int end = len - a.Tq + pair / G + 1;            // keys up to the row's own position
  if (end <= 0 && (a.causal || docs)) return 0;
  return a.causal ? max(end, prefix) : len;
}

// Keys per ring chunk: 128 for contiguous caches of narrow rows, else 64.
template <typename T, int D, int MODE>
constexpr int mod_chunk() {
  return MODE == kKvContig && D * (int)sizeof(T) <= (sizeof(T) == 2 ? 128 : 256) ? 128 : 64;
}
// Chunk buffers in the ring: four if they leave the workgroups per CU that the
// registers allow (two up to 16-bit D = 128, else one), else two. Either divides
// the chunks of a whole split, so every split starts in buffer 0.
template <typename T, int D, int MODE>
constexpr int mod_ring() {
  constexpr int budget = sizeof(T) == 2 && D <= 128 && MODE != kKvRowPaged ? 80 << 10 : 160 << 10;
  constexpr int fit = (budget - 64 * D - (11 << 8)) / (mod_chunk<T, D, MODE>() * D * (int)sizeof(T));
  return fit < 4 ? 2 : 4;
}
// Workgroups per CU the registers are held to (see prefill_min_blocks).
template <typename T, int D, int MODE>
constexpr int mod_min_blocks() {
  return sizeof(T) != 2 || D > 128 || MODE == kKvRowPaged ? 1 : 2;
}

// A wave-uniform pointer held in scalar registers, whatever the compiler can prove.
template <typename P>
__device__ __forceinline__ const P* uniform_ptr(const P* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint64_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)u);
  const uint64_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(u >> 32));
  return reinterpret_cast<const P*>(hi << 32 | lo);
}

template <typename T, int D, int MODE, int MOD>
__global__ __launch_bounds__(256, (mod_min_blocks<T, D, MODE>())) void attn_prefill_mod(ModPrefillArgs a) {
  constexpr bool ROWPAGED = MODE == kKvRowPaged, TILED = MODE == kKvTilePaged;
  constexpr bool PIPE = sizeof(T) == 2 && !ROWPAGED;
  constexpr int CH = mod_chunk<T, D, MODE>(), NBUF = mod_ring<T, D, MODE>();
  static_assert(2 * (kSplit / CH) % NBUF == 0, "attn_prefill_mod: ring depth");
  typedef typename Frag<T>::type F;
  typedef KVTile<T, D> KV;
  constexpr int KC = kSplit / CH;                       // chunks per split (of K, then of V)
  constexpr int TPC = CH / 16;                          // 16-key score tiles per chunk
  constexpr int CHB = CH * KV::kRowBytes;               // bytes per chunk
  constexpr int CPW = KV::copies(CH) / 4;               // copy instructions per wave per chunk
  constexpr int NDT = D / 16, KS = D / 32;
  static_assert(CPW >= 1 && (CH == 64 || (CH == 128 && MODE == kKvContig)), "attn_prefill_mod: chunk size");
  // LDS: the ring; the document numbers of this split and the next; for each of 64
  // rows its key limit and document (for the masked splits: a register more would
  // spill, and its reload waits for the copies in flight); the poison, a byte for
  // each of 64 rows and D dims. One array: of several, the compiler tells the reads
  // of each from the copies into it and waits for those in flight at every read.
  constexpr int kDocs = NBUF * CHB, kRows = kDocs + 2 * kSplit * 4, kPoison = kRows + 2 * 64 * 4 + 32;
  __shared__ __attribute__((aligned(1024))) char ring[kPoison + 64 * D];
  int* const split_docs = reinterpret_cast<int*>(ring + kDocs);
  int* const row_nkeys = reinterpret_cast<int*>(ring + kRows);
  int* const row_doc = row_nkeys + 64;
  int* const doc_range = row_doc + 64;
  uint32_t* const poison = reinterpret_cast<uint32_t*>(ring + kPoison);

  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane % 16, qq = lane / 16;
  const int G = a.Hq / a.Hkv;
  const int npairs = a.Tq * G;
  // Work items: a (sequence, kv head) pair's run one after another on one XCD, as in
  // the plain kernel, and share K and V in its L2. But up to 1024 items, two rounds of
  // the chip, run the longest of every pair first, over all XCDs: none waits for one
  // that has the longest sequences. In order / spread: 3 ragged x 500 tokens over up
  // to 4000 keys, 14 / 2 heads of 64, fp16 (330 items): 72.5 / 62.7 us; 4 x 2048, 8 / 8
  // heads of 128, bf16 (1024): 105 / 83; 16 ragged x 500 over up to 4000 keys, 32 / 8
  // heads (4096, whose K and V are read again when spread): 654 / 794.
  const int wgs = (npairs + 63) / 64, pairs_bh = a.Hkv * a.B;
  const int64_t items = (int64_t)wgs * pairs_bh;
  const int64_t per_xcd = (items + 7) / 8;
  const bool spread = items <= 1024;
  const int64_t item = spread ? blockIdx.x : (int64_t)(blockIdx.x % 8) * per_xcd + blockIdx.x / 8;
  if (item >= items) return;                            // uniform per workgroup, before any barrier
  const int wg = wgs - 1 - (int)(spread ? item / pairs_bh : item % wgs);
  const int bh = (int)(spread ? item % pairs_bh : item / wgs);
  const int hk = __builtin_amdgcn_readfirstlane(bh % a.Hkv);
  const int b = __builtin_amdgcn_readfirstlane(bh / a.Hkv);
  const int len = __builtin_amdgcn_readfirstlane(a.kv_lens ? min(max(a.kv_lens[b], 0), a.L) : a.L);
  const int prefix = a.mod.prefix ? min(max(a.mod.prefix[b], 0), len) : 0;
  const int32_t* docs = a.mod.docs ? a.mod.docs + (int64_t)b * a.mod.docs_sb : nullptr;
  auto nkeys_of = [&](int pair) -> int { return mod_nkeys(a, docs, len, prefix, G, npairs, pair); };
  const int maxkeys = nkeys_of(min(64 * wg + 63, npairs - 1));
  const int my_pair = 64 * wg + 16 * wave + r;          // score-layout row of this lane
  const int my_nkeys = nkeys_of(my_pair);
  if (qq == 0) row_nkeys[16 * wave + r] = my_nkeys;     // (read by the wave that wrote it)
  const int my_pos = len - a.Tq + my_pair / G;
  // Every row of the wave sees all keys below this limit (the first row's).
  const int wave_min_nkeys = __builtin_amdgcn_readfirstlane(nkeys_of(64 * wg + 16 * wave));
  float slope2 = 0.0f;
  if constexpr ((MOD & kModBias) != 0) {
    if (a.mod.slopes && my_pair < npairs) slope2 = a.mod.slopes[hk * G + my_pair % G] * kLog2e;
  }
  // The workgroup's smallest and largest document.
  int doc_lo = 0x7fffffff, doc_hi = -0x7fffffff - 1;
  if (docs) {
    if (my_nkeys > 0) doc_lo = doc_hi = docs[my_pos];
    if (qq == 0) row_doc[16 * wave + r] = doc_lo;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
      doc_lo = min(doc_lo, __shfl_xor(doc_lo, off, kWave));
      doc_hi = max(doc_hi, __shfl_xor(doc_hi, off, kWave));
    }
    if (lane == 0) {
      doc_range[wave] = doc_lo;
      doc_range[4 + wave] = doc_hi;
    }
    __syncthreads();
    doc_lo = __builtin_amdgcn_readfirstlane(
        min(min(doc_range[0], doc_range[1]), min(doc_range[2], doc_range[3])));
    doc_hi = __builtin_amdgcn_readfirstlane(
        max(max(doc_range[4], doc_range[5]), max(doc_range[6], doc_range[7])));
  }

  const T* kbase = static_cast<const T*>(a.k);
  const T* vbase = static_cast<const T*>(a.v);
  const T* kb = kbase + (int64_t)b * a.k_sb + (int64_t)hk * a.k_sh;   // contiguous caches
  const T* vb = vbase + (int64_t)b * a.v_sb + (int64_t)hk * a.v_sh;
  F qf[KS];
  {
    const bool ok = my_pair < npairs;
    const T* qrow = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb +
                    (ok ? (int64_t)(hk * G + my_pair % G) * a.q_sh + (int64_t)(my_pair / G) * a.q_st : 0);
#pragma unroll
    for (int st = 0; st < KS; ++st) qf[st] = ok ? frag_load(qrow + 32 * st + 8 * qq) : frag_zero<F>();
  }

  // A split's chunks: K 0 .. n - 1, then V 0 .. n - 1, through the ring; n = KC but
  // for the last split, which has enough for maxkeys.
  const int nsplit = maxkeys > 0 ? (maxkeys + kSplit - 1) / kSplit : 0;
  const int nkc_last = nsplit > 0 ? (maxkeys - (nsplit - 1) * kSplit + CH - 1) / CH : 0;
  // Copy offsets as in the plain kernel: a per-lane byte offset that is the same
  // for every chunk, the rest a wave-uniform row step.
  constexpr bool kFixed = 64 % KV::kCPR == 0;
  constexpr int kRPC = kFixed ? 64 / KV::kCPR : 1;
  constexpr auto period = [](int key_rows) {
    return !kFixed || TILED ? CPW : kRPC >= key_rows ? 1 : key_rows / kRPC < CPW ? key_rows / kRPC : CPW;
  };
  constexpr int kKPeriod = period(KV::template kKeyRows<false>), kVPeriod = period(KV::template kKeyRows<true>);
  constexpr bool kRowPerCopy = KV::kCPR == 64 && !TILED && !ROWPAGED;
  int koff[kKPeriod], voff[kVPeriod];
  if constexpr (!ROWPAGED && !kRowPerCopy) {
    const int c0 = TILED ? 0 : wave * CPW;              // a tile's offsets start at its own first row
#pragma unroll
    for (int i = 0; i < kKPeriod; ++i) koff[i] = KV::template tile_off<false>(c0 + i, lane, a.k_sl);
#pragma unroll
    for (int i = 0; i < kVPeriod; ++i) voff[i] = KV::template tile_off<true>(c0 + i, lane, a.v_sl);
  }
  // Requests the chunk of keys key0 .. key0 + CH - 1 of K (or V) into buffer `slot`.
  auto request = [&](auto is_v, int at, int slot) __attribute__((always_inline)) {
    constexpr bool V = decltype(is_v)::value;
    const int key0 = __builtin_amdgcn_readfirstlane(at);
    const int64_t sl = V ? a.v_sl : a.k_sl;
    char* buf = ring + slot * CHB;
    if constexpr (MODE == kKvContig || MODE == kKvPaged) {
      const int rows = min(CH, len - key0);             // >= 1: chunks start below maxkeys <= len
      const T* base = MODE == kKvContig
                          ? (V ? vb : kb) + (int64_t)key0 * sl
                          : kv_segment<MODE>(a, V ? vbase : kbase, V ? a.v_sb : a.k_sb, V ? a.v_sh : a.k_sh, sl, b, hk, key0);
      const auto rs = buffer_rsrc(base, (int)(rows * sl * (int64_t)sizeof(T)));
      char* dst = buf + 1024 * wave * CPW;
      constexpr int kP = V ? kVPeriod : kKPeriod;
      const int rows_b = kP * kRPC * (int)(sl * (int64_t)sizeof(T));
      if constexpr (kRowPerCopy) {
        int row_b = (int)(sl * (int64_t)sizeof(T)), l = lane;
        asm volatile("" : "+v"(l), "+s"(row_b));        // (not kept live across chunks)
#pragma unroll
        for (int i = 0; i < CPW; ++i)
          copy_to_lds16(rs, ((l ^ KV::template key<V>(wave * CPW + i)) << 4) + (wave * CPW + i) * row_b, dst + 1024 * i);
        return;
      }
#pragma unroll
      for (int i = 0; i < kP; ++i) {
        int o = V ? voff[i % kVPeriod] : koff[i % kKPeriod];
        asm volatile("" : "+v"(o));                     // the stepped offsets are not kept live across chunks
#pragma unroll
        for (int i2 = i; i2 < CPW; i2 += kP) copy_to_lds16(rs, o + i2 / kP * rows_b, dst + 1024 * i2);
      }
    } else if constexpr (TILED) {
      // Wave w copies the chunk's 16-key tile w; a tile past the sequence
      // reads as zero (and its table entry is the last tile's).
      static_assert(!TILED || (CH == 64 && CPW == KV::kTileCopies), "attn_prefill_mod: a tile per wave");
      const int pos = __builtin_amdgcn_readfirstlane(min(key0 + 16 * wave, (len - 1) & ~15));
      const int rows = uniform_clamp(len - key0 - 16 * wave, 16);
      const int e = load_uniform_i32(uniform_ptr(kv_entry(a, b, pos)));
      const auto rs = buffer_rsrc(uniform_ptr(kv_tile(a, V ? vbase : kbase, V ? a.v_sb : a.k_sb, V ? a.v_sh : a.k_sh, sl,
                                                      e, hk, pos)),
                                  (int)(rows * sl * (int64_t)sizeof(T)));
      char* dst = buf + 1024 * wave * CPW;
#pragma unroll
      for (int i = 0; i < CPW; ++i) copy_to_lds16(rs, V ? voff[i % kVPeriod] : koff[i % kKPeriod], dst + 1024 * i);
    } else {
      auto row = [&](int i) {
        return (V ? vbase : kbase) + kv_row_off(a, V ? a.v_sb : a.k_sb, V ? a.v_sh : a.k_sh, sl, b, hk, key0 + i);
      };
#pragma unroll
      for (int i = 0; i < CPW; ++i) KV::template copy<V>(buf, wave * CPW + i, row, len - key0, lane);
    }
  };

  // Splits [sp0, sp1) hold all of the workgroup's documents' keys: 64 splits'
  // ranges tested at once, before the first copy (a vector load inside the loop
  // would make the compiler wait for the copies in flight).
  int sp0 = 0, sp1 = nsplit;
  if (docs) {
    sp0 = nsplit;
    sp1 = 0;
    for (int g = 0; g < nsplit; g += 64) {
      // (lanes past the last split have no vote: documents of both -2^31 and 2^31 - 1
      // meet every range, an empty one too)
      int2 range = {0x7fffffff, -0x7fffffff - 1};
      if (g + lane < nsplit) range = a.mod.ranges[(int64_t)b * ((a.L + kSplit - 1) / kSplit) + g + lane];
      const uint64_t hit = __ballot(g + lane < nsplit && range.y >= doc_lo && range.x <= doc_hi);
      if (hit) {
        sp0 = min(sp0, g + __builtin_ctzll(hit));
        sp1 = g + 64 - __builtin_clzll(hit);
      }
    }
    sp0 = __builtin_amdgcn_readfirstlane(sp0);          // (known to be one for the wave: copies take it so)
    sp1 = __builtin_amdgcn_readfirstlane(sp1);
  }
  auto chunks_of = [&](int sp) { return sp + 1 < nsplit ? KC : nkc_last; };
  // The chunks of split sp0 in front of the documents' first key are left out too,
  // as packed documents begin anywhere in a split: 8192 tokens, 32 / 8 heads of 128,
  // bf16, documents of 100 keys on average 128 -> 112 us, of 700 252 -> 244. Its
  // first buffer, 2 kc0 mod NBUF, lets the next split start in buffer 0.
  int kc0 = 0;
  if (docs && sp0 < sp1) {
    int first = kSplit / 64 - 1;
#pragma unroll
    for (int j = kSplit / 64 - 1; j >= 0; --j) {
      const int key = sp0 * kSplit + 64 * j + lane;
      const int d = docs[min(key, len - 1)];
      if (__ballot(key < len && d >= doc_lo && d <= doc_hi)) first = j;
    }
    kc0 = __builtin_amdgcn_readfirstlane(min(first / (CH / 64), chunks_of(sp0) - 1));
  }
  // Whether the workgroup's only document is split sp's only one.
  auto own_doc = [&](int sp) __attribute__((always_inline)) {
    if (!docs) return true;
    const int32_t* at = reinterpret_cast<const int32_t*>(a.mod.ranges + (int64_t)b * ((a.L + kSplit - 1) / kSplit) + sp);
    return doc_lo == doc_hi && load_uniform_i32(uniform_ptr(at)) == doc_lo &&
           load_uniform_i32(uniform_ptr(at + 1)) == doc_lo;
  };
  // The chunks in the order they are used, requested NBUF - 1 ahead: the next one
  // to request is chunk r_i of split r_sp's K (r_v: of its V), of which r_0 .. r_n -
  // 1 are read, into buffer r_slot; `ahead` of them are requested and not yet
  // opened. A split's document numbers come in front of its first K chunk.
  int r_sp = 0, r_i = 0, r_n = 0, r_slot = 0, ahead = 0, docs_slot = 0;
  bool r_v = false;
  auto request_next = [&]() __attribute__((always_inline)) {
    if (r_sp >= sp1) return;
    const int r_0 = r_sp == sp0 ? kc0 : 0, key0 = r_sp * kSplit + r_i * CH;
    if (docs && !r_v && r_i == r_0) {
      copy_to_lds4(docs + min(r_sp * kSplit + tid, len - 1), split_docs + kSplit * docs_slot + 64 * wave);
      docs_slot ^= 1;
    }
    if (!r_v) request(std::false_type(), key0, r_slot);
    else request(std::true_type(), key0, r_slot);
    r_slot = (r_slot + 1) % NBUF;
    ++ahead;
    if (++r_i == r_n) {
      r_i = r_0;
      if (r_v) {
        r_i = 0;
        r_n = chunks_of(++r_sp);
      }
      r_v = !r_v;
    }
  };
  // Opens the chunk in buffer `slot`: waits until it is there (the copies requested
  // behind it may be in flight) and every wave is done with the one before it,
  // whose buffer takes the next request (`behind`: work on this chunk before that).
  auto open_chunk = [&](int slot, auto behind) __attribute__((always_inline)) {
    --ahead;
    if (NBUF >= 4 && ahead >= 2) stage_barrier<2 * CPW>();
    else if (NBUF >= 4 && ahead >= 1) stage_barrier<CPW>();
    else stage_barrier<0>();
    char* buf = ring + slot * CHB;
    behind(buf);
    request_next();
    return buf;
  };
  int doc_buf = 0;                                      // the split's document numbers
  // The keys of a chunk that the document mask leaves to this lane's row, bit
  // 4 t + i for key 16 t + 4 qq + i.
  auto doc_bits = [&](int kc) __attribute__((always_inline)) {
    const int my_doc = row_doc[16 * wave + r];
    uint32_t ok = 0;
#pragma unroll
    for (int t = 0; t < TPC; ++t) {
      // (a vector type, not int4: its reads carry type information, see lds_read_tr16)
      const u32x4 d = *reinterpret_cast<const u32x4*>(split_docs + kSplit * doc_buf + CH * kc + 16 * t + 4 * qq);
#pragma unroll
      for (int i = 0; i < 4; ++i) ok |= ((int)d[i] == my_doc ? 1u : 0u) << (4 * t + i);
    }
    return ok;
  };
  // The second run: clears the infinities and NaN in the V chunk of keys key0 ..
  // and notes the rows that see them.
  bool careful = false;
  auto clean_v = [&](char* buf, int key0) __attribute__((always_inline)) {
    constexpr int kPer = 16 / (int)sizeof(T);
    for (int f = tid; f < CH * KV::kCPR; f += 256) {
      const int row = f / KV::kCPR, slot = f % KV::kCPR, key = key0 + row;
      T e[kPer];
      u32x4 raw = *reinterpret_cast<u32x4*>(buf + 16 * f);
      __builtin_memcpy(e, &raw, 16);
      bool changed = false;
      for (int j = 0; j < kPer; ++j) {
        const float x = to_f32(e[j]);
        if (fabsf(x) < INFINITY) continue;
        changed = true;
        e[j] = (T)0.0f;
        const int dim = (slot ^ KV::template key<true>(row)) * kPer + j;
        const uint32_t bit = v_kind(x) << (8 * (dim % 4));
        for (int p = 0; p < 64; ++p) {
          if (key >= nkeys_of(64 * wg + p)) continue;
          if (docs && docs[len - a.Tq + (64 * wg + p) / G] != docs[key]) continue;
          atomicOr(&poison[(p * D + dim) / 4], bit);
        }
      }
      if (changed) {
        __builtin_memcpy(&raw, e, 16);
        *reinterpret_cast<u32x4*>(buf + 16 * f) = raw;
      }
    }
    __syncthreads();
  };

  float M[4], Lsum[4];
  f32x4 A[NDT];
  const int kbase0 = KV::kbase(r, qq), vbase0 = KV::vbase(lane);
  // One split: scores of the wave's 16 rows (kept in registers), their maximum
  // and weights, P.V and the weight sum, the merge. PIPE: software-pipelined
  // inside the wave as attn_prefill_mfma's split_body_pipe, whose comment says how.
  auto split_body = [&](const int sp, auto masked) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked)::value > 0, DOCS = decltype(masked)::value > 1;
    const int j0 = sp * kSplit;
    const int nkc = MASKED ? chunks_of(sp) : KC;
    const int kc_0 = DOCS && sp == sp0 ? kc0 : 0, slot_0 = DOCS && sp == sp0 ? (2 * kc0) % NBUF - kc0 : 0;
    float s[16][4];
    float m = -INFINITY;
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      if (kc < kc_0 || kc >= nkc) {
#pragma unroll
        for (int t = 0; t < TPC; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[TPC * kc + t][i] = -INFINITY;
        continue;
      }
      const char* buf = open_chunk((kc + slot_0) % NBUF, [](char*) {});
      const int lim = MASKED ? row_nkeys[16 * wave + r] - (j0 + CH * kc + 4 * qq) : 0;
      const uint32_t seen = DOCS ? doc_bits(kc) : ~0u;
      const float far = (MOD & kModBias) != 0 ? (float)(my_pos - (j0 + CH * kc + 4 * qq)) : 0.0f;
      auto finish = [&](int t, f32x4 dot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // (materialised here: left alone the compiler moves the whole split's score
          // arithmetic behind its last K chunk, away from the MFMAs that hide it, or
          // branches around it for every hidden key)
          const float y = materialize(mod_score<T, MOD>(dot[i], a, slope2, far - (float)(16 * t + i)));
          const float x = (!MASKED || 16 * t + i < lim) && (!DOCS || (seen >> (4 * t + i) & 1u)) ? y : -INFINITY;
          s[TPC * kc + t][i] = x;
          m = fmaxf(m, x);
        }
      };
      if constexpr (PIPE) {
        int ko = kbase0;
        asm volatile("" : "+v"(ko));                    // recomputed per chunk, not kept live across them
        F kf[2][KS];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int st = 0; st < KS; ++st) kf[t][st] = KV::kfrag_at(buf, ko, 16 * t, st);
        f32x4 prev = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < TPC; ++t) {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < KS; ++st) {
            acc = mfma_step(kf[t & 1][st], qf[st], acc);
            if (t + 2 < TPC) kf[t & 1][st] = KV::kfrag_at(buf, ko, 16 * (t + 2), st);
          }
          if (t > 0) finish(t - 1, prev);
          prev = acc;
          __builtin_amdgcn_sched_barrier(0);
        }
        finish(TPC - 1, prev);
      } else {
#pragma unroll
        for (int t = 0; t < TPC; ++t) {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < KS; ++st) acc = mfma_step(KV::kfrag(buf, 16 * t + r, st, qq), qf[st], acc);
          finish(t, acc);
        }
      }
    }
    m = quarter_max(m);
    // Weights exp2(s - m): exactly +0 for a hidden key (s = -inf). A row without a
    // visible key in the split subtracts 0 instead, so that they are 0, not NaN.
    const float msub = m == -INFINITY ? 0.0f : m;
    float mi[4];                                        // accumulator-layout rows' maxima
#pragma unroll
    for (int i = 0; i < 4; ++i) mi[i] = __shfl(m, 4 * qq + i, kWave);
    auto weight_pair = [&](PFrag<T>& pf, int ks, int j) __attribute__((always_inline)) {
      const int t = 2 * ks + j / 2, i = 2 * (j % 2);
      const float p0 = __builtin_amdgcn_exp2f(s[t][i] - msub), p1 = __builtin_amdgcn_exp2f(s[t][i + 1] - msub);
      if constexpr (std::is_same_v<T, f16>) {
        // pfrag_pair's values: p - hi is exact, and v_fma_mix_f32 takes hi unwidened
        // (written out, since the compiler turns the fma back into a widening and a
        // subtraction; it follows the conversion, so nothing reads an exp too early).
        const f16x2_t h = __builtin_convertvector(f32x2_t{p0, p1}, f16x2_t);
        float l0, l1;
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(l0) : "v"(h), "v"(p0));
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(l1) : "v"(h), "v"(p1));
        const f16x2_t l = __builtin_convertvector(f32x2_t{l0, l1}, f16x2_t);
        pf.hi[2 * j] = h[0];
        pf.hi[2 * j + 1] = h[1];
        pf.lo[2 * j] = l[0];
        pf.lo[2 * j + 1] = l[1];
      } else if constexpr (sizeof(T) == 2) {
        pfrag_pair<T>(pf, j, p0, p1);
      } else {
        f32x4& half = j < 2 ? pf.f.lo : pf.f.hi;
        half[i] = p0;
        half[i + 1] = p1;
      }
    };
    f32x4 acc[NDT];
    f32x4 lsum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    PFrag<T> pf;
#pragma unroll
    for (int j = 0; j < 4; ++j) weight_pair(pf, 0, j);
    constexpr int HS = CH / 32, NB = NDT / 2;           // 32-key steps per chunk, dim-tile pairs
    if constexpr (DOCS && PIPE) {                       // (here, where the accumulators take no registers yet)
#pragma unroll
      for (int kc = 1; kc < KC; ++kc) {
        if (kc != kc_0) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) weight_pair(pf, HS * kc, j);
      }
    }
#pragma unroll
    for (int kc = 0; kc < KC; ++kc) {
      if ((DOCS && kc < kc_0) || kc >= nkc) continue;
      const char* buf = open_chunk((nkc - kc_0 + kc + slot_0) % NBUF, [&](char* v) __attribute__((always_inline)) {
        if (MASKED && careful) clean_v(v, j0 + CH * kc);
      });
      if constexpr (PIPE) {
        int vo = vbase0;
        asm volatile("" : "+v"(vo));
        F vf[NDT];
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt) vf[dt] = KV::vfrag_at(buf, vo, 0, dt);
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int h = 0; h < HS; ++h) {
          const int ks = HS * kc + h;
          PFrag<T> after = pf;
#pragma unroll
          for (int b2 = 0; b2 < NB; ++b2) {
            const int d0 = 2 * b2, d1 = 2 * b2 + 1;
            acc[d0] = mfma_step(pf.hi, vf[d0], acc[d0]);
            acc[d1] = mfma_step(pf.hi, vf[d1], acc[d1]);
            acc[d0] = mfma_step(pf.lo, vf[d0], acc[d0]);
            if (h + 1 < HS) vf[d0] = KV::vfrag_at(buf, vo, 32 * (h + 1), d0);
            acc[d1] = mfma_step(pf.lo, vf[d1], acc[d1]);
            if (h + 1 < HS) vf[d1] = KV::vfrag_at(buf, vo, 32 * (h + 1), d1);
            if (b2 == 0) lsum = pv_step<T>(pf, ones_frag<T>(), lsum);
            if (ks + 1 < kSplit / 32) {
#pragma unroll
              for (int j = 4 * b2 / NB; j < 4 * (b2 + 1) / NB; ++j) weight_pair(after, ks + 1, j);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          pf = after;
        }
        __builtin_amdgcn_s_setprio(0);
      } else {
#pragma unroll
        for (int h = 0; h < HS; ++h) {
          const int ks = HS * kc + h;
          if (ks > 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) weight_pair(pf, ks, j);
          }
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int dt = 0; dt < NDT; ++dt) acc[dt] = pv_step<T>(pf, KV::vfrag(buf, 32 * h, dt, lane), acc[dt]);
          __builtin_amdgcn_s_setprio(0);
          lsum = pv_step<T>(pf, ones_frag<T>(), lsum);
        }
      }
    }
    // Merge into the running state (accumulator layout: rows 4 qq + i). A row
    // that sees no key of the split skips it.
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (merge_split's operations; a row that skips the split multiplies by 1 and
      // adds -0 instead of branching, which leaves its state's every bit)
      const bool sees = mi[i] > -INFINITY || lsum[i] != 0.0f;
      const float top = sees ? fmaxf(M[i], mi[i]) : M[i];
      const float c_old = sees ? __builtin_amdgcn_exp2f(M[i] - top) : 1.0f;
      const float c_new = sees ? __builtin_amdgcn_exp2f(mi[i] - top) : -0.0f;
      Lsum[i] = __builtin_fmaf(Lsum[i], c_old, lsum[i] * c_new);
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) A[dt][i] = __builtin_fmaf(A[dt][i], c_old, acc[dt][i] * c_new);
      M[i] = top;
    }
  };

  for (;;) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      M[i] = -INFINITY;
      Lsum[i] = 0.0f;
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) A[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    r_sp = sp0;
    r_i = kc0;
    r_n = chunks_of(r_sp);
    r_slot = (2 * kc0) % NBUF;
    r_v = false;
    ahead = docs_slot = doc_buf = 0;
#pragma unroll
    for (int c = 0; c < NBUF - 1; ++c) request_next();
    for (int sp = sp0; sp < sp1; ++sp) {
      if (sp * kSplit + kSplit <= wave_min_nkeys && !careful && own_doc(sp))
        split_body(sp, std::integral_constant<int, 0>());
      else if (!docs) split_body(sp, std::integral_constant<int, 1>());
      else split_body(sp, std::integral_constant<int, 2>());
      doc_buf ^= 1;
    }
    bool finite = true;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (64 * wg + 16 * wave + 4 * qq + i >= npairs) continue;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) finite = finite && fabsf(A[dt][i]) < INFINITY;
    }
    if (careful) break;
    const bool bad = __ballot(!finite) != 0;            // (the library's vote would be a second LDS array)
    if (lane == 0) doc_range[wave] = bad ? 1 : 0;
    __syncthreads();
    if (!__builtin_amdgcn_readfirstlane(doc_range[0] | doc_range[1] | doc_range[2] | doc_range[3])) break;
    careful = true;
    for (int i = tid; i < 16 * D; i += 256) poison[i] = 0;
    __syncthreads();
  }

#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 16 * wave + 4 * qq + i, pair = 64 * wg + row;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const float x = materialize(A[dt][i] / Lsum[i]);
      A[dt][i] = Lsum[i] != 0.0f ? x : 0.0f;            // no key: 0
    }
    if (careful) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const int at = row * D + 16 * dt + r;
        const uint32_t kinds = poison[at / 4] >> (8 * (at % 4)) & 7u;
        if (kinds) A[dt][i] = seen_value(kinds, Lsum[i]);
      }
    }
    if (pair >= npairs) continue;
    T* o = static_cast<T*>(a.out) +
           ((((int64_t)b * a.Hq + hk * G + pair % G) * a.Tq) + pair / G) * D + r;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) o[16 * dt] = to_store<T>(A[dt][i]);
  }
}

// ---------------------------------------------------------------------------
// Few rows: one 256-thread workgroup per (sequence, kv head, 16 (token, head)
// rows, split), so that a short chunk against a long cache has as many
// workgroups as there are splits instead of walking them one after another.
// Wave w scores keys 64 w .. 64 w + 63 (K in registers), the split's maximum is
// exchanged through LDS, each wave writes its keys' weights there, and wave w
// computes P.V of dims 16 dt, dt = w, w + 4, ..., from the split's V in LDS
// (attn_decode_mfma's scheme with rows for heads). Writes (m, l, acc) of its
// split; attn_rows_combine merges them in order, so the results are the bits of
// attn_prefill_mod. LDS is up to 64 KB of the split's V and 16 KB of weights, the
// wave maxima inside them: two workgroups per CU.
// ---------------------------------------------------------------------------
// V slices of 64 KB at most, copied one after another, so that two workgroups
// share a CU and one computes while the other's K and V come: fp32, 2 x 601 tokens,
// 8 / 8 heads of 128, 84 -> 69 us against the whole 128 KB at once.
template <typename T, int D>
constexpr int rows_v_slices() {
  return (kSplit * D * (int)sizeof(T) + (64 << 10) - 1) >> 16;
}

template <typename T, int D, int MODE>
__global__ __launch_bounds__(256) void attn_rows_mod(ModRowsArgs a) {
  constexpr bool ROWPAGED = MODE == kKvRowPaged, TILED = MODE == kKvTilePaged;
  typedef typename Frag<T>::type F;
  constexpr int NVP = rows_v_slices<T, D>();
  constexpr int DV = D / NVP;                           // dims per V slice
  typedef KVTile<T, DV> KV;
  constexpr int KT = 4, KS = D / 32;                    // score tiles per wave
  constexpr int NDTV = DV / 16, NJ = (NDTV + 3) / 4;    // P.V dim tiles per slice, per wave
  constexpr int CPW = KV::copies(kSplit) / 4;           // V copy instructions per wave and slice
  static_assert(DV % 16 == 0 && CPW >= 1 && CPW < 64, "attn_rows_mod: V slice tiling");
  __shared__ __attribute__((aligned(1024))) char Vs[kSplit * KV::kRowBytes];
  __shared__ __attribute__((aligned(16))) float Ps[16][kSplit];

  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane % 16, qq = lane / 16;
  const int G = a.Hq / a.Hkv, npairs = a.Tq * G;
  // Items (b, hk, split, row chunk) in that nesting order, a contiguous range of
  // them per XCD: the row chunks that read one split's K and V share an L2.
  // (In 32 bits, as the host keeps the items below 2^31: a table wider than its
  // sequences has many workgroups that only find out that they have no keys. 4 x 16
  // tokens, 32 / 8 heads of 128, bf16, 300 keys in tables of 512 / 32768: 20.8 / 43.5 us
  // with 64-bit divisions, 20.8 / 38.8 so.)
  const unsigned nchunks = (unsigned)(npairs + 15) / 16, nsplits = (unsigned)a.nsplit, nhk = (unsigned)a.Hkv;
  const unsigned items = nchunks * nsplits * nhk * (unsigned)a.B;
  const unsigned per_xcd = (items + 7) / 8;
  const unsigned item = blockIdx.x % 8 * per_xcd + blockIdx.x / 8;
  if (blockIdx.x / 8 >= per_xcd || item >= items) return;
  const unsigned at = item / nchunks, pair_bh = at / nsplits;
  const int chunk = __builtin_amdgcn_readfirstlane((int)(item - at * nchunks));
  const int split = __builtin_amdgcn_readfirstlane((int)(at - pair_bh * nsplits));
  const int hk = __builtin_amdgcn_readfirstlane((int)(pair_bh % nhk));
  const int b = __builtin_amdgcn_readfirstlane((int)(pair_bh / nhk));
  const int len = __builtin_amdgcn_readfirstlane(a.kv_lens ? min(max(a.kv_lens[b], 0), a.L) : a.L);
  const int prefix = a.mod.prefix ? min(max(a.mod.prefix[b], 0), len) : 0;
  const int32_t* docs = a.mod.docs ? a.mod.docs + (int64_t)b * a.mod.docs_sb : nullptr;
  auto nkeys_of = [&](int pair) -> int { return mod_nkeys(a, docs, len, prefix, G, npairs, pair); };
  const int j0 = split * kSplit;
  const int maxkeys = nkeys_of(min(16 * chunk + 15, npairs - 1));
  const bool direct = a.nsplit == 1;                    // one split: the results themselves, nothing to merge
  // Index of a row's partial: rows in the output's order, splits inside them.
  auto partial = [&](int p) -> int64_t {
    return ((((int64_t)b * a.Hq + hk * G + p % G) * a.Tq) + p / G) * a.nsplit + split;
  };
  if (j0 >= maxkeys) {                                  // the merge reads no such split of these rows
    if (direct) {
      for (int i = tid; i < 16 * D; i += 256)
        if (16 * chunk + i / D < npairs)
          static_cast<T*>(a.out)[partial(16 * chunk + i / D) * D + i % D] = (T)0.0f;
    }
    return;
  }
  const int n_act = __builtin_amdgcn_readfirstlane(min(kSplit, maxkeys - j0));
  const int pair = 16 * chunk + r;                      // score-layout row of this lane
  const int lim = nkeys_of(pair) - j0;                  // keys of the split it may see
  const int pos = len - a.Tq + pair / G;
  float slope2 = 0.0f;
  if (a.mod.slopes && pair < npairs) slope2 = a.mod.slopes[hk * G + pair % G] * kLog2e;
  // Document mask: bit 4 t + i: the lane's row is of key 64 wave + 16 t + 4 qq + i's document.
  unsigned seen = ~0u;
  if (docs) {
    seen = 0;
    const bool row = lim > -j0;                         // a row that exists (its position has a document)
    const int mine = row ? docs[pos] : 0;
#pragma unroll
    for (int t = 0; t < KT; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        seen |= (row && docs[j0 + min(64 * wave + 16 * t + 4 * qq + i, n_act - 1)] == mine ? 1u : 0u) << (4 * t + i);
    // (the vote goes through Ps: the library's own would take LDS past 80 KB)
    const bool hit = __ballot(seen != 0) != 0;
    if (lane == 0) Ps[0][wave] = hit ? 1.0f : 0.0f;
    __syncthreads();
    const float any = Ps[0][0] + Ps[0][1] + Ps[0][2] + Ps[0][3];
    __syncthreads();
    if (any == 0.0f) {
      if (direct) {
        for (int i = tid; i < 16 * D; i += 256)
          if (16 * chunk + i / D < npairs)
            static_cast<T*>(a.out)[partial(16 * chunk + i / D) * D + i % D] = (T)0.0f;
      } else if (tid < 16 && 16 * chunk + tid < npairs) {
        a.pm[partial(16 * chunk + tid)] = NAN;           // (no acc is written: the merge reads none)
        a.pl[partial(16 * chunk + tid)] = 0.0f;
      }
      return;
    }
  }

  // Memory requests, in this order: Q^T, this wave's K rows, its V copies. A
  // wave's keys are one 64-key segment or four 16-key tiles, clamped to the last
  // active one (attn_decode_mfma).
  F qf[KS];
  {
    const bool ok = pair < npairs;
    const T* qrow = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb +
                    (ok ? (int64_t)(hk * G + pair % G) * a.q_sh + (int64_t)(pair / G) * a.q_st : 0);
#pragma unroll
    for (int st = 0; st < KS; ++st) qf[st] = ok ? frag_load(qrow + 32 * st + 8 * qq) : frag_zero<F>();
  }
  const T* kbase = static_cast<const T*>(a.k);
  const T* vbase = static_cast<const T*>(a.v);
  const int seg = __builtin_amdgcn_readfirstlane(min(wave, (n_act - 1) >> 6));
  const T* kseg = kbase;
  const T* vseg = vbase;
  int ktile[4], entry[4];                               // TILED: first key and table entry of each tile
  if constexpr (TILED) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      ktile[t] = __builtin_amdgcn_readfirstlane(min(64 * wave + 16 * t, (n_act - 1) & ~15));
      entry[t] = load_uniform_i32(uniform_ptr(kv_entry(a, b, j0 + ktile[t])));
    }
  } else if constexpr (MODE == kKvPaged) {
    const int key0 = j0 + 64 * seg;
    const int64_t page = clamp_page(load_uniform_i32(uniform_ptr(kv_entry(a, b, key0))), a.num_pages);
    const int64_t row = key0 & ((1 << a.page_shift) - 1);
    kseg = uniform_ptr(kbase + page * a.k_sb + hk * a.k_sh + row * a.k_sl);
    vseg = uniform_ptr(vbase + page * a.v_sb + hk * a.v_sh + row * a.v_sl);
  } else if constexpr (MODE == kKvContig) {
    kseg = uniform_ptr(kv_segment<MODE>(a, kbase, a.k_sb, a.k_sh, a.k_sl, b, hk, j0 + 64 * seg));
    vseg = uniform_ptr(kv_segment<MODE>(a, vbase, a.v_sb, a.v_sh, a.v_sl, b, hk, j0 + 64 * seg));
  }
  F kf[KT][KS];
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int key = min(64 * wave + 16 * t + r, n_act - 1);
    const T* kr;
    if constexpr (TILED)
      kr = kv_tile(a, kbase, a.k_sb, a.k_sh, a.k_sl, entry[t], hk, j0 + ktile[t]) +
           (int64_t)min(r, n_act - 1 - ktile[t]) * a.k_sl;
    else if constexpr (ROWPAGED) kr = kbase + kv_row_off(a, a.k_sb, a.k_sh, a.k_sl, b, hk, j0 + key);
    else kr = kseg + (int64_t)(key - 64 * seg) * a.k_sl;
#pragma unroll
    for (int st = 0; st < KS; ++st) kf[t][st] = frag_load(kr + 32 * st + 8 * qq);
  }
  asm volatile("" ::: "memory");
  constexpr bool kVFixed = (MODE == kKvContig || MODE == kKvPaged) && (64 % KV::kCPR) == 0;
  constexpr int kRowsPerCopy = kVFixed ? 64 / KV::kCPR : 1;
  constexpr int kKeyRows = KV::template kKeyRows<true>;
  constexpr int kVPeriod = TILED ? KV::kTileCopies : kRowsPerCopy >= kKeyRows ? 1 : kKeyRows / kRowsPerCopy;
  auto copy_v = [&](int vp) __attribute__((always_inline)) {
    const int vbytes = vp * DV * (int)sizeof(T);
    const int left = n_act - 64 * wave;                 // active rows from this wave's first
    if constexpr (kVFixed) {
      const auto rs = buffer_rsrc(vseg, (int)(uniform_clamp(left, 64) * a.v_sl * (int64_t)sizeof(T)));
      const int v_step = kVPeriod * kRowsPerCopy * (int)(a.v_sl * (int64_t)sizeof(T));
#pragma unroll
      for (int c = 0; c < CPW; ++c)
        copy_to_lds16(rs, KV::template tile_off<true>(c % kVPeriod, lane, a.v_sl) + (c / kVPeriod) * v_step + vbytes,
                      Vs + 1024 * (wave * CPW + c));
    } else if constexpr (TILED) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const auto rs = buffer_rsrc(uniform_ptr(kv_tile(a, vbase, a.v_sb, a.v_sh, a.v_sl, entry[t], hk, j0 + ktile[t])),
                                    (int)(uniform_clamp(left - 16 * t, 16) * a.v_sl * (int64_t)sizeof(T)));
#pragma unroll
        for (int c = 0; c < KV::kTileCopies; ++c)
          copy_to_lds16(rs, KV::template tile_off<true>(c, lane, a.v_sl) + vbytes,
                        Vs + 1024 * (wave * CPW + KV::kTileCopies * t + c));
      }
    } else {
      auto vrow = [&](int key) {
        if constexpr (ROWPAGED) return vbase + kv_row_off(a, a.v_sb, a.v_sh, a.v_sl, b, hk, j0 + key) + vp * DV;
        else return vseg + (int64_t)(key - 64 * seg) * a.v_sl + vp * DV;
      };
#pragma unroll
      for (int c = 0; c < CPW; ++c) KV::template copy<true>(Vs, wave * CPW + c, vrow, n_act, lane);
    }
  };
  copy_v(0);

  float s[KT][4];
  float m = -INFINITY;
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int st = 0; st < KS; ++st) acc = mfma_step(kf[t][st], qf[st], acc);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = 64 * wave + 16 * t + 4 * qq + i;
      const float far = (float)(pos - j0 - key);
      const float y = a.mod.cap_log2 != 0.0f ? mod_score<T, (kModAny | kModCap | kModBias)>(acc[i], a, slope2, far)
                                             : mod_score<T, (kModAny | kModBias)>(acc[i], a, slope2, far);
      s[t][i] = key < lim && (seen >> (4 * t + i) & 1u) ? y : -INFINITY;
      m = fmaxf(m, s[t][i]);
    }
  }
  m = quarter_max(m);
  if (qq == 0) Ps[0][16 * wave + r] = m;
  stage_barrier<CPW>();                                 // the wave maxima visible; V copies may still be in flight
  m = fmaxf(fmaxf(Ps[0][r], Ps[0][16 + r]), fmaxf(Ps[0][32 + r], Ps[0][48 + r]));
  stage_barrier<CPW>();                                 // read by everyone: the weights go over them
  const float msub = m == -INFINITY ? 0.0f : m;         // no visible key: weights 0, not NaN
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    f32x4 p;
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(s[t][i] - msub);
    *reinterpret_cast<f32x4*>(&Ps[r][64 * wave + 16 * t + 4 * qq]) = p;
  }
  if (!direct && wave == 0 && qq == 0 && pair < npairs) a.pm[partial(pair)] = m;
  stage_barrier<0>();                                   // V landed, weights visible

  f32x4 lsum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int vp = 0; vp < NVP; ++vp) {
    if (vp > 0) {
      __syncthreads();                                  // every wave is done with the previous slice
      copy_v(vp);
      stage_barrier<0>();
    }
    f32x4 acc[NJ];
    // P.V of this wave's dim tiles; `clean` takes infinities and NaN of V as 0.
    auto weigh = [&](bool clean, bool sum) __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
      for (int ks = 0; ks < kSplit / 32; ++ks) {
        const f32x4 x0 = *reinterpret_cast<const f32x4*>(&Ps[r][32 * ks + 4 * qq]);
        const f32x4 x1 = *reinterpret_cast<const f32x4*>(&Ps[r][32 * ks + 16 + 4 * qq]);
        const float p8[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
        const PFrag<T> pf = make_pfrag<T>(p8);
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (wave + 4 * j >= NDTV) continue;
          F v = KV::vfrag(Vs, 32 * ks, wave + 4 * j, lane);
          if (clean) v = finite_frag(v);
          acc[j] = pv_step<T>(pf, v, acc[j]);
        }
        if (sum) lsum = pv_step<T>(pf, ones_frag<T>(), lsum);
      }
    };
    weigh(false, vp == 0 && (wave == 0 || direct));
    // A hidden key's weight 0 times an infinity or NaN of its V row is NaN: such a
    // wave weighs again without them and notes the ones its rows see (kSeenTag).
    bool finite = true;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) finite = finite && (wave + 4 * j >= NDTV || fabsf(acc[j][i]) < INFINITY);
    if (__ballot(!finite)) {
      weigh(true, false);
      for (int key = 0; key < n_act; ++key) {
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          if (wave + 4 * j >= NDTV) continue;
          const int dim = 16 * (wave + 4 * j) + r;
          constexpr int kPer = 16 / (int)sizeof(T);
          const float x = to_f32(reinterpret_cast<const T*>(Vs + KV::template off<true>(key, dim / kPer))[dim % kPer]);
          if (fabsf(x) < INFINITY) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int p = 16 * chunk + 4 * qq + i;
            if (j0 + key < nkeys_of(p) && (!docs || docs[j0 + key] == docs[len - a.Tq + p / G]))
              acc[j][i] = note_seen(acc[j][i], x);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if (wave + 4 * j >= NDTV) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = 16 * chunk + 4 * qq + i;
        if (p >= npairs) continue;
        const int64_t at = partial(p) * D + vp * DV + 16 * (wave + 4 * j) + r;
        if (direct)
          static_cast<T*>(a.out)[at] = to_store<T>(only_split(acc[j][i], lsum[i]));
        else
          a.pacc[at] = acc[j][i];
      }
    }
  }
  if (!direct && wave == 0 && r == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = 16 * chunk + 4 * qq + i;
      if (p < npairs) a.pl[partial(p)] = lsum[i];
    }
  }
}

// Merges the splits of every row that attn_rows_mod left, left to right, and
// divides: one thread per four dims of a row. A split in which the row sees
// nothing (l = 0 at m = -inf) is passed over; one at m = NaN has no acc.
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_rows_combine(ModRowsArgs a) {
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = id / (D / 4);                     // (b, head, token), the output's order
  if (row >= (int64_t)a.B * a.Hq * a.Tq) return;
  const int d = (int)(id % (D / 4)) * 4;
  const int t = (int)(row % a.Tq), b = (int)(row / a.Tq / a.Hq);
  const int len = a.kv_lens ? min(max(a.kv_lens[b], 0), a.L) : a.L;
  const int prefix = a.mod.prefix ? min(max(a.mod.prefix[b], 0), len) : 0;
  const int ns = (mod_nkeys(a, a.mod.docs, len, prefix, 1, a.Tq, t) + kSplit - 1) / kSplit;
  float M = -INFINITY, Ls = 0.0f, A[4] = {0.f, 0.f, 0.f, 0.f};
  uint32_t kinds[4] = {0, 0, 0, 0};
  const int64_t p0 = row * a.nsplit;
  for (int i0 = 0; i0 < ns; i0 += 4) {                  // four splits' partials requested together
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
    if (odd != odd) {                                   // a NaN among them
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) kinds[e] |= pm[j] == pm[j] ? seen_kinds(pa[j][e]) : 0u;
    }
  }
  T* o = static_cast<T*>(a.out) + row * D + d;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    o[e] = to_store<T>(kinds[e] ? seen_value(kinds[e], Ls) : Ls != 0.0f ? A[e] / Ls : 0.0f);
}

}  // namespace bi
