// pa_shared.hpp -- attention of groups of sequences that share a prefix, on the
// matrix cores of gfx950.
//
// Sequence b of group g attends the first P_g tokens through the pages of its
// group's first sequence and its own tokens, from P_g on, through its own.  Row
// r (position n_r) of the result is softmax(scale q_r . k_j) v_j over j <= n_r, so
// it splits by keys into any number of states (m, l, acc) that the merge joins:
//   m = max s_j, l = sum 2^(s_j - m), acc = sum 2^(s_j - m) v_j   (s in log2 units).
//
// Work.  A unit is a block of query rows against one run of keys under one KV
// head: the rows of a whole group against its prefix, the rows of a sequence
// against its own keys.  The units' key tiles lie end to end on a line, measured in
// cost, and every worker takes an equal stretch of it, cutting units where the
// stretch ends: nobody waits for a longer one whatever the lengths, and
// compute-bound prefixes run beside memory-bound tails.  A worker's piece of a unit
// leaves one state per row.  Its place in the workspace needs no table: worker w's
// stretch and unit u's first row only grow along the line, so w * 128 + row (16 for
// thin units) is unique.
//
// Two bodies, on v_mfma_f32_{32x32x16,16x16x32}:
//  * wide, up to 128 rows (every prefix, and own keys under more than 16 rows): a
//    work-group is the worker.  A wave owns 32 rows; a tile's K and V go through
//    LDS once for all four, the next tile's loads in flight.  One read of the
//    prefix serves 128 rows.
//  * thin, up to 16 rows: memory-bound.  A wave is the worker, each with its own
//    units and no barrier, since tails are short and a unit's chain of loads long.
//    K goes straight into the operand registers, V through the wave's own LDS.
// Both compute S^T = K Q^T, whose accumulator layout is the operand layout of
// O^T += V^T P^T: the probabilities stay in registers.
//
// What bounds it.  A CU takes a wide tile of 128 rows and 64 keys of 128 per 1.3 us
// (0.83 PFLOP/s over the card, where a large library product reaches 1.2):
// neither the matrix cores (27 % busy), the vector ALU (32 %) nor LDS (22 %) is full,
// but a wave's chain (scores, maximum, weights, products) and the two waves of a SIMD
// fill each other's gaps only in part; one work-group a CU takes 1.9 us a tile.  Eight
// waves sharing a tile (256 rows, one work-group a CU) ran at the same rate a row with
// a state of twice the size to write, and alternating their phases did not fit the
// registers.  Thin tiles run at the memory's rate (64 x 4096 tokens of 32/8 heads of
// 128 in bf16: 183 us, 5.9 TB/s).  A call is 2.4 us until its line is known, 2 to 6
// until a first tile (FP8 codes and long tables the most), and the merge, 4 us or the
// time of the states' bytes (8192 rows over 512 pieces of 128: 42 MB, 12 us).
//
// Variants, with both sides measured.  Thin units up to 16 rows: 64 x 4096 tokens,
// 32/8 heads of 128, 4 rows 183 us (wide 200), 16 rows 198 (210); at 32 rows a thin
// unit of two row blocks gained 2 to 8 % at D <= 128 and lost 45 % at 256.  Pages of a
// multiple of 16 tokens: one page id a wave (128 rows over 8192 tokens 48.0 us; a page
// id a row, taken for other sizes, 49.1).
//
// Types.  FP8 codes widen exactly to the 16-bit type of q.  q of another type than
// the tiles' is carried as hi + lo (2^-17 of bf16 pieces, 2^-22 of fp16); the
// probabilities as two fp16 or three bf16 pieces where the output is fp32 (2^-22,
// 2^-25: two bf16 pieces left an error of 2.1e-6 where fp32 sums have 4e-7), else
// rounded to the tiles' type, as the output is.  Sums, maxima and states are fp32.
//
// Masked keys.  A key behind a row's position never meets its weight: the scores
// are selected to -inf, V rows past the unit are zeroed, and a non-finite V element
// in a tile that some row does not see whole is taken out of the product and added
// to the rows that see it afterwards.
#pragma once

#include "pa_prefill.hpp"
#include "pa_decode_mfma.hpp"

namespace pa {

constexpr int kShThreads = 256;
constexpr int kShWaves = 4;

// 16 bytes per lane straight to LDS byte address `to` (wave-uniform) + 16 lane, from a
// uniform base and a 32-bit lane offset, or from a lane's address.  The compiler does not
// see the loads: the caller waits for vmcnt before the barrier that publishes the data.
// (A spilled lane address cost a wait for every earlier load; the scalar base leaves
// one register a load.)
__device__ inline void dma_at(const char* base, uint32_t off, uint32_t to) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "{m0}"(to));
}
__device__ inline void dma_at(const char* from, uint32_t to) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(from), "{m0}"(to));
}

// Tile type of a cache: FP8 codes widen to fp16 or bf16.
template <typename KV, bool kBf>
struct ShTile {
  static constexpr bool kF8 = KV::kCode == kFP8;
  static constexpr int kPair = kBf ? kBF16 : kF16;
  using Raw = typename KV::Raw;
  __device__ static inline u32x4_t widen(const Raw& r) {
    if constexpr (kF8) {
      uint32_t w[4];
      KvFP8::to_pairs<kPair>(r, w);
      return u32x4_t{w[0], w[1], w[2], w[3]};
    } else {
      return r;
    }
  }
};

// Whether any 16-bit element of the chunk is not finite; those that are not, zeroed.
template <bool kBf>
__device__ inline bool sanitize(u32x4_t& x) {
  constexpr uint32_t e = kBf ? 0x7f80u : 0x7c00u;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w = x[i];
    if ((w & e) == e) {
      w &= 0xffff0000u;
      any = true;
    }
    if (((w >> 16) & e) == e) {
      w &= 0xffffu;
      any = true;
    }
    x[i] = w;
  }
  return any;
}

// V element d of the row at byte offset `off`, as fp32.
template <typename KV>
__device__ inline float v_elem(const char* vbase, uint64_t off, int d) {
  if constexpr (KV::kCode == kFP8) {
    const uint32_t c = reinterpret_cast<const uint8_t*>(vbase + off)[d];
    return __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false)[0];
  } else {
    return load_elem(vbase + off, KV::kCode, d);
  }
}

// ------------------------------------------------------------------- plan --

struct ShPlan {
  int total;  // end of the line
  int own;    // where the sequences' own keys begin
  int share;  // a work-group's stretch, a multiple of 4
};

// A sequence's group, or -1.  starts: [NG + 1], non-decreasing.
template <typename T>
__device__ inline int group_of(const T* starts, int NG, int b) {
  if (b < starts[0] || b >= starts[NG]) return -1;
  int lo = 0, hi = NG;  // last g with starts[g] <= b
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= b) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ inline int row_blocks(int rows) { return (rows + kSharedWide - 1) / kSharedWide; }
__device__ inline int wide_tiles(int n) { return (n + kSharedWideTile - 1) / kSharedWideTile; }
__device__ inline int own_tiles(const SharedParams& p, int n) {
  return p.thin ? (n + kSharedThinTile - 1) / kSharedThinTile : wide_tiles(n);
}
__device__ inline int wide_cost(int tiles) { return kSharedWideStart + tiles * kSharedWideCost; }
__device__ inline int own_cost(const SharedParams& p, int tiles) {
  return p.thin ? kSharedThinStart + tiles * kSharedThinCost : wide_cost(tiles);
}
// First key of the tiles of a sequence's own keys: sixteen rows of a tile then lie
// in one page where pages hold a multiple of 16.
__device__ inline int own_first(int prefix) { return prefix & ~15; }
// Prefix of a group as attended: none where it is negative.
__device__ inline int prefix_of(int n) { return n > 0 ? n : 0; }

// What a work-group knows of the batch: where the units lie on the line, and each
// sequence's prefix and context.
struct ShTables {
  int32_t cum[kSharedMaxGroups + kSharedMaxSeqs + 1];  // cost before entry i: groups, then sequences
  int32_t pre[kSharedMaxSeqs];                         // prefix of the sequence's group, 0: none
  int32_t ctx[kSharedMaxSeqs];
  uint16_t start[kSharedMaxGroups + 2];                // first sequence of each group, and the end
};

// Fills the tables.  s_tmp: scratch of NG + 8 words.  Every thread of the work-group;
// fault: the group starts are unusable.
__device__ inline ShPlan plan_scan(const SharedParams& p, ShTables& s, int32_t* s_tmp, int& fault) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* s_len = s_tmp + 8;
  const int maxctx = p.MB * p.BS;
  // (The first round's loads are all in flight before any is used.)
  int bad = 0;
  const bool own0 = tid < p.B, end0 = tid <= p.NG, len0 = tid < p.NG;
  const int c0 = own0 ? p.context_lens[tid] : 0, a0 = end0 ? p.group_starts[tid] : 0;
  const int b0 = len0 ? p.group_starts[tid + 1] : 0, l0 = len0 ? p.prefix_lens[tid] : 0;
  auto group = [&](int g, int a, int next, int len) {
    bad |= a < 0 || a > p.B || (g < p.NG && next < a);
    s.start[g] = (uint16_t)a;
    if (g < p.NG) s_len[g] = prefix_of(len);
  };
  if (own0) s.ctx[tid] = c0;
  if (end0) group(tid, a0, b0, l0);
  for (int b = tid + kShThreads; b < p.B; b += kShThreads) s.ctx[b] = p.context_lens[b];
  for (int g = tid + kShThreads; g <= p.NG; g += kShThreads)
    group(g, p.group_starts[g], g < p.NG ? p.group_starts[g + 1] : 0, g < p.NG ? p.prefix_lens[g] : 0);
  fault = __syncthreads_or(bad);
  if (fault) return {0, 0, 4};
  // Costs of the groups, then of the sequences, and their prefix sums.
  int carry = 0;
  const int n = p.NG + p.B;
  for (int i0 = 0; i0 < n; i0 += kShThreads) {
    const int i = i0 + tid, b = i - p.NG;
    int c = 0;
    if (i < p.NG) {
      if (s_len[i] > 0 && s_len[i] <= maxctx)
        c = p.HKV * row_blocks((s.start[i + 1] - s.start[i]) * p.SG) * wide_cost(wide_tiles(s_len[i]));
    } else if (i < n) {
      const int g = group_of(s.start, p.NG, b);
      const int P = g < 0 ? 0 : s_len[g], ctx = s.ctx[b];
      s.pre[b] = P;
      if (ctx > P && ctx <= maxctx) c = p.HKV * p.own_rb * own_cost(p, own_tiles(p, ctx - own_first(P)));
    }
    int x = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    if (i0 > 0) __syncthreads();  // s_tmp has been read
    if (lane == 63) s_tmp[wave] = x;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) {
      before += w < wave ? s_tmp[w] : 0;
      carry += s_tmp[w];
    }
    if (i < n) s.cum[i] = before + x - c;
  }
  if (tid == 0) s.cum[n] = carry;
  __syncthreads();
  const int own = s.cum[p.NG];
  const int even = (carry + p.wgs - 1) / p.wgs;
  return {carry, own, max(kSharedMinShare, (even + 3) & ~3)};
}

// The last entry that begins at or before `pos` of the line, by 64-way search.
__device__ inline int entry_at(const ShTables& s, int n, int pos) {
  const int lane = threadIdx.x & 63, step = (n + 63) / 64;
  const int i = lane * step;
  const int block = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < n && s.cum[min(i, n)] <= pos)) - 1;
  const int j = block * step + lane;
  return block * step +
         __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < step && j < n && s.cum[min(j, n)] <= pos)) - 1;
}

// Which states a unit left: workers first .. last, for tiles of `cost` behind `start`
// of a unit that begins at `begin`.
__device__ inline void unit_workers(int begin, int start, int cost, int tiles, int share, int& first, int& count) {
  first = (begin + start) / share;
  count = (begin + start + (tiles - 1) * cost) / share - first + 1;
}

// Rows of the workspace: the prefixes' states, then the own keys'.
__host__ __device__ inline int64_t prefix_slots(const SharedParams& p) {
  return (int64_t)p.wgs * kSharedWide + (int64_t)p.HKV * p.B * p.SG;
}
__host__ __device__ inline int64_t own_slots(const SharedParams& p) {
  return (int64_t)p.wgs * (p.thin ? kShWaves * kSharedThin : kSharedWide) + (int64_t)p.HKV * p.B * p.SG;
}
__device__ inline int64_t prefix_slot(const SharedParams& p, int worker, int b0, int rows, int kvh, int row) {
  return (int64_t)worker * kSharedWide + (int64_t)p.HKV * b0 * p.SG + (int64_t)kvh * rows + row;
}
__device__ inline int64_t own_slot(const SharedParams& p, int worker, int b, int kvh, int row) {
  return prefix_slots(p) + (int64_t)worker * (p.thin ? kSharedThin : kSharedWide) +
         ((int64_t)b * p.HKV + kvh) * p.SG + row;
}

// One piece: rows [row0, row0 + rows) of the unit's numbering against the keys of
// tiles [k0, k1).
struct ShPiece {
  int kvh;
  int b0;       // sequence of row 0 of the unit's numbering
  int row0;     // first row of the block
  int rows;     // rows of the block
  int first;    // first key of tile 0
  int lo;       // keys below it are not attended
  int end;      // end of the unit's keys
  int k0, k1;   // tiles
  const int32_t* table;
  int64_t slot;  // workspace row of the block's row 0
};

// Row `r` of a piece: its q row (index of [B, S, H]) and the end of the keys it
// attends; a row past the block attends whatever is there (it is not written).
__device__ inline void row_of(const SharedParams& p, const ShPiece& u, const ShTables& tab, int r, bool& live,
                              int64_t& qrow, int& lim) {
  live = r < u.rows;
  const uint32_t R = (uint32_t)(u.row0 + (live ? r : 0));
  const uint32_t i = fastdiv(R, p.sg_div);
  const uint32_t t = R - i * (uint32_t)p.SG;
  const uint32_t s = fastdiv(t, p.g_div);
  const int b = u.b0 + (int)i;
  qrow = ((int64_t)b * p.S + s) * p.H + (int64_t)u.kvh * p.G + (t - s * (uint32_t)p.G);
  const int ctx = max(tab.ctx[b], 0);
  const int n = ctx <= p.MB * p.BS ? min(ctx - p.S + (int)s + 1, u.end) : 0;
  lim = live ? n : 0x7fffffff;
}

// q row at dims d0 + kStep ks .. of 8 as hi (+ lo) words of the tiles' type, with the
// scale's sign.  fp16 hi + lo rows are scaled by the power of two that puts the row's
// largest element in [2^14, 2^15), and their scores by the inverse, returned in
// `back` (lanes kFrom, 2 kFrom, .. apart hold the row's other dims).
template <bool kBf, bool kSplit, int NS, int kStep, int kFrom>
__device__ inline void load_q(const SharedParams& p, bool live, int64_t qrow, int d0, u32x4_t (&hi)[NS],
                              u32x4_t (&lo)[kSplit ? NS : 1], float& back) {
  back = 1.0f;
  if constexpr (!kSplit) {
    const uint32_t a = live ? p.q_and : 0u, x = live ? p.q_xor : 0u;
#pragma unroll
    for (int ks = 0; ks < NS; ++ks) hi[ks] = load16(p.q, (qrow * p.D + d0 + kStep * ks) * 2);
#pragma unroll
    for (int ks = 0; ks < NS; ++ks) {
#pragma unroll
      for (int j = 0; j < 4; ++j) hi[ks][j] = (hi[ks][j] & a) ^ x;
    }
    return;
  }
  float x[NS][8];
  const float sign = live ? p.q_sign : 0.0f;
#pragma unroll
  for (int ks = 0; ks < NS; ++ks) {
    load8f(p.q, p.q_dtype, qrow * p.D + d0 + kStep * ks, x[ks]);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[ks][e] = sign == 0.0f ? 0.0f : x[ks][e] * sign;
  }
  if constexpr (kSplit && !kBf) {
    float mx = 0.0f;
#pragma unroll
    for (int ks = 0; ks < NS; ++ks) {
#pragma unroll
      for (int e = 0; e < 8; ++e) mx = fmaxf(mx, __builtin_fabsf(x[ks][e]));
    }
#pragma unroll
    for (int o = kFrom; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    const int ex = (int)(__builtin_bit_cast(uint32_t, mx) >> 23) - 127;
    const int k = ex > 127 ? 0 : max(-113, min(100, 14 - ex));
    const float up = __builtin_bit_cast(float, (uint32_t)(127 + k) << 23);
    back = __builtin_bit_cast(float, (uint32_t)(127 - k) << 23);
#pragma unroll
    for (int ks = 0; ks < NS; ++ks) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[ks][e] *= up;
    }
  }
#pragma unroll
  for (int ks = 0; ks < NS; ++ks) {
    uint32_t w[4], wl[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = pack2<kBf>(x[ks][2 * j], x[ks][2 * j + 1]);
      if constexpr (kSplit) {
        const float2_t r = unpack2<kBf>(w[j]);
        wl[j] = pack2<kBf>(x[ks][2 * j] - r[0], x[ks][2 * j + 1] - r[1]);
      }
    }
    hi[ks] = u32x4_t{w[0], w[1], w[2], w[3]};
    if constexpr (kSplit) lo[ks] = u32x4_t{wl[0], wl[1], wl[2], wl[3]};
  }
}

// Byte offsets of one key row's K and V under the piece's head.  A row past the
// unit, or on a page outside the cache, is read at row 0 of block 0 (in bounds, NB >=
// 1) and not used.
struct ShRow {
  uint64_t k, v;
  bool use, bad;
};
__device__ inline ShRow key_row(const SharedParams& p, int32_t blk, int off, bool inside, int es) {
  ShRow r;
  const bool ok = (uint64_t)(int64_t)blk < (uint64_t)p.num_blocks;
  r.bad = inside && !ok;
  r.use = inside && ok;
  const uint32_t ub = r.use ? (uint32_t)blk : 0u, uo = r.use ? (uint32_t)off : 0u;
  r.k = (uint64_t)ub * (uint32_t)(p.k_sb * es) + uo * (uint32_t)(p.k_st * es);
  r.v = (uint64_t)ub * (uint32_t)(p.v_sb * es) + uo * (uint32_t)(p.v_st * es);
  return r;
}
__device__ inline uint64_t shfl64(uint64_t x, int lane) {
  const uint32_t a = __shfl((int)(uint32_t)x, lane, 64), b = __shfl((int)(uint32_t)(x >> 32), lane, 64);
  return ((uint64_t)b << 32) | a;
}

// ------------------------------------------------------------------- tiles --

template <int D>
struct ShShape {
  static constexpr int KB = D <= 128 ? 64 : 32;  // keys per LDS tile of the wide body
  static constexpr int MT = KB / 32;
  static constexpr int KS = D / 16;
  static constexpr int DT = D / 32;
  static constexpr int NCH = D / 8;
  static constexpr int TPD = 64 / NCH;       // rows per 1 KB load
  static constexpr int RPW = KB / kShWaves;  // rows a wave loads
  static constexpr int NP = RPW / TPD;       // loads per wave and tile
  static constexpr int TILE = KB * D;        // 16-bit elements
  static constexpr int NDMA = kSharedThinTile / TPD;  // V loads of a thin tile
  static constexpr int LDS_WIDE = 4 * TILE * 2;       // K and V, two tiles
  static constexpr int LDS_THIN = kShWaves * kSharedThinTile * D * 2;
  static constexpr int LDS_PLAN = (8 + kSharedMaxGroups) * 4;
  static constexpr int LDS_BODY = LDS_WIDE > LDS_THIN ? LDS_WIDE : LDS_THIN;
  static constexpr int LDS = LDS_BODY > LDS_PLAN ? LDS_BODY : LDS_PLAN;
  static_assert(NP >= 1 && RPW % TPD == 0, "tile shape");
};

struct ShFlags {
  unsigned long long bad[3];  // per tile, three in turn: keys on pages outside the cache
  int odd;                    // something was taken out of V (restore_odd)
  int lim[kSharedWide];       // end of the keys that each row attends
  int shortest[kShWaves];
};

// Adds to the piece's states what sanitize() took out of V: the elements that are not
// finite, in tiles of KT keys that some row does not see whole (the shortest row ends
// at `least`), for the rows that see their keys.  `tid` of `threads` threads.
template <typename KV>
__device__ __forceinline__ void restore_odd(const SharedParams& p, const ShPiece& u, const int* lim, int least, int KT,
                                            int step, int tid, int threads) {
  const char* vbase = static_cast<const char*>(p.v) + (int64_t)u.kvh * p.v_sh * KV::kBytes;
  const int n0 = u.first + u.k0 * step, n1 = min(u.first + u.k1 * step, u.end);
  for (int key = max(n0, u.lo); key < n1; ++key) {
    const int t0 = n0 + (key - n0) / KT * KT;
    if (t0 >= u.lo && t0 + KT <= least) continue;
    const int pg = (int)fastdiv((uint32_t)key, p.bs_div);
    const ShRow row = key_row(p, u.table[pg], key - pg * p.BS, true, KV::kBytes);
    if (row.bad) continue;
    for (int d = tid; d < p.D; d += threads) {
      const float x = v_elem<KV>(vbase, row.v, d);
      if (__builtin_isfinite(x)) continue;
      for (int r = 0; r < u.rows; ++r)
        if (key < lim[r]) p.ws_acc[(u.slot + r) * p.D + d] += x;
    }
  }
}

// Two weights as pieces of the tiles' type, each what the ones before left.
template <bool kBf, int N>
__device__ inline void pieces(float a, float b, uint32_t (&w)[N][4], int j) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    w[n][j] = pack2<kBf>(a, b);
    const float2_t r = unpack2<kBf>(w[n][j]);
    a -= r[0];
    b -= r[1];
  }
}

// The softmax step over N raw scores of a lane's row (kOther: the lanes that hold its
// other keys): raises the running maximum m (log2 units) where it is passed by more
// than 2^8 and says by what the sums shrink.
template <int kOther>
__device__ inline float raise_max(float mx, float qscale, float& m) {
#pragma unroll
  for (int o = kOther; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  mx *= qscale;
  if (__builtin_amdgcn_ballot_w64(mx > m + kLazyRescale) == 0) return 1.0f;
  asm volatile("");
  const float mn = fmaxf(m, mx);
  const float corr = mn == -__builtin_inff() ? 1.0f : fast_exp2(m - mn);
  m = mn;
  return corr;
}

// ------------------------------------------------------------------- wide --

template <typename KV, bool kBf, int D, bool kSplitQ, bool kSplitP>
__device__ __forceinline__ void wide_piece(const SharedParams& p, const ShPiece& u, const ShTables& s,
                                           char* lds, ShFlags* fl) {
  using Sh = ShShape<D>;
  using Tl = ShTile<KV, kBf>;
  constexpr int KB = Sh::KB, MT = Sh::MT, KS = Sh::KS, DT = Sh::DT, NCH = Sh::NCH, TPD = Sh::TPD, RPW = Sh::RPW,
                NP = Sh::NP;
  constexpr int EB = KV::kBytes, kPieces = !kSplitP ? 1 : kBf ? 3 : 2;
  uint16_t* sK = reinterpret_cast<uint16_t*>(lds);
  uint16_t* sV = sK + 2 * Sh::TILE;
  int lane = threadIdx.x & 63;
  // What follows from the lane is made anew each piece where registers are short, instead
  // of kept in scratch meanwhile (64/8 heads of 128 in FP8 111.3 -> 109.6 us; 12 heads of
  // 64, which have registers to spare, 17.8 -> 18.8).
  if constexpr (D >= 128) asm volatile("" : "+v"(lane));
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hh = lane >> 5;

  const char* kbase = static_cast<const char*>(p.k) + (int64_t)u.kvh * p.k_sh * EB;
  const char* vbase = static_cast<const char*>(p.v) + (int64_t)u.kvh * p.v_sh * EB;
  const int n0 = u.first + u.k0 * kSharedWideTile;  // first key of the piece
  const int n1 = min(u.first + u.k1 * kSharedWideTile, u.end);
  const int ntiles = (n1 - n0 + KB - 1) / KB;

  // This wave loads rows [RPW wave, RPW wave + RPW) of a tile.  Where they lie in one
  // page its block id is a scalar and a lane's part of the addresses a constant;
  // else lane r holds the page of row r % RPW.
  const int myrow = wave * RPW + (p.page16 ? 0 : lane % RPW);
  auto page_at = [&](int tile) {
    const int pg = (int)fastdiv((uint32_t)min(n0 + tile * KB + myrow, n1 - 1), p.bs_div);
    return u.table[pg];
  };
  int32_t blk = page_at(0);
  uint32_t klane[NP], vlane[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = i * TPD + lane / NCH, row = wave * RPW + r;
    klane[i] = (uint32_t)r * (uint32_t)(p.k_st * EB) + kpos<D>(row, lane % NCH) * 8 * EB;
    vlane[i] = (uint32_t)r * (uint32_t)(p.v_st * EB) + vpos<D>(row, lane % NCH) * 8 * EB;
  }

  bool live;
  int64_t qrow;
  int lim;
  row_of(p, u, s, wave * 32 + (lane & 31), live, qrow, lim);
  const bool busy = wave * 32 < u.rows;
  u32x4_t qf[KS], ql[kSplitQ ? KS : 1];
  float back;
  load_q<kBf, kSplitQ, KS, 16, 32>(p, live, qrow, hh * 8, qf, ql, back);
  const float qscale = kSplitQ && !kBf ? fmaxf(p.qscale * back, 0x1p-126f) : p.qscale;

  // The shortest row of this wave and of the block.
  int wmin = lim;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) wmin = min(wmin, __shfl_xor(wmin, o, 64));
  wmin = __builtin_amdgcn_readfirstlane(wmin);
  if (lane == 0) fl->shortest[wave] = wmin;
  if (hh == 0) fl->lim[wave * 32 + lane] = lim;
  if (threadIdx.x < 3) fl->bad[threadIdx.x] = 0;
  if (threadIdx.x == 0) fl->odd = 0;
  __syncthreads();
  const int bmin = __builtin_amdgcn_readfirstlane(
      min(min(fl->shortest[0], fl->shortest[1]), min(fl->shortest[2], fl->shortest[3])));

  uint32_t dead = 0;  // bit i: this lane's row of load i is not used
  typename Tl::Raw kr[Tl::kF8 ? NP : 1], vr[Tl::kF8 ? NP : 1];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)lds + wave * (RPW * D * 2);
  auto issue = [&](int tile, int slot3) {
    const uint32_t toK = lds0 + (tile & 1) * (Sh::TILE * 2), toV = toK + 2 * Sh::TILE * 2;
    const int key = n0 + tile * KB + wave * RPW;  // first of this wave's rows
    dead = 0;
    if (p.page16) {
      const int32_t id = __builtin_amdgcn_readfirstlane(blk);
      const bool ok = (uint64_t)(int64_t)id < (uint64_t)p.num_blocks;
      const bool use = ok && key < n1;
      if (!ok && key < n1 && lane == 0)
        atomicOr(&fl->bad[slot3], ((1ull << min(RPW, n1 - key)) - 1) << (wave * RPW));
      const uint32_t ub = use ? (uint32_t)id : 0u;
      const uint32_t uo = use ? (uint32_t)key - fastdiv((uint32_t)key, p.bs_div) * (uint32_t)p.BS : 0u;
      const char* ka = kbase + ((uint64_t)ub * (uint32_t)(p.k_sb * EB) + uo * (uint32_t)(p.k_st * EB));
      const char* va = vbase + ((uint64_t)ub * (uint32_t)(p.v_sb * EB) + uo * (uint32_t)(p.v_st * EB));
      // (A page holds RPW rows and more, so those past the unit's end exist too.)
      if (!use || key + RPW > n1) {
#pragma unroll
        for (int i = 0; i < NP; ++i) dead |= (uint32_t)(!use || key + i * TPD + lane / NCH >= n1) << i;
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if constexpr (Tl::kF8) {
          kr[i] = *reinterpret_cast<const typename Tl::Raw*>(ka + klane[i]);
          vr[i] = *reinterpret_cast<const typename Tl::Raw*>(va + vlane[i]);
        } else {
          dma_at(ka, klane[i], toK + i * 1024);
          dma_at(va, vlane[i], toV + i * 1024);
        }
      }
    } else {
      const int mine = n0 + tile * KB + myrow;
      const int kk = min(mine, n1 - 1);
      const ShRow row = key_row(p, blk, kk - (int)fastdiv((uint32_t)kk, p.bs_div) * p.BS, mine < n1, EB);
      if (row.bad && lane < RPW) atomicOr(&fl->bad[slot3], 1ull << myrow);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int r = i * TPD + lane / NCH;
        dead |= (uint32_t)(__shfl((int)row.use, r, 64) == 0) << i;
        const char* ka = kbase + shfl64(row.k, r) + kpos<D>(wave * RPW + r, lane % NCH) * 8 * EB;
        const char* va = vbase + shfl64(row.v, r) + vpos<D>(wave * RPW + r, lane % NCH) * 8 * EB;
        if constexpr (Tl::kF8) {
          kr[i] = *reinterpret_cast<const typename Tl::Raw*>(ka);
          vr[i] = *reinterpret_cast<const typename Tl::Raw*>(va);
        } else {
          dma_at(ka, toK + i * 1024);
          dma_at(va, toV + i * 1024);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  // The tile's loads have landed: widen FP8 codes, zero the V rows that are not
  // used, take out what is not finite where some row does not see the whole tile.
  auto finish = [&](int tile, uint16_t* dK, uint16_t* dV) {
    const int t0 = n0 + tile * KB;
    const bool masked = t0 < u.lo || t0 + KB > bmin;
    dK += wave * RPW * D + lane * 8;
    dV += wave * RPW * D + lane * 8;
    if constexpr (Tl::kF8) {
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        *reinterpret_cast<u32x4_t*>(dK + i * 512) = Tl::widen(kr[i]);
        *reinterpret_cast<u32x4_t*>(dV + i * 512) = Tl::widen(vr[i]);
      }
    }
    if (masked || __builtin_amdgcn_ballot_w64(dead != 0) != 0) {
#pragma unroll 1
      for (int i = 0; i < NP; ++i) {
        u32x4_t x = *reinterpret_cast<const u32x4_t*>(dV + i * 512);
        if ((dead >> i) & 1u) {
          x = u32x4_t{0u, 0u, 0u, 0u};
        } else if (masked && sanitize<kBf>(x)) {
          fl->odd = 1;
        }
        *reinterpret_cast<u32x4_t*>(dV + i * 512) = x;
      }
    }
  };

  f32x16_t o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
    for (int i = 0; i < 16; ++i) o[dt][i] = 0.0f;
  }
  float m = -__builtin_inff(), l = 0.0f;

  // LDS places of the operands: the swizzles flip bits of the chunk number, so K's
  // k-step ks is ks * 16 elements away by exclusive or, V's dim tile dt dt * 32; m-tiles
  // of K lie 32 rows apart, 16-key steps of V 16 rows, an operand's second half 8.
  const int kat = swk<D>(lane & 31, hh);
  const int vat = swv<D>(4 * hh + ((lane & 15) >> 2), ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) + (lane & 1) * 4;
  static_assert(((8 >> PfShape<D>::VSH) & PfShape<D>::VSW) == 0 && ((16 >> PfShape<D>::VSH) & PfShape<D>::VSW) == 0 &&
                    ((32 >> PfShape<D>::KSH) & PfShape<D>::KSW) == 0,
                "the swizzles repeat every 8 rows of V and 32 of K");

  auto compute = [&](int tile, int slot3, const uint16_t* cK, const uint16_t* cV) {
    const int t0 = n0 + tile * KB;
    // K operands are read four k-steps ahead of their products and V operands two key
    // steps ahead (the first before the softmax), so that LDS answers while the matrix
    // cores and the vector ALU work.  (All of them ahead spilled at D = 128.)
    constexpr int WK = KS < 4 ? KS : 4, TS = KB / 16;
    f32x16_t st[MT];
    u32x4_t a[WK][MT];
    auto load_a = [&](int ks) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        a[ks % WK][mt] = *reinterpret_cast<const u32x4_t*>(cK + (kat ^ (ks * 16)) + mt * 32 * D);
    };
    short4_t vf[2][DT][2];
    auto load_vf = [&](int ts) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          vf[ts & 1][dt][e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_short4_t*)(cV + (vat ^ (dt * 32)) + (ts * 16 + e * 8) * D));
      }
    };
#pragma unroll
    for (int ks = 0; ks < WK; ++ks) load_a(ks);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[mt][i] = 0.0f;
    }
    __builtin_amdgcn_sched_barrier(0);
    // (A wave at its scores goes before the CU's other work-group at its softmax.)
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        st[mt] = mfma32<kBf>(a[ks % WK][mt], qf[ks], st[mt]);
        if constexpr (kSplitQ) st[mt] = mfma32<kBf>(a[ks % WK][mt], ql[ks], st[mt]);
      }
      if (ks + WK < KS) load_a(ks + WK);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    load_vf(0);
    if constexpr (TS > 1) load_vf(1);
    __builtin_amdgcn_sched_barrier(0);
    // This lane's key of slot i is t0 + 4 hh + mt 32 + 8 (i / 4) + i % 4.
    const unsigned long long bad = fl->bad[slot3];
    if (__builtin_amdgcn_ballot_w64(bad != 0) != 0) {
      asm volatile("");
      const unsigned long long b = bad >> (4 * hh);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if ((b >> (mt * 32 + 8 * (i >> 2) + (i & 3))) & 1ull) st[mt][i] = __builtin_nanf("");
      }
    }
    if (t0 < u.lo || t0 + KB > wmin) {
      asm volatile("");
      const int from = u.lo - t0 - 4 * hh, to = lim - t0 - 4 * hh;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int r = mt * 32 + 8 * (i >> 2) + (i & 3);
          st[mt][i] = r < from || r >= to ? -__builtin_inff() : st[mt][i];
        }
      }
    }
    float mx = st[0][0];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[mt][i]);
    }
    const float corr = raise_max<32>(mx, qscale, m);
    if (__builtin_amdgcn_ballot_w64(corr != 1.0f) != 0) {
      asm volatile("");
      l *= corr;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= corr;
      }
    }
    const float negm = m == -__builtin_inff() ? 0.0f : -m;
#pragma unroll
    for (int ts = 0; ts < TS; ++ts) {
      uint32_t w[kPieces][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 8 * (ts & 1) + 2 * j;
        const float p0 = fast_exp2(fmaf(st[ts >> 1][i], qscale, negm));
        const float p1 = fast_exp2(fmaf(st[ts >> 1][i + 1], qscale, negm));
        l += p0 + p1;
        pieces<kBf>(p0, p1, w, j);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const uint64_t x0 = __builtin_bit_cast(uint64_t, vf[ts & 1][dt][0]),
                       x1 = __builtin_bit_cast(uint64_t, vf[ts & 1][dt][1]);
        const u32x4_t av = u32x4_t{(uint32_t)x0, (uint32_t)(x0 >> 32), (uint32_t)x1, (uint32_t)(x1 >> 32)};
#pragma unroll
        for (int n = 0; n < kPieces; ++n)
          o[dt] = mfma32<kBf>(av, u32x4_t{w[n][0], w[n][1], w[n][2], w[n][3]}, o[dt]);
      }
      if (ts + 2 < TS) load_vf(ts + 2);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  issue(0, 0);
  if (ntiles > 1) blk = page_at(1);
  int t3 = 0;  // tile % 3
#pragma unroll 1
  for (int i = 0; i < ntiles; ++i) {
    uint16_t* cK = sK + (i & 1) * Sh::TILE;
    uint16_t* cV = sV + (i & 1) * Sh::TILE;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of tile i
    finish(i, cK, cV);
    __syncthreads();
    asm volatile("" ::: "memory");
    const int next3 = t3 == 2 ? 0 : t3 + 1;
    if (threadIdx.x == 0) fl->bad[next3 == 2 ? 0 : next3 + 1] = 0;
    if (i + 1 < ntiles) {
      issue(i + 1, next3);
      if (i + 2 < ntiles) blk = page_at(i + 2);
    }
    if (busy) compute(i, t3, cK, cV);
    t3 = next3;
  }

  // The state of each row.
  l += __shfl_xor(l, 32, 64);
  if (live) {
    const int64_t at = u.slot + wave * 32 + (lane & 31);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4_t*>(p.ws_acc + at * D + dt * 32 + 8 * q + 4 * hh) =
            float4_t{o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]};
    }
    if (hh == 0) {
      p.ws_m[at] = m;
      p.ws_l[at] = l;
    }
  }
  __syncthreads();
  if (fl->odd) restore_odd<KV>(p, u, fl->lim, bmin, KB, kSharedWideTile, threadIdx.x, kShThreads);
  __syncthreads();  // (the next piece reuses the tiles and flags)
}

// ------------------------------------------------------------------- thin --

// One wave's piece; sV: the wave's own LDS tile.
template <typename KV, bool kBf, int D, bool kSplitQ, bool kSplitP>
__device__ __forceinline__ void thin_piece(const SharedParams& p, const ShPiece& u, const ShTables& s,
                                           uint16_t* sV, int* s_lim) {
  using Sh = ShShape<D>;
  using Tl = ShTile<KV, kBf>;
  constexpr int KT = kSharedThinTile, KS = D / 32, NDT = D / 16, NCH = Sh::NCH, TPD = Sh::TPD, NDMA = Sh::NDMA;
  constexpr int EB = KV::kBytes, kPieces = !kSplitP ? 1 : kBf ? 3 : 2;
  int lane = threadIdx.x & 63;
  if constexpr (D >= 128) asm volatile("" : "+v"(lane));  // (as wide_piece)
  const int col = lane & 15, kg = lane >> 4;
  const char* kbase = static_cast<const char*>(p.k) + (int64_t)u.kvh * p.k_sh * EB;
  const char* vbase = static_cast<const char*>(p.v) + (int64_t)u.kvh * p.v_sh * EB;
  const int n0 = u.first + u.k0 * KT;
  const int n1 = min(u.first + u.k1 * KT, u.end);
  const int ntiles = (n1 - n0 + KT - 1) / KT;

  // One tile in registers.  Its V is freed into LDS and its K into the scores at the
  // start of a round, and the next tile's loads take their place at once: eight
  // waves of a CU keep 128 KB in flight (D = 128) at half the registers of two tiles.
  typename Tl::Raw tk[2][KS], tv[NDMA];
  const int myrow = lane & 31;
  auto page_at = [&](int tile) {
    return u.table[(int)fastdiv((uint32_t)min(n0 + tile * KT + myrow, n1 - 1), p.bs_div)];
  };
  auto row_at = [&](int tile, int32_t blk) {
    const int key = n0 + tile * KT + myrow, kk = min(key, n1 - 1);
    return key_row(p, blk, kk - (int)fastdiv((uint32_t)kk, p.bs_div) * p.BS, key < n1, EB);
  };
  auto load_k = [&](const ShRow& r) {
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      const char* a = kbase + shfl64(r.k, mt * 16 + col) + kg * 8 * EB;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) tk[mt][ks] = *reinterpret_cast<const typename Tl::Raw*>(a + ks * 32 * EB);
    }
  };
  auto load_v = [&](const ShRow& r) {
#pragma unroll
    for (int i = 0; i < NDMA; ++i) {
      const int row = i * TPD + lane / NCH;
      // (Streamed: read once.  32/8 heads of 128, 4 x 32 sequences: 93 -> 88 us.)
      tv[i] = load_raw<KV>(vbase, (int64_t)(shfl64(r.v, row) + (lane % NCH) * 8 * EB));
    }
  };
  int32_t blk = page_at(0);
  bool live;
  int64_t qrow;
  int lim;
  row_of(p, u, s, col, live, qrow, lim);
  u32x4_t qf[KS], ql[kSplitQ ? KS : 1];
  float back;
  load_q<kBf, kSplitQ, KS, 32, 16>(p, live, qrow, kg * 8, qf, ql, back);
  ShRow row = row_at(0, blk);
  load_k(row);
  load_v(row);
  if (ntiles > 1) blk = page_at(1);
  const float qscale = kSplitQ && !kBf ? fmaxf(p.qscale * back, 0x1p-126f) : p.qscale;
  int wmin = lim;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) wmin = min(wmin, __shfl_xor(wmin, o, 64));
  wmin = __builtin_amdgcn_readfirstlane(wmin);

  float4_t o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = float4_t{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), l = 0.0f;
  bool odd = false;
#pragma unroll 1
  for (int i = 0; i < ntiles; ++i) {
    const int first = n0 + i * KT;
    const uint32_t bad = (uint32_t)__builtin_amdgcn_ballot_w64(row.bad);    // keys on pages outside the cache
    const uint32_t dead = (uint32_t)__builtin_amdgcn_ballot_w64(!row.use);  // keys not used
    const bool masked = first < u.lo || first + KT > wmin;
    const bool more = i + 1 < ntiles;
    if (more) row = row_at(i + 1, blk);
    if (i + 2 < ntiles) blk = page_at(i + 2);
    // V to LDS; rows not used are zeroed, what is not finite taken out where a row
    // does not see the whole tile.
#pragma unroll
    for (int j = 0; j < NDMA; ++j) {
      u32x4_t x = Tl::widen(tv[j]);
      const int r = j * TPD + lane / NCH;
      if (dead != 0 || masked) {
        if ((dead >> r) & 1u) {
          x = u32x4_t{0u, 0u, 0u, 0u};
        } else if (masked) {
          odd |= sanitize<kBf>(x);
        }
      }
      *reinterpret_cast<u32x4_t*>(sV + r * D + (dm_vpos<D>(r, lane % NCH) << 3)) = x;
    }
    if (more) load_v(row);
    __builtin_amdgcn_sched_barrier(0);
    float4_t st[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
      st[mt] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4_t a = Tl::widen(tk[mt][ks]);
        st[mt] = mfma16<kBf>(a, qf[ks], st[mt]);
        if constexpr (kSplitQ) st[mt] = mfma16<kBf>(a, ql[ks], st[mt]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (more) load_k(row);
    if (masked || bad != 0) {
      asm volatile("");
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = mt * 16 + kg * 4 + e;
          const bool seen = first + r >= u.lo && first + r < lim;
          st[mt][e] = !seen ? -__builtin_inff() : ((bad >> r) & 1u) ? __builtin_nanf("") : st[mt][e];
        }
      }
    }
    const float mx = fmaxf(fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3])),
                           fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
    const float corr = raise_max<16>(mx, qscale, m);
    if (__builtin_amdgcn_ballot_w64(corr != 1.0f) != 0) {
      asm volatile("");
      l *= corr;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[dt][e] *= corr;
      }
    }
    const float negm = m == -__builtin_inff() ? 0.0f : -m;
    uint32_t w[kPieces][4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float p0 = fast_exp2(fmaf(st[mt][2 * j], qscale, negm));
        const float p1 = fast_exp2(fmaf(st[mt][2 * j + 1], qscale, negm));
        l += p0 + p1;
        pieces<kBf>(p0, p1, w, mt * 2 + j);
      }
    }
    const int r0 = kg * 4 + (col >> 2);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const int c = dt * 16 + (col & 3) * 4;
      const short4m_t a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_short4m_t*)(sV + r0 * D + (dm_vpos<D>(r0, c >> 3) << 3) + (c & 7)));
      const short4m_t a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_short4m_t*)(sV + (r0 + 16) * D + (dm_vpos<D>(r0 + 16, c >> 3) << 3) + (c & 7)));
      const uint64_t x0 = __builtin_bit_cast(uint64_t, a0), x1 = __builtin_bit_cast(uint64_t, a1);
      const u32x4_t a = u32x4_t{(uint32_t)x0, (uint32_t)(x0 >> 32), (uint32_t)x1, (uint32_t)(x1 >> 32)};
#pragma unroll
      for (int n = 0; n < kPieces; ++n) o[dt] = mfma16<kBf>(a, u32x4_t{w[n][0], w[n][1], w[n][2], w[n][3]}, o[dt]);
    }
  }

  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (live) {
    const int64_t at = u.slot + col;
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) *reinterpret_cast<float4_t*>(p.ws_acc + at * D + dt * 16 + kg * 4) = o[dt];
    if (kg == 0) {
      p.ws_m[at] = m;
      p.ws_l[at] = l;
    }
  }
  if (__builtin_amdgcn_ballot_w64(odd) != 0) {
    if (lane < 16) s_lim[lane] = lim;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");  // the states and limits are written
    __builtin_amdgcn_wave_barrier();
    restore_odd<KV>(p, u, s_lim, wmin, KT, KT, lane, 64);
    __builtin_amdgcn_wave_barrier();
  }
}

// ----------------------------------------------------------------- kernel --

template <typename KV, bool kBf, int D, bool kSplitQ, bool kSplitP>
__global__ __launch_bounds__(kShThreads) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1)))
void shared_kernel(const SharedParams p) {
  __shared__ __attribute__((aligned(16))) char lds[ShShape<D>::LDS];
  __shared__ ShTables s_tab;
  __shared__ ShFlags s_fl;
  int fault;
  const ShPlan pl = plan_scan(p, s_tab, reinterpret_cast<int32_t*>(lds), fault);
  const int n = p.NG + p.B;
  if (blockIdx.x == gridDim.x - 1) {  // (the last stretch is the shortest)
    if (threadIdx.x == 0) {
      p.ws_meta[0] = pl.share;
      p.ws_meta[1] = fault;
    }
    for (int b = threadIdx.x; b < p.B && !fault; b += kShThreads) {
      const int g = group_of(s_tab.start, p.NG, b), b0 = g < 0 ? b : s_tab.start[g];
      int32_t* m = p.ws_meta + kSharedMeta * (b + 1);
      m[0] = s_tab.pre[b];
      m[1] = s_tab.ctx[b];
      m[2] = b0;
      m[3] = g < 0 ? 0 : (s_tab.start[g + 1] - b0) * p.SG;
      m[4] = g < 0 ? 0 : s_tab.cum[g];
      m[5] = s_tab.cum[p.NG + b];
    }
  }
  if (fault) return;

  // The piece at `pos` of a stretch that ends at `stop`; pos moves to the unit's end.
  auto piece = [&](int& pos, int stop, int worker, ShPiece& u) {
    const int entry = __builtin_amdgcn_readfirstlane(entry_at(s_tab, n, pos));
    const bool prefix = entry < p.NG, thin = !prefix && p.thin;
    int rows, blocks, tiles;
    if (prefix) {
      u.b0 = __builtin_amdgcn_readfirstlane(s_tab.start[entry]);
      rows = (__builtin_amdgcn_readfirstlane(s_tab.start[entry + 1]) - u.b0) * p.SG;
      u.end = __builtin_amdgcn_readfirstlane(s_tab.pre[u.b0]);
      u.first = u.lo = 0;
      tiles = wide_tiles(u.end);
      blocks = row_blocks(rows);
    } else {
      u.b0 = entry - p.NG;
      rows = p.SG;
      u.lo = __builtin_amdgcn_readfirstlane(s_tab.pre[u.b0]);
      u.first = own_first(u.lo);
      u.end = __builtin_amdgcn_readfirstlane(s_tab.ctx[u.b0]);
      tiles = own_tiles(p, u.end - u.first);
      blocks = p.own_rb;
    }
    const int start = thin ? kSharedThinStart : kSharedWideStart;
    const int whole = thin ? kSharedThinStart + tiles * kSharedThinCost : wide_cost(tiles);
    const int at = __builtin_amdgcn_readfirstlane(s_tab.cum[entry]);
    const int unit = (int)((uint32_t)(pos - at) / (uint32_t)whole);
    const int begin = at + unit * whole;
    // Tiles that start within the stretch.
    auto tile_from = [&](int x) {
      const uint32_t d = (uint32_t)max(x - begin - start, 0);
      return (int)min(thin ? (d + kSharedThinCost - 1) / kSharedThinCost : (d + kSharedWideCost - 1) / kSharedWideCost,
                      (uint32_t)tiles);
    };
    u.k0 = tile_from(pos);
    u.k1 = tile_from(stop);
    pos = begin + whole;
    u.kvh = blocks == 1 ? unit : (int)((uint32_t)unit / (uint32_t)blocks);
    u.row0 = (unit - u.kvh * blocks) * kSharedWide;
    u.rows = min(rows - u.row0, kSharedWide);
    u.table = p.block_tables + (int64_t)u.b0 * p.bt_stride;
    u.slot = prefix ? prefix_slot(p, worker, u.b0, rows, u.kvh, u.row0) : own_slot(p, worker, u.b0, u.kvh, u.row0);
    return u.k0 < u.k1;
  };

  ShPiece u;
  const int wide_end = p.thin ? pl.own : pl.total;
  int pos = blockIdx.x * pl.share, stop = min(pos + pl.share, wide_end);
  while (pos < stop)
    if (piece(pos, stop, blockIdx.x, u)) wide_piece<KV, kBf, D, kSplitQ, kSplitP>(p, u, s_tab, lds, &s_fl);
  if (!p.thin) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int worker = blockIdx.x * kShWaves + wave, share = pl.share / kShWaves;
  pos = max(worker * share, pl.own);
  stop = min((worker + 1) * share, pl.total);
  while (pos < stop)
    if (piece(pos, stop, worker, u))
      thin_piece<KV, kBf, D, kSplitQ, kSplitP>(p, u, s_tab, reinterpret_cast<uint16_t*>(lds) + wave * kSharedThinTile * D,
                                               s_fl.lim + 16 * wave);
}

template <typename KV, bool kBf, int D>
hipError_t launch_shared_d(const SharedParams& p, hipStream_t stream) {
  const bool sq = p.q_dtype != (kBf ? kBF16 : kF16), sp = p.out_dtype == kF32;
  void (*kernel)(const SharedParams);
  if constexpr (KV::kCode == kFP8 && kBf)  // (the tiles take q's type)
    kernel = sp ? shared_kernel<KV, kBf, D, false, true> : shared_kernel<KV, kBf, D, false, false>;
  else if (sq)
    kernel = sp ? shared_kernel<KV, kBf, D, true, true> : shared_kernel<KV, kBf, D, true, false>;
  else
    kernel = sp ? shared_kernel<KV, kBf, D, false, true> : shared_kernel<KV, kBf, D, false, false>;
  note_launch("pa::shared_kernel<%s, %s, %d, %s, %s>", KV::kName, kBf ? "true" : "false", D, sq ? "true" : "false",
              sp ? "true" : "false");
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.wgs), dim3(kShThreads), 0, stream, p);
  return hipGetLastError();
}

template <typename KV, bool kBf>
hipError_t launch_shared_kv(const SharedParams& p, hipStream_t stream) {
  switch (p.D) {
    case 32: return launch_shared_d<KV, kBf, 32>(p, stream);
    case 64: return launch_shared_d<KV, kBf, 64>(p, stream);
    case 128: return launch_shared_d<KV, kBf, 128>(p, stream);
    case 256: return launch_shared_d<KV, kBf, 256>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pa
