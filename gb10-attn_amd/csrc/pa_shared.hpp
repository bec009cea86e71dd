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
// against its own keys.  The units' tiles of 64 keys lie end to end on a line, in
// units of cost, and every work-group takes an equal stretch of it, cutting units
// where the stretch ends: no work-group waits for a longer one whatever the
// lengths, and compute-bound prefixes run beside memory-bound tails.  A stretch's
// piece of a unit is one state per row.  A piece's rows have a place of their own
// in the workspace without any table: work-group w's stretch and unit u's first row
// only grow along the line, so w * 128 + row is unique.
//
// Two bodies, on v_mfma_f32_{32x32x16,16x16x32}:
//  * wide, up to 128 rows: a wave owns 32 rows, the tile's K and V go through LDS
//    once for all four (two tiles in flight).  One read of the prefix serves 128
//    rows.
//  * thin, up to 16 rows: memory-bound.  The waves take 32-key tiles in turn, K
//    straight into the operand registers, V through the wave's own LDS; their
//    states are joined in LDS at the end of the piece.
// Both compute S^T = K Q^T, whose accumulator layout is the operand layout of
// O^T += V^T P^T: the probabilities stay in registers.
//
// Types.  FP8 codes widen exactly to the 16-bit type of q.  q of another type than
// the tiles' is carried as hi + lo; the probabilities as hi + lo where the output is
// fp32 (2^-17 of bf16 pieces, 2^-22 of fp16), else rounded to the tiles' type, as
// the output is.  Sums, maxima and states are fp32.
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
  int total, share;
};

// A sequence's group, or -1.  starts: [NG + 1], non-decreasing.
__device__ inline int group_of(const int32_t* starts, int NG, int b) {
  if (b < starts[0] || b >= starts[NG]) return -1;
  int lo = 0, hi = NG;  // last g with starts[g] <= b
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= b) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ inline int tiles_of(int n) { return (n + kSharedTile - 1) / kSharedTile; }
__device__ inline int row_blocks(int rows) { return (rows + kSharedWide - 1) / kSharedWide; }
__device__ inline int tile_cost(const SharedParams& p, int rows) {
  return rows <= kSharedThin ? p.cost_thin : p.cost_wide;
}
// First key of the tiles of a sequence's own keys: pages of 16 and more tokens
// then hold 16 rows of a tile each.
__device__ inline int own_first(int prefix) { return prefix & ~15; }
// Prefix of a group as attended: none where it is negative.
__device__ inline int prefix_of(int n) { return n > 0 ? n : 0; }

// Sums of the units' costs, prefixes first, in s_cum [NG + 1 + B] (s_cum[i]: before
// entry i), and whether the group starts are unusable.  s_tmp: scratch of 2 NG + 1
// + 8 words.  Every thread of the work-group.
__device__ inline ShPlan plan_scan(const SharedParams& p, int32_t* s_cum, int32_t* s_tmp, int& fault) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int32_t* s_start = s_tmp + 8;
  int32_t* s_len = s_start + p.NG + 1;
  const int maxctx = p.MB * p.BS;
  int bad = 0;
  for (int g = tid; g <= p.NG; g += kShThreads) {
    const int a = p.group_starts[g];
    bad |= a < 0 || a > p.B || (g > 0 && p.group_starts[g - 1] > a);
    s_start[g] = a;
    if (g < p.NG) s_len[g] = prefix_of(p.prefix_lens[g]);
  }
  fault = __syncthreads_or(bad);
  if (fault) return {0, 1};
  int carry = 0;
  const int n = p.NG + p.B;
  for (int i0 = 0; i0 < n; i0 += kShThreads) {
    const int i = i0 + tid;
    int c = 0;
    if (i < p.NG) {
      const int rows = (s_start[i + 1] - s_start[i]) * p.SG, len = s_len[i];
      if (len <= maxctx) c = p.HKV * row_blocks(rows) * tiles_of(len) * tile_cost(p, rows);
    } else if (i < n) {
      const int b = i - p.NG;
      const int g = group_of(s_start, p.NG, b);
      const int P = g < 0 ? 0 : s_len[g], ctx = p.context_lens[b];
      if (ctx > P && ctx <= maxctx) c = p.HKV * p.own_rb * tiles_of(ctx - own_first(P)) * tile_cost(p, p.SG);
    }
    int x = c;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(x, o, 64);
      if (lane >= o) x += y;
    }
    if (lane == 63) s_tmp[wave] = x;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) {
      before += w < wave ? s_tmp[w] : 0;
      carry += s_tmp[w];
    }
    if (i < n) s_cum[i] = before + x - c;
    __syncthreads();
  }
  if (tid == 0) s_cum[n] = carry;
  __syncthreads();
  return {carry, max(p.min_share, (carry + p.wgs - 1) / p.wgs)};
}

// One piece: rows [row0, row0 + rows) of the block's numbering against the keys of
// tiles [k0, k1) of a unit.
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
__device__ inline void row_of(const SharedParams& p, const ShPiece& u, int r, bool& live, int64_t& qrow, int& lim) {
  live = r < u.rows;
  const uint32_t R = (uint32_t)(u.row0 + (live ? r : 0));
  const uint32_t i = fastdiv(R, p.sg_div);
  const uint32_t t = R - i * (uint32_t)p.SG;
  const uint32_t s = fastdiv(t, p.g_div);
  const int b = u.b0 + (int)i;
  qrow = ((int64_t)b * p.S + s) * p.H + (int64_t)u.kvh * p.G + (t - s * (uint32_t)p.G);
  const int ctx = max(p.context_lens[b], 0);
  const int n = ctx <= p.MB * p.BS ? min(ctx - p.S + (int)s + 1, u.end) : 0;
  lim = live ? n : 0x7fffffff;
}

// q row at dims d0 + 32 st .. of 8 (NS steps of `stride` dims) as hi (+ lo) words of
// the tiles' type.  fp16 hi + lo rows are scaled by the power of two that puts the
// row's largest element in [2^14, 2^15), and their scores by the inverse, returned
// in `back` (other: a lane that holds other dims of the row, xor'ed in steps).
template <bool kBf, bool kSplit, int NS, int kStep, int kFrom>
__device__ inline void load_q(const SharedParams& p, bool live, int64_t qrow, int d0, u32x4_t (&hi)[NS],
                              u32x4_t (&lo)[kSplit ? NS : 1], float& back) {
  back = 1.0f;
  if constexpr (!kSplit) {
#pragma unroll
    for (int ks = 0; ks < NS; ++ks) {
      hi[ks] = load16(p.q, (qrow * p.D + d0 + kStep * ks) * 2);
      if (!live) hi[ks] = u32x4_t{0u, 0u, 0u, 0u};
    }
    return;
  }
  float x[NS][8];
#pragma unroll
  for (int ks = 0; ks < NS; ++ks) {
    load8f(p.q, p.q_dtype, qrow * p.D + d0 + kStep * ks, x[ks]);
    if (!live) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[ks][e] = 0.0f;
    }
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

// Byte offsets of one key row's K and V under the piece's head, and what is wrong
// with it: a row past the unit, or on a page outside the cache, is read at row 0 of
// block 0 (in bounds, NB >= 1) and not used.
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

// ------------------------------------------------------------------- wide --

template <int D>
struct ShShape {
  static constexpr int KB = D <= 128 ? 64 : 32;    // keys per LDS tile of the wide body
  static constexpr int MT = KB / 32;
  static constexpr int KS = D / 16;
  static constexpr int DT = D / 32;
  static constexpr int NCH = D / 8;
  static constexpr int TPD = 64 / NCH;             // rows per 1 KB load
  static constexpr int RPW = KB / kShWaves;        // rows a wave loads
  static constexpr int NP = RPW / TPD;             // loads per wave and tile
  static constexpr int TILE = KB * D;              // 16-bit elements
  static constexpr int KT = 32;                    // keys per wave tile of the thin body
  static constexpr int NDMA = KT / TPD;
  static constexpr int LDS_WIDE = 4 * TILE * 2;    // K and V, two tiles
  static constexpr int LDS_THIN = kShWaves * KT * D * 2 > kShWaves * 16 * D * 4 ? kShWaves * KT * D * 2
                                                                               : kShWaves * 16 * D * 4;
  static constexpr int LDS_BODY = LDS_WIDE > LDS_THIN ? LDS_WIDE : LDS_THIN;
  static constexpr int LDS_PLAN = (8 + 2 * kSharedMaxSeqs + 1) * 4;
  static constexpr int LDS = LDS_BODY > LDS_PLAN ? LDS_BODY : LDS_PLAN;
  static_assert(NP >= 1 && RPW % TPD == 0, "tile shape");
};

struct ShFlags {
  unsigned long long bad[3];  // per tile, three in turn: keys on pages outside the cache
  int odd;                    // something was taken out of V (restore_odd)
  int lim[kSharedWide];       // end of the keys that each row attends
};

// Adds to the piece's states what sanitize() took out of V: the elements that are not
// finite, in tiles of KT keys that some row does not see whole (the shortest row ends
// at `least`), for the rows that see their keys.
template <typename KV>
__device__ __forceinline__ void restore_odd(const SharedParams& p, const ShPiece& u, const int* lim, int least, int KT) {
  __syncthreads();  // the states and limits are written
  const char* vbase = static_cast<const char*>(p.v) + (int64_t)u.kvh * p.v_sh * KV::kBytes;
  const int n0 = u.first + u.k0 * kSharedTile, n1 = min(u.first + u.k1 * kSharedTile, u.end);
  for (int key = max(n0, u.lo); key < n1; ++key) {
    const int t0 = n0 + (key - n0) / KT * KT;
    if (t0 >= u.lo && t0 + KT <= least) continue;
    const int pg = (int)fastdiv((uint32_t)key, p.bs_div);
    const ShRow row = key_row(p, u.table[pg], key - pg * p.BS, true, KV::kBytes);
    if (row.bad) continue;
    for (int d = threadIdx.x; d < p.D; d += kShThreads) {
      const float x = v_elem<KV>(vbase, row.v, d);
      if (__builtin_isfinite(x)) continue;
      for (int r = 0; r < u.rows; ++r)
        if (key < lim[r]) p.ws_acc[(u.slot + r) * p.D + d] += x;
    }
  }
}

template <typename KV, bool kBf, int D, bool kSplitQ, bool kSplitP>
__device__ __forceinline__ void wide_piece(const SharedParams& p, const ShPiece& u, char* lds, ShFlags* fl, int* s_min) {
  using Sh = ShShape<D>;
  using Tl = ShTile<KV, kBf>;
  constexpr int KB = Sh::KB, MT = Sh::MT, KS = Sh::KS, DT = Sh::DT, NCH = Sh::NCH, TPD = Sh::TPD, RPW = Sh::RPW,
                NP = Sh::NP;
  constexpr int EB = KV::kBytes;
  uint16_t* sK = reinterpret_cast<uint16_t*>(lds);
  uint16_t* sV = sK + 2 * Sh::TILE;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int hh = lane >> 5;

  bool live;
  int64_t qrow;
  int lim;
  row_of(p, u, wave * 32 + (lane & 31), live, qrow, lim);
  const bool busy = wave * 32 < u.rows;
  u32x4_t qf[KS], ql[kSplitQ ? KS : 1];
  float back;
  load_q<kBf, kSplitQ, KS, 16, 32>(p, live, qrow, hh * 8, qf, ql, back);
  const float qscale = p.qscale * back;

  // The shortest row of this wave and of the block.
  int wmin = lim;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) wmin = min(wmin, __shfl_xor(wmin, o, 64));
  wmin = __builtin_amdgcn_readfirstlane(wmin);
  if (lane == 0) s_min[wave] = wmin;
  if (hh == 0) fl->lim[wave * 32 + lane] = lim;
  if (threadIdx.x < 3) fl->bad[threadIdx.x] = 0;
  if (threadIdx.x == 0) fl->odd = 0;
  __syncthreads();
  const int bmin = min(min(s_min[0], s_min[1]), min(s_min[2], s_min[3]));

  const char* kbase = static_cast<const char*>(p.k) + (int64_t)u.kvh * p.k_sh * EB;
  const char* vbase = static_cast<const char*>(p.v) + (int64_t)u.kvh * p.v_sh * EB;
  const int n0 = u.first + u.k0 * kSharedTile;  // first key of the piece
  const int n1 = min(u.first + u.k1 * kSharedTile, u.end);
  const int ntiles = (n1 - n0 + KB - 1) / KB;

  // This wave loads rows [RPW wave, RPW wave + RPW) of a tile; lane r holds row
  // r % RPW's page.
  const int myrow = wave * RPW + lane % RPW;
  auto page_at = [&](int tile, int& off) {
    const int key = n0 + tile * KB + myrow;
    const int kk = min(key, n1 - 1);
    const int pg = (int)fastdiv((uint32_t)kk, p.bs_div);
    off = kk - pg * p.BS;
    return u.table[pg];
  };
  uint32_t use = 0;                      // bit i: this lane's row of load i is used
  typename Tl::Raw kr[Tl::kF8 ? NP : 1], vr[Tl::kF8 ? NP : 1];
  ShRow mine;
  auto issue = [&](int tile, int32_t blk, int off) {
    mine = key_row(p, blk, off, n0 + tile * KB + myrow < n1, EB);
    if (mine.bad && lane < RPW) atomicOr(&fl->bad[tile % 3], 1ull << myrow);
    use = 0;
    uint16_t* dK = sK + (tile & 1) * Sh::TILE + wave * RPW * D;
    uint16_t* dV = sV + (tile & 1) * Sh::TILE + wave * RPW * D;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = i * TPD + lane / NCH, row = wave * RPW + r;
      const uint64_t ko = shfl64(mine.k, r), vo = shfl64(mine.v, r);
      use |= (uint32_t)__shfl((int)mine.use, r, 64) << i;
      const char* ka = kbase + ko + kpos<D>(row, lane % NCH) * 8 * EB;
      const char* va = vbase + vo + vpos<D>(row, lane % NCH) * 8 * EB;
      if constexpr (Tl::kF8) {
        kr[i] = *reinterpret_cast<const typename Tl::Raw*>(ka);
        vr[i] = *reinterpret_cast<const typename Tl::Raw*>(va);
      } else {
        lds_dma16_async(ka, (lds_void_t*)(dK + i * 512));
        lds_dma16_async(va, (lds_void_t*)(dV + i * 512));
      }
    }
  };
  // The tile's loads have landed: widen FP8 codes, zero the V rows that are not
  // used, take out what is not finite where some row does not see the whole tile.
  auto finish = [&](int tile) {
    const int t0 = n0 + tile * KB;
    const bool masked = t0 < u.lo || t0 + KB > bmin;
    uint16_t* dK = sK + (tile & 1) * Sh::TILE + wave * RPW * D + lane * 8;
    uint16_t* dV = sV + (tile & 1) * Sh::TILE + wave * RPW * D + lane * 8;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      u32x4_t x;
      if constexpr (Tl::kF8) {
        *reinterpret_cast<u32x4_t*>(dK + i * 512) = Tl::widen(kr[i]);
        x = Tl::widen(vr[i]);
      }
      const bool dead = !((use >> i) & 1u);
      if (Tl::kF8 || dead || masked) {
        if constexpr (!Tl::kF8) x = *reinterpret_cast<const u32x4_t*>(dV + i * 512);
        if (dead) {
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

  auto compute = [&](int tile) {
    const uint16_t* cK = sK + (tile & 1) * Sh::TILE;
    const uint16_t* cV = sV + (tile & 1) * Sh::TILE;
    const int t0 = n0 + tile * KB;
    f32x16_t st[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int i = 0; i < 16; ++i) st[mt][i] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const u32x4_t a = *reinterpret_cast<const u32x4_t*>(cK + swk<D>(mt * 32 + (lane & 31), 2 * ks + hh));
        st[mt] = mfma32<kBf>(a, qf[ks], st[mt]);
        if constexpr (kSplitQ) st[mt] = mfma32<kBf>(a, ql[ks], st[mt]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    const unsigned long long bad = fl->bad[tile % 3];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) st[mt] *= qscale;
    // This lane's key of slot i is t0 + 4 hh + mt 32 + 8 (i / 4) + i % 4.
    if (bad != 0) {
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
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__builtin_amdgcn_ballot_w64(mx > m + kLazyRescale) != 0) {
      asm volatile("");
      const float mn = fmaxf(m, mx);
      const float corr = mn == -__builtin_inff() ? 1.0f : fast_exp2(m - mn);
      m = mn;
      l *= corr;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= corr;
    }
    const float negm = m == -__builtin_inff() ? 0.0f : -m;
#pragma unroll
    for (int ts = 0; ts < KB / 16; ++ts) {
      uint32_t w[4], wl[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = 8 * (ts & 1) + 2 * j;
        const float p0 = fast_exp2(st[ts >> 1][i] + negm), p1 = fast_exp2(st[ts >> 1][i + 1] + negm);
        l += p0 + p1;
        w[j] = pack2<kBf>(p0, p1);
        if constexpr (kSplitP) {
          const float2_t r = unpack2<kBf>(w[j]);
          wl[j] = pack2<kBf>(p0 - r[0], p1 - r[1]);
        }
      }
      const u32x4_t pb = u32x4_t{w[0], w[1], w[2], w[3]};
      const int r0 = ts * 16 + 4 * hh + ((lane & 15) >> 2);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int c = dt * 32 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        const short4_t a0 =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)(cV + swv<D>(r0, c >> 3) + (c & 7)));
        const short4_t a1 =
            __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4_t*)(cV + swv<D>(r0 + 8, c >> 3) + (c & 7)));
        const uint64_t x0 = __builtin_bit_cast(uint64_t, a0), x1 = __builtin_bit_cast(uint64_t, a1);
        const u32x4_t a = u32x4_t{(uint32_t)x0, (uint32_t)(x0 >> 32), (uint32_t)x1, (uint32_t)(x1 >> 32)};
        o[dt] = mfma32<kBf>(a, pb, o[dt]);
        if constexpr (kSplitP) o[dt] = mfma32<kBf>(a, u32x4_t{wl[0], wl[1], wl[2], wl[3]}, o[dt]);
      }
    }
  };

  int off;
  int32_t blk = page_at(0, off);
  issue(0, blk, off);
  if (ntiles > 1) blk = page_at(1, off);
#pragma unroll 1
  for (int i = 0; i < ntiles; ++i) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of tile i
    finish(i);
    __syncthreads();
    asm volatile("" ::: "memory");
    if (threadIdx.x == 0) fl->bad[(i + 2) % 3] = 0;
    if (i + 1 < ntiles) {
      issue(i + 1, blk, off);
      if (i + 2 < ntiles) blk = page_at(i + 2, off);
    }
    if (busy) compute(i);
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
  if (fl->odd) restore_odd<KV>(p, u, fl->lim, bmin, KB);
  __syncthreads();  // (the next piece reuses the tiles and flags)
}

// ------------------------------------------------------------------- thin --

template <typename KV, bool kBf, int D, bool kSplitQ, bool kSplitP>
__device__ __forceinline__ void thin_piece(const SharedParams& p, const ShPiece& u, char* lds, ShFlags* fl,
                                           float (*s_m)[16], float (*s_l)[16]) {
  using Sh = ShShape<D>;
  using Tl = ShTile<KV, kBf>;
  constexpr int KT = Sh::KT, KS = D / 32, NDT = D / 16, NCH = Sh::NCH, TPD = Sh::TPD, NDMA = Sh::NDMA;
  constexpr int EB = KV::kBytes;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, kg = lane >> 4;
  uint16_t* sV = reinterpret_cast<uint16_t*>(lds) + wave * KT * D;

  bool live;
  int64_t qrow;
  int lim;
  row_of(p, u, col, live, qrow, lim);
  u32x4_t qf[KS], ql[kSplitQ ? KS : 1];
  float back;
  load_q<kBf, kSplitQ, KS, 32, 16>(p, live, qrow, kg * 8, qf, ql, back);
  const float qscale = p.qscale * back;
  int wmin = lim;
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) wmin = min(wmin, __shfl_xor(wmin, o, 64));
  wmin = __builtin_amdgcn_readfirstlane(wmin);
  if (threadIdx.x < 16) fl->lim[col] = lim;
  if (threadIdx.x == 0) fl->odd = 0;
  __syncthreads();

  const char* kbase = static_cast<const char*>(p.k) + (int64_t)u.kvh * p.k_sh * EB;
  const char* vbase = static_cast<const char*>(p.v) + (int64_t)u.kvh * p.v_sh * EB;
  const int n0 = u.first + u.k0 * kSharedTile;
  const int n1 = min(u.first + u.k1 * kSharedTile, u.end);
  constexpr int kStep = kShWaves * KT;
  const int base = n0 + wave * KT;
  const int ntiles = base < n1 ? (n1 - base + kStep - 1) / kStep : 0;

  // One tile in registers.  Its V is freed into LDS and its K into the scores at the
  // start of a round, and the next tile's loads take their place at once: eight
  // waves of a CU keep 128 KB in flight (D = 128) at half the registers of two tiles.
  typename Tl::Raw tk[2][KS], tv[NDMA];
  const int myrow = lane & 31;
  auto page_at = [&](int tile, int& off) {
    const int kk = min(base + tile * kStep + myrow, n1 - 1);
    const int pg = (int)fastdiv((uint32_t)kk, p.bs_div);
    off = kk - pg * p.BS;
    return u.table[pg];
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
      tv[i] = *reinterpret_cast<const typename Tl::Raw*>(vbase + shfl64(r.v, row) + (lane % NCH) * 8 * EB);
    }
  };

  float4_t o[NDT];
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt) o[dt] = float4_t{0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), l = 0.0f;

  int off = 0;
  int32_t blk = 0;
  ShRow row;
  if (ntiles > 0) {
    blk = page_at(0, off);
    row = key_row(p, blk, off, base + myrow < n1, EB);
    load_k(row);
    load_v(row);
    if (ntiles > 1) blk = page_at(1, off);
  }
#pragma unroll 1
  for (int i = 0; i < ntiles; ++i) {
    const int first = base + i * kStep;
    const uint32_t bad = (uint32_t)__builtin_amdgcn_ballot_w64(row.bad);    // keys on pages outside the cache
    const uint32_t dead = (uint32_t)__builtin_amdgcn_ballot_w64(!row.use);  // keys not used
    const bool masked = first < u.lo || first + KT > wmin;
    const bool more = i + 1 < ntiles;
    if (more) row = key_row(p, blk, off, first + kStep + myrow < n1, EB);
    if (i + 2 < ntiles) blk = page_at(i + 2, off);
    // V to LDS; rows not used are zeroed, what is not finite taken out where a row
    // does not see the whole tile.
#pragma unroll
    for (int j = 0; j < NDMA; ++j) {
      u32x4_t x = Tl::widen(tv[j]);
      const int r = j * TPD + lane / NCH;
      if (dead != 0 || masked) {
        if ((dead >> r) & 1u) {
          x = u32x4_t{0u, 0u, 0u, 0u};
        } else if (masked && sanitize<kBf>(x)) {
          fl->odd = 1;
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
      st[mt] *= qscale;
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
    float mx = fmaxf(fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3])),
                     fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    if (__builtin_amdgcn_ballot_w64(mx > m + kLazyRescale) != 0) {
      asm volatile("");
      const float mn = fmaxf(m, mx);
      const float corr = mn == -__builtin_inff() ? 1.0f : fast_exp2(m - mn);
      m = mn;
      l *= corr;
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o[dt] *= corr;
    }
    const float negm = m == -__builtin_inff() ? 0.0f : -m;
    uint32_t w[4], wl[4];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float p0 = fast_exp2(st[mt][2 * j] + negm), p1 = fast_exp2(st[mt][2 * j + 1] + negm);
        l += p0 + p1;
        w[mt * 2 + j] = pack2<kBf>(p0, p1);
        if constexpr (kSplitP) {
          const float2_t r = unpack2<kBf>(w[mt * 2 + j]);
          wl[mt * 2 + j] = pack2<kBf>(p0 - r[0], p1 - r[1]);
        }
      }
    }
    const u32x4_t pb = u32x4_t{w[0], w[1], w[2], w[3]};
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
      o[dt] = mfma16<kBf>(a, pb, o[dt]);
      if constexpr (kSplitP) o[dt] = mfma16<kBf>(a, u32x4_t{wl[0], wl[1], wl[2], wl[3]}, o[dt]);
    }
  }

  // Join the waves' states.
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  __syncthreads();
  float* s_acc = reinterpret_cast<float*>(lds);  // [waves][16][D]
#pragma unroll
  for (int dt = 0; dt < NDT; ++dt)
    *reinterpret_cast<float4_t*>(s_acc + (wave * 16 + col) * D + dt * 16 + kg * 4) = o[dt];
  if (kg == 0) {
    s_m[wave][col] = m;
    s_l[wave][col] = l;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < u.rows * (D / 4); x += kShThreads) {
    const int r = x / (D / 4), d = (x - r * (D / 4)) * 4;
    float M = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) M = fmaxf(M, s_m[w][r]);
    float L = 0.0f;
    float4_t A = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kShWaves; ++w) {
      const float f = s_m[w][r] == -__builtin_inff() ? (s_l[w][r] != 0.0f ? s_l[w][r] : 0.0f) : fast_exp2(s_m[w][r] - M);
      L += s_l[w][r] * f;
      const float4_t a = *reinterpret_cast<const float4_t*>(s_acc + (w * 16 + r) * D + d);
      if (f != 0.0f) A += a * f;
    }
    const int64_t at = u.slot + r;
    *reinterpret_cast<float4_t*>(p.ws_acc + at * D + d) = A;
    if (d == 0) {
      p.ws_m[at] = M;
      p.ws_l[at] = L;
    }
  }
  __syncthreads();
  if (fl->odd) restore_odd<KV>(p, u, fl->lim, wmin, KT);
  __syncthreads();
}

// ----------------------------------------------------------------- kernel --

template <typename KV, bool kBf, int D, bool kSplitQ, bool kSplitP>
__global__ __launch_bounds__(kShThreads) __attribute__((amdgpu_waves_per_eu(D <= 128 ? 2 : 1)))
void shared_kernel(const SharedParams p) {
  __shared__ __attribute__((aligned(16))) char lds[ShShape<D>::LDS];
  __shared__ int32_t s_cum[2 * kSharedMaxSeqs + 1];
  __shared__ ShFlags s_fl;
  __shared__ float s_m[kShWaves][16], s_l[kShWaves][16];
  __shared__ int s_min[kShWaves];
  int fault;
  const ShPlan pl = plan_scan(p, s_cum, reinterpret_cast<int32_t*>(lds), fault);
  const int n = p.NG + p.B;
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) {
      p.ws_meta[0] = pl.share;
      p.ws_meta[1] = fault;
    }
    for (int i = threadIdx.x; i <= n; i += kShThreads) p.ws_meta[2 + i] = fault ? 0 : s_cum[i];
  }
  if (fault) return;
  const int w = blockIdx.x;
  int64_t pos = (int64_t)w * pl.share;
  const int64_t stop = min(pos + pl.share, (int64_t)pl.total);
  while (pos < stop) {
    // The entry (group or sequence) that holds `pos`: the last with s_cum <= pos.
    int lo = 0, hi = n;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_cum[mid] <= pos) lo = mid; else hi = mid;
    }
    const int entry = __builtin_amdgcn_readfirstlane(lo);
    ShPiece u;
    int tiles, rows, blocks;
    if (entry < p.NG) {
      u.b0 = p.group_starts[entry];
      rows = (p.group_starts[entry + 1] - u.b0) * p.SG;
      u.end = prefix_of(p.prefix_lens[entry]);
      u.first = u.lo = 0;
      tiles = tiles_of(u.end);
      blocks = row_blocks(rows);
    } else {
      u.b0 = entry - p.NG;
      const int g = group_of(p.group_starts, p.NG, u.b0);
      rows = p.SG;
      u.lo = g < 0 ? 0 : prefix_of(p.prefix_lens[g]);
      u.first = own_first(u.lo);
      u.end = p.context_lens[u.b0];
      tiles = tiles_of(u.end - u.first);
      blocks = p.own_rb;
    }
    const int c = tile_cost(p, rows);
    const int local = (int)(pos - s_cum[entry]);
    const int unit = local / (tiles * c);
    const int64_t begin = (int64_t)s_cum[entry] + (int64_t)unit * tiles * c;  // the unit's place on the line
    u.k0 = (int)((pos - begin + c - 1) / c);
    u.k1 = (int)min((int64_t)tiles, (stop - begin + c - 1) / c);
    pos = begin + (int64_t)tiles * c;
    if (u.k0 >= u.k1) continue;
    u.kvh = unit / blocks;
    u.row0 = (unit - u.kvh * blocks) * kSharedWide;
    u.rows = min(rows - u.row0, kSharedWide);
    u.table = p.block_tables + (int64_t)u.b0 * p.bt_stride;
    if (entry < p.NG) {
      u.slot = (int64_t)w * kSharedWide + (int64_t)p.HKV * u.b0 * p.SG + (int64_t)u.kvh * rows + u.row0;
    } else {
      const int64_t prefix_rows = (int64_t)p.wgs * kSharedWide + (int64_t)p.HKV * p.B * p.SG;
      u.slot = prefix_rows + (int64_t)w * (p.SG <= kSharedThin ? kSharedThin : kSharedWide) +
               ((int64_t)u.b0 * p.HKV + u.kvh) * p.SG + u.row0;
    }
    if (rows <= kSharedThin)
      thin_piece<KV, kBf, D, kSplitQ, kSplitP>(p, u, lds, &s_fl, s_m, s_l);
    else
      wide_piece<KV, kBf, D, kSplitQ, kSplitP>(p, u, lds, &s_fl, s_min);
  }
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
