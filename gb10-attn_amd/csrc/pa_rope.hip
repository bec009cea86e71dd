// pa_rope.hip -- norm and rotation of new query and key heads, and the write of
// the keys and values into the paged cache, in one pass on gfx950.
//
// For every query and key head x of a token at position n (D elements, the
// first `rot` of them rotated):
//   y = x rsqrt(mean(x^2) + eps) w              (only where a weight is given)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)
// over pairs (i, i + rot / 2), or (2 i, 2 i + 1) interleaved, with cos and sin
// of pair i from row n of the caller's table.  Queries go to q_out, keys and
// values to the cache row of the token's slot (divided by the cache's scale).
// All arithmetic is fp32 and each result is rounded once, to the type it is
// stored in.
//
// Byte work: a head's row is read once, 16 bytes a load, and written once.  A
// lane holds two chunks of eight elements chosen so that both elements of each
// of its pairs are its own (chunks u and u + rot / 16; interleaved pairs are
// neighbours): the rotation needs no exchange, the norm one sum over the D / 16
// lanes of a row.  A lane group takes one head: two or four with the same cosines,
// sines and weights were slower at nearly every size, since fewer waves are in
// flight (32/8 heads of 128 in bf16, 1, 2 and 4 heads: 512 tokens 5.1, 5.6, 6.9 us;
// 8192 tokens 43.7, 45.4, 47.0).
//
// HBM-bound where the tokens are many: 8192 tokens of 32/8 heads of 128, 251 MB read
// and written, in 43.7 us (5.8 TB/s), into FP8 189 MB in 42; a launch and its chain of
// dependent loads (position, table row) where they are few: 32 tokens 3.6 us.
#include "pa_convert.hpp"

#include <algorithm>

namespace pa {

constexpr int kRopeThreads = 256;

__device__ inline void load8_any(const void* base, int dtype, int64_t idx, float (&x)[8]) {
  switch (dtype) {
    case kF16: load8<kF16>(base, idx, x); break;
    case kBF16: load8<kBF16>(base, idx, x); break;
    default: load8<kF32>(base, idx, x); break;
  }
}

__device__ inline int64_t load_index(const void* p, int i64, int64_t i) {
  return i64 ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int32_t*>(p)[i];
}

enum RopeKind { kRopeQ, kRopeK, kRopeV };

// x / s rounded to nearest: fast as div_rn; exact: 1 / s is a power of two.
__device__ inline void divide8(float (&x)[8], float s, float r, bool exact, bool fast) {
  if (exact) {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= r;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = div_rn(x[e], s, r, fast);
  }
}

// One work-group's share of the query, key or value heads: a group of LPR lanes (a
// power of two, D / 16 of them in use) takes one head of one token.  idx: the thread
// among those of its kind.
template <int ACT, int DST, int LPR, int kKind>
__device__ __forceinline__ void rope_heads(const RopeParams& p, uint32_t idx, const FastDiv& heads) {
  const uint32_t grp = idx / LPR;
  const uint32_t tl = fastdiv(grp, heads);  // token of this launch
  if (tl >= (uint32_t)p.T) return;
  const int h = (int)(grp - tl * heads.d);
  const int64_t t = p.t_base + tl;
  const int u = (int)(idx % LPR);
  const bool on = u < p.D / 16;
  const bool turned = kKind != kRopeV && u < p.rot / 16;
  int a0, a1;  // first elements of this lane's chunks
  if (p.interleaved || !turned) {
    a0 = 16 * u;
    a1 = a0 + 8;
  } else {
    a0 = 8 * u;
    a1 = p.rot / 2 + 8 * u;
  }
  const void* src = kKind == kRopeQ ? p.q : kKind == kRopeK ? p.key : p.value;
  const int64_t sh = kKind == kRopeQ ? p.q_sh : kKind == kRopeK ? p.key_sh : p.val_sh;
  const int64_t st = kKind == kRopeQ ? p.q_st : kKind == kRopeK ? p.key_st : p.val_st;

  float x[16], c[8], d[8];
  if (on) {
    const int64_t off = t * st + (int64_t)h * sh;
    load8<ACT>(src, off + a0, c);
    load8<ACT>(src, off + a1, d);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = d[e] = 0.0f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = c[e];
    x[8 + e] = d[e];
  }
  int64_t slot = 0;
  if constexpr (kKind != kRopeQ) slot = load_index(p.slots, p.slot_i64, t);
  float cs[8], sn[8], w0[8], w1[8];
  const void* w = kKind == kRopeQ ? p.q_weight : p.k_weight;
  if constexpr (kKind != kRopeV) {
    if (turned) {
      const int64_t pos = load_index(p.positions, p.pos_i64, t);
      if (pos >= 0 && pos < p.table_rows) {
        load8_any(p.table, p.table_dtype, pos * p.table_st + 8 * u, cs);
        load8_any(p.table, p.table_dtype, pos * p.table_st + p.rot / 2 + 8 * u, sn);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] = sn[e] = __builtin_nanf("");
      }
    }
    if (w && on) {
      load8_any(w, p.weight_dtype, a0, w0);
      load8_any(w, p.weight_dtype, a1, w1);
    }
  }

  if constexpr (kKind != kRopeV) {
    if (w) {  // (the same for every lane)
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) ss = fmaf(x[e], x[e], ss);
      ss = group_sum<LPR>(ss);  // (every lane of the group takes part)
      const float rms = 1.0f / __builtin_sqrtf(fmaf(ss, p.inv_d, p.eps));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] *= rms * w0[e];
        x[8 + e] *= rms * w1[e];
      }
    }
  }
  if (!on) return;
  if constexpr (kKind != kRopeV) {
    if (turned) {
      if (p.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = x[2 * e], b = x[2 * e + 1];
          x[2 * e] = a * cs[e] - b * sn[e];
          x[2 * e + 1] = b * cs[e] + a * sn[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = x[e], b = x[8 + e];
          x[e] = a * cs[e] - b * sn[e];
          x[8 + e] = b * cs[e] + a * sn[e];
        }
      }
    }
  }
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo[e] = x[e];
    hi[e] = x[8 + e];
  }
  if constexpr (kKind == kRopeQ) {
    const int64_t o = t * p.out_st + (int64_t)h * p.out_sh;
    switch (p.out_dtype) {
      case kF16: store8<kF16>(p.q_out, o + a0, lo); store8<kF16>(p.q_out, o + a1, hi); break;
      case kBF16: store8<kBF16>(p.q_out, o + a0, lo); store8<kBF16>(p.q_out, o + a1, hi); break;
      default: store8<kF32>(p.q_out, o + a0, lo); store8<kF32>(p.q_out, o + a1, hi); break;
    }
  } else {
    if (slot < 0 || slot >= p.nslots) return;
    const uint32_t blk = fastdiv((uint32_t)slot, p.bs_div);
    const uint32_t row = (uint32_t)slot - blk * (uint32_t)p.BS;
    if (!p.unit_scale) {
      const float s = kKind == kRopeV ? p.v_scale : p.k_scale, rc = kKind == kRopeV ? p.v_rcp : p.k_rcp;
      const bool fast = kKind == kRopeV ? p.v_fast : p.k_fast, exact = kKind == kRopeV ? p.v_exact : p.k_exact;
      divide8(lo, s, rc, exact, fast);
      divide8(hi, s, rc, exact, fast);
    }
    void* c = kKind == kRopeV ? p.vc : p.kc;
    const int64_t d = kKind == kRopeV ? (int64_t)blk * p.vc_sb + (int64_t)row * p.vc_st + (int64_t)h * p.vc_sh
                                      : (int64_t)blk * p.kc_sb + (int64_t)row * p.kc_st + (int64_t)h * p.kc_sh;
    store8<DST>(c, d + a0, lo);
    store8<DST>(c, d + a1, hi);
  }
}

// Query heads' work-groups first, then keys', then values': a wave serves one kind
// (with the kinds mixed in a wave it ran every kind's code: 8192 tokens of 32/8
// heads of 128 into FP8 63 us, so 43).
template <int ACT, int DST, int LPR>
__global__ __launch_bounds__(kRopeThreads) void qk_norm_rope_kernel(const RopeParams p) {
  int b = blockIdx.x;
  if (b < p.q_blocks) {
    rope_heads<ACT, DST, LPR, kRopeQ>(p, (uint32_t)b * kRopeThreads + threadIdx.x, p.q_heads);
  } else if ((b -= p.q_blocks) < p.kv_blocks) {
    rope_heads<ACT, DST, LPR, kRopeK>(p, (uint32_t)b * kRopeThreads + threadIdx.x, p.kv_heads);
  } else {
    b -= p.kv_blocks;
    rope_heads<ACT, DST, LPR, kRopeV>(p, (uint32_t)b * kRopeThreads + threadIdx.x, p.kv_heads);
  }
}

// Lane groups per launch and kind: fewer than 2^27, so that thread indices stay below 2^31.
constexpr int64_t kRopeMaxGroups = (int64_t)1 << 26;

template <int ACT, int DST, int LPR>
static hipError_t launch_r(const RopeParams& p0, hipStream_t stream) {
  RopeParams p = p0;
  p.q_heads = make_fastdiv((uint32_t)std::max(1, p.H));
  p.kv_heads = make_fastdiv((uint32_t)std::max(1, p.HKV));
  const int64_t step = std::max<int64_t>(1, kRopeMaxGroups / std::max(1, std::max(p.H, p.HKV)));
  note_launch("pa::qk_norm_rope_kernel<%d, %d, %d>", ACT, DST, LPR);
  for (int64_t t = 0; t < p0.T; t += step) {
    p.t_base = t;
    p.T = (int32_t)std::min<int64_t>(step, p0.T - t);
    auto blocks = [&](int64_t heads) { return (int32_t)((p.T * heads * LPR + kRopeThreads - 1) / kRopeThreads); };
    p.q_blocks = blocks(p.H);
    p.kv_blocks = blocks(p.HKV);
    hipLaunchKernelGGL((qk_norm_rope_kernel<ACT, DST, LPR>), dim3((unsigned)(p.q_blocks + 2 * p.kv_blocks)),
                       dim3(kRopeThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int ACT, int DST>
static hipError_t launch_r_d(const RopeParams& p, hipStream_t stream) {
  const int n = p.D / 16;
  if (n <= 2) return launch_r<ACT, DST, 2>(p, stream);
  if (n <= 4) return launch_r<ACT, DST, 4>(p, stream);
  if (n <= 8) return launch_r<ACT, DST, 8>(p, stream);
  return launch_r<ACT, DST, 16>(p, stream);
}

template <int ACT>
static hipError_t launch_r_act(const RopeParams& p, hipStream_t stream) {
  switch (p.cache_dtype) {
    case kF16: return launch_r_d<ACT, kF16>(p, stream);
    case kBF16: return launch_r_d<ACT, kBF16>(p, stream);
    case kF32: return launch_r_d<ACT, kF32>(p, stream);
    case kFP8: return launch_r_d<ACT, kFP8>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_qk_norm_rope(const RopeParams& p, hipStream_t stream) {
  switch (p.act_dtype) {
    case kF16: return launch_r_act<kF16>(p, stream);
    case kBF16: return launch_r_act<kBF16>(p, stream);
    case kF32: return launch_r_act<kF32>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace pa
