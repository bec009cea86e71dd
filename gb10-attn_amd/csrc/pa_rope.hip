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
// lanes of a row.  A lane group takes kRows heads of one token, all loaded
// before the first is used, with the same eight cosines and sines.
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

// LPR: lanes per row (a power of two, D / 16 of them in use).
template <int ACT, int DST, int LPR, int kRows>
__global__ __launch_bounds__(kRopeThreads) void qk_norm_rope_kernel(const RopeParams p) {
  const uint32_t idx = blockIdx.x * kRopeThreads + threadIdx.x;
  const uint32_t grp = idx / LPR;
  const uint32_t tl = fastdiv(grp, p.slice_div);  // token of this launch
  if (tl >= (uint32_t)p.T) return;
  const int head0 = (int)(grp - tl * p.slice_div.d) * kRows;
  const int64_t t = p.t_base + tl;
  const int u = (int)(idx % LPR);
  const bool on = u < p.D / 16;
  const bool turned = u < p.rot / 16;
  int a0, a1;  // first elements of this lane's chunks
  if (p.interleaved || !turned) {
    a0 = 16 * u;
    a1 = a0 + 8;
  } else {
    a0 = 8 * u;
    a1 = p.rot / 2 + 8 * u;
  }
  const int heads = p.H + 2 * p.HKV;

  float x[kRows][16];
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int h = head0 + r;
    const void* src = nullptr;
    int64_t off = 0;
    if (h < p.H) {
      src = p.q;
      off = t * p.q_st + (int64_t)h * p.q_sh;
    } else if (h < p.H + p.HKV) {
      src = p.key;
      off = t * p.key_st + (int64_t)(h - p.H) * p.key_sh;
    } else {
      src = p.value;
      off = t * p.val_st + (int64_t)(h - p.H - p.HKV) * p.val_sh;
    }
    if (on && h < heads) {
      float c[8], d[8];
      load8<ACT>(src, off + a0, c);
      load8<ACT>(src, off + a1, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[r][e] = c[e];
        x[r][8 + e] = d[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[r][e] = 0.0f;
    }
  }

  float cs[8], sn[8];
  if (turned && head0 < p.H + p.HKV) {
    const int64_t pos = load_index(p.positions, p.pos_i64, t);
    if (pos >= 0 && pos < p.table_rows) {
      load8_any(p.table, p.table_dtype, pos * p.table_st + 8 * u, cs);
      load8_any(p.table, p.table_dtype, pos * p.table_st + p.rot / 2 + 8 * u, sn);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) cs[e] = sn[e] = __builtin_nanf("");
    }
  }
  const int64_t slot = head0 + kRows > p.H ? load_index(p.slots, p.slot_i64, t) : -1;

#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const int h = head0 + r;
    const bool is_q = h < p.H, is_v = h >= p.H + p.HKV;
    const void* w = is_q ? p.q_weight : p.k_weight;
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 16; ++e) ss = fmaf(x[r][e], x[r][e], ss);
    ss = group_sum<LPR>(ss);  // (every lane of the group takes part)
    if (!on || h >= heads) continue;
    if (!is_v) {
      if (w) {
        const float rms = 1.0f / __builtin_sqrtf(fmaf(ss, p.inv_d, p.eps));
        float w0[8], w1[8];
        load8_any(w, p.weight_dtype, a0, w0);
        load8_any(w, p.weight_dtype, a1, w1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[r][e] = x[r][e] * rms * w0[e];
          x[r][8 + e] = x[r][8 + e] * rms * w1[e];
        }
      }
      if (turned) {
        if (p.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = x[r][2 * e], b = x[r][2 * e + 1];
            x[r][2 * e] = a * cs[e] - b * sn[e];
            x[r][2 * e + 1] = b * cs[e] + a * sn[e];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float a = x[r][e], b = x[r][8 + e];
            x[r][e] = a * cs[e] - b * sn[e];
            x[r][8 + e] = b * cs[e] + a * sn[e];
          }
        }
      }
    }
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      lo[e] = x[r][e];
      hi[e] = x[r][8 + e];
    }
    if (is_q) {
      const int64_t o = t * p.out_st + (int64_t)h * p.out_sh;
      switch (p.out_dtype) {
        case kF16: store8<kF16>(p.q_out, o + a0, lo); store8<kF16>(p.q_out, o + a1, hi); break;
        case kBF16: store8<kBF16>(p.q_out, o + a0, lo); store8<kBF16>(p.q_out, o + a1, hi); break;
        default: store8<kF32>(p.q_out, o + a0, lo); store8<kF32>(p.q_out, o + a1, hi); break;
      }
      continue;
    }
    if (slot < 0 || slot >= p.nslots) continue;
    const uint32_t blk = fastdiv((uint32_t)slot, p.bs_div);
    const uint32_t row = (uint32_t)slot - blk * (uint32_t)p.BS;
    if (!p.unit_scale) {
      const float s = is_v ? p.v_scale : p.k_scale, rc = is_v ? p.v_rcp : p.k_rcp;
      const bool fast = is_v ? p.v_fast : p.k_fast;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        lo[e] = div_rn(lo[e], s, rc, fast);
        hi[e] = div_rn(hi[e], s, rc, fast);
      }
    }
    const int hk = is_v ? h - p.H - p.HKV : h - p.H;
    const int64_t d = is_v ? (int64_t)blk * p.vc_sb + (int64_t)row * p.vc_st + (int64_t)hk * p.vc_sh
                           : (int64_t)blk * p.kc_sb + (int64_t)row * p.kc_st + (int64_t)hk * p.kc_sh;
    void* c = is_v ? p.vc : p.kc;
    store8<DST>(c, d + a0, lo);
    store8<DST>(c, d + a1, hi);
  }
}

// Lane groups per launch: fewer than 2^27, so that thread indices stay below 2^31.
constexpr int64_t kRopeMaxGroups = (int64_t)1 << 26;

template <int ACT, int DST, int LPR, int kRows>
static hipError_t launch_r(const RopeParams& p0, hipStream_t stream) {
  RopeParams p = p0;
  const int64_t slices = (p.H + 2 * (int64_t)p.HKV + kRows - 1) / kRows;
  p.slice_div = make_fastdiv((uint32_t)slices);
  const int64_t step = std::max<int64_t>(1, kRopeMaxGroups / slices);
  note_launch("pa::qk_norm_rope_kernel<%d, %d, %d, %d>", ACT, DST, LPR, kRows);
  for (int64_t t = 0; t < p0.T; t += step) {
    p.t_base = t;
    p.T = (int32_t)std::min<int64_t>(step, p0.T - t);
    const int64_t threads = p.T * slices * LPR;
    hipLaunchKernelGGL((qk_norm_rope_kernel<ACT, DST, LPR, kRows>),
                       dim3((unsigned)((threads + kRopeThreads - 1) / kRopeThreads)), dim3(kRopeThreads), 0, stream, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int ACT, int DST>
static hipError_t launch_r_d(const RopeParams& p, hipStream_t stream) {
  const int n = p.D / 16;
  const bool many = (int64_t)p.T * (p.H + 2 * p.HKV) >= 16384;
#define PA_ROPE(L) return many ? launch_r<ACT, DST, L, 4>(p, stream) : launch_r<ACT, DST, L, 1>(p, stream)
  if (n <= 2) PA_ROPE(2);
  if (n <= 4) PA_ROPE(4);
  if (n <= 8) PA_ROPE(8);
  PA_ROPE(16);
#undef PA_ROPE
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
