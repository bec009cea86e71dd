// pa_shared_merge.hip -- joins the states of a shared-prefix call (pa_shared.hpp) into
// the output rows:
//   M = max_i m_i, out = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i
// over the pieces of the row's prefix unit and of its own keys' unit, whose places
// follow from the plan that the first launch left in the workspace.  One wave
// per row, as pa_reduce.hip: lane (r, c) reads dims 4c .. 4c + 3 of every RI-th
// state, a round of NL loads covers NL * RI of them.
//
// Its chain of round trips bounds it where states are few (the plan, then the states:
// 3.6 us with the launch), their bytes where they are many (8192 rows of ten states of
// 128: 42 MB in 11.7 us, 3.6 TB/s).  Joining in the last work-group to arrive would save
// the launch, but needs counters that somebody clears between calls.
#include "pa_shared.hpp"

namespace pa {

constexpr int kMergeWaves = 4;

template <int D>
__global__ __launch_bounds__(64 * kMergeWaves) void shared_merge_kernel(const SharedParams p) {
  constexpr int LR = D / 4;   // lanes per state
  constexpr int RI = 64 / LR; // states per load instruction
  constexpr int NL = 8;       // loads per lane per round
  const int lane = threadIdx.x & 63;
  const int r = lane / LR, c = lane % LR;
  const int64_t f = (int64_t)blockIdx.x * kMergeWaves + (threadIdx.x >> 6);
  const int64_t row = f / p.H;  // [B, S]
  if (row >= (int64_t)p.B * p.S) return;
  const int h = (int)(f - row * p.H);
  const int b = (int)(row / p.S), s = (int)(row - (int64_t)b * p.S);
  const int kvh = h / p.G;
  const int mine = s * p.G + (h - kvh * p.G);  // row among the sequence's
  const int32_t* meta = p.ws_meta + kSharedMeta * (b + 1);
  const int share = p.ws_meta[0], maxctx = p.MB * p.BS;
  const int P = meta[0], ctx = max(meta[1], 0), b0 = meta[2], rows = meta[3], cum_group = meta[4], cum_own = meta[5];
  const int keys = ctx - p.S + s + 1;  // that the row attends
  const bool bad = p.ws_meta[1] != 0 || ctx > maxctx || (P > maxctx && ctx > 0);

  // The states: n1 of the prefix from workspace row a1 on, n2 of the own keys from a2.
  int n1 = 0, n2 = 0, step2 = kSharedWide;
  int64_t a1 = 0, a2 = 0;
  if (!bad && keys > 0) {
    int first;
    if (P > 0) {
      const int at = (b - b0) * p.SG + mine, tiles = wide_tiles(P);
      const int unit = kvh * row_blocks(rows) + at / kSharedWide;
      unit_workers(cum_group + unit * wide_cost(tiles), kSharedWideStart, kSharedWideCost, tiles, share, first, n1);
      a1 = prefix_slot(p, first, b0, rows, kvh, at);
    }
    if (ctx > P) {
      const int tiles = own_tiles(p, ctx - own_first(P));
      const int begin = cum_own + (kvh * p.own_rb + mine / kSharedWide) * own_cost(p, tiles);
      if (p.thin) {
        unit_workers(begin, kSharedThinStart, kSharedThinCost, tiles, share / kShWaves, first, n2);
        step2 = kSharedThin;
      } else {
        unit_workers(begin, kSharedWideStart, kSharedWideCost, tiles, share, first, n2);
      }
      a2 = own_slot(p, first, b, kvh, mine);
    }
  }
  auto place = [&](int i) { return i < n1 ? a1 + (int64_t)i * kSharedWide : a2 + (int64_t)(i - n1) * step2; };
  const int all = n1 + n2;
  // One round trip: the first 64 states' maxima and sums, and the first round of rows.
  float4_t x[NL];
  auto load_rows = [&](int i0) {
#pragma unroll
    for (int j = 0; j < NL; ++j) {
      const int i = i0 + j * RI + r;
      x[j] = i < all ? *reinterpret_cast<const float4_t*>(p.ws_acc + place(i) * D + 4 * c) : float4_t{0.f, 0.f, 0.f, 0.f};
    }
  };
  float m = -__builtin_inff(), l = 0.0f;
  auto load_states = [&](int i0) {
    const bool on = i0 + lane < all;
    const int64_t at = place(on ? i0 + lane : 0);
    m = on ? p.ws_m[at] : -__builtin_inff();
    l = on ? p.ws_l[at] : 0.0f;
  };
  load_states(0);
  load_rows(0);
  float M = m;
  for (int i0 = 64; i0 < all; i0 += 64) M = fmaxf(M, i0 + lane < all ? p.ws_m[place(i0 + lane)] : -__builtin_inff());
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  float4_t acc = float4_t{0.f, 0.f, 0.f, 0.f};
  float L = 0.0f;
  for (int i0 = 0; i0 < all; i0 += 64) {
    if (i0 > 0) load_states(i0);
    // (A state that saw no key, or a key that cannot be read, has m = -inf: l says which.)
    const float w = m == -__builtin_inff() ? 0.0f : fast_exp2(m - M);
    L += l != l ? l : w * l;
    for (int k = 0; k < 64 && i0 + k < all; k += NL * RI) {
      if (i0 + k > 0) load_rows(i0 + k);
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const float wi = __shfl(w, (k + j * RI + r) & 63, 64);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = wi == 0.0f ? acc[e] : fmaf(wi, x[j][e], acc[e]);
      }
    }
  }
#pragma unroll
  for (int o = LR; o < 64; o <<= 1) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o, 64);
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) L += __shfl_xor(L, o, 64);
  if (r == 0) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      store_elem(p.out, p.out_dtype, f * D + 4 * c + e,
                 bad ? __builtin_nanf("") : keys <= 0 ? 0.0f : acc[e] * p.vscale / L);
  }
}

hipError_t launch_shared_merge(const SharedParams& p, hipStream_t stream) {
  const int64_t waves = (int64_t)p.B * p.S * p.H;
  const dim3 grid((unsigned)((waves + kMergeWaves - 1) / kMergeWaves)), block(64 * kMergeWaves);
  note_launch("pa::shared_merge_kernel<%d>", p.D);
  switch (p.D) {
    case 32: hipLaunchKernelGGL(shared_merge_kernel<32>, grid, block, 0, stream, p); break;
    case 64: hipLaunchKernelGGL(shared_merge_kernel<64>, grid, block, 0, stream, p); break;
    case 128: hipLaunchKernelGGL(shared_merge_kernel<128>, grid, block, 0, stream, p); break;
    case 256: hipLaunchKernelGGL(shared_merge_kernel<256>, grid, block, 0, stream, p); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace pa
