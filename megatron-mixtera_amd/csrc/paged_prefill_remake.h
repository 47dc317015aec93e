// Rows of the windowed prompt kernels whose result is not finite, made again from the keys that the row sees.
//
// A tile's products take every key of the tile: a key that a row does not see has probability zero there, and zero times a NaN
// or an infinity among the values is NaN.  The tile kernels look at their results once, at the end (one multiply-add per
// value: not measurable), and hand such rows to this walk, a wavefront per row, a lane per key for the scores and a lane per
// column for the values, with a running maximum: slow, and run only where there is something not finite in the tiles.  It stops at
// the first tile that leaves nothing but NaN, so that a model that gives NaN everywhere does not wait for it (15 565 rows of 32
// heads, window 1 024, 0.27 ms: all values NaN 2.7 ms, one column of them 76).  It also serves rows whose sums overflow 32 bits
// against a reference far below their largest score.
#pragma once

#include "mi_common.h"
#include "paged_prefill_params.h"

namespace mi {

// One row: query head hq (KV head h) of row `row` at position `pos` of request r, over tiles [v0, v1) of the walk `wt` (and tile
// 0 where `sinks_too`).  Every argument is the same in all lanes.  `split` >= 0: the row's partial of that range instead of its result.
template <int HD, int TILE, bool FP8, bool F16>
static __device__ __forceinline__ void remake_row(const PrefillParams& p, int r, int row, int h, int hq, int pos, int Lk, const WindowTiles& wt,
                                                  bool sinks_too, int v0, int v1, int split) {
  static_assert(TILE <= 64, "a lane per key");
  constexpr int ESZ = FP8 ? 1 : 2, NC = (HD + 63) / 64;
  const int lane = threadIdx.x & 63;
  const uint16_t* q = p.q + (int64_t)row * p.q_st + (int64_t)hq * p.q_sh;
  auto number = [](uint32_t bits) { return FP8 ? fp8x2_lo_to_f32(bits).x : to_f32<F16>((uint16_t)bits); };
  auto chunk_of_key = [&](int key) { return clamp_chunk(p.bt[(int64_t)r * p.bt_stride + key / p.chunk], p.n_chunks); };
  auto seen = [&](int key) {
    return lane < TILE && key <= pos && key < Lk && (key > pos - p.window || key < p.sinks);
  };
  auto score = [&](int key) {   // in powers of two
    const int pc = chunk_of_key(key);
    const uint8_t* k = p.kc + ((int64_t)pc * p.kv_sc + (int64_t)(key % p.chunk) * p.kv_st + (int64_t)h * p.kv_sh) * ESZ;
    float s = 0.f;
    for (int d = 0; d < HD; ++d)
      s = __builtin_fmaf(to_f32<F16>(q[d]), number(FP8 ? (uint32_t)k[d] : (uint32_t)reinterpret_cast<const uint16_t*>(k)[d]), s);
    return s * (FP8 ? p.k_scale[(int64_t)pc * p.Hkv + h] : 1.f) * p.scale_log2;
  };
  float m = -INFINITY, l = 0.f, acc[NC] = {};
  const int before = sinks_too ? v0 - 1 : v0;
  bool nan = false;   // (uniform) a score in sight is no number, or no column's sum is one any more
  for (int v = before; v < v1 && !nan; ++v) {
    const int key0 = (v < v0 ? 0 : wt.real(v)) * TILE, key = key0 + lane;
    const bool mine = seen(key);
    const float s = mine ? score(key) : -INFINITY;
    nan = __builtin_amdgcn_ballot_w64(__builtin_isnan(s)) != 0;
    if (nan) break;
    float most = s;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    const float moved = fmaxf(m, most), ref = moved == -INFINITY ? 0.f : moved;
    const float shrink = fast_exp2(m - ref), e = fast_exp2(s - ref);
    m = moved;
    l = l * shrink + e;
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c] = __builtin_isinf(acc[c]) ? acc[c] : acc[c] * shrink;   // (an infinity stays one)
    for (uint64_t left = __builtin_amdgcn_ballot_w64(mine); left; left &= left - 1) {
      const int j = __builtin_ctzll(left);
      const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(e), j));
      const int pc = chunk_of_key(key0 + j);
      const uint8_t* x = p.vc + ((int64_t)pc * p.kv_sc + (int64_t)((key0 + j) % p.chunk) * p.kv_st + (int64_t)h * p.kv_sh) * ESZ;
      const float scale = FP8 ? p.v_scale[(int64_t)pc * p.Hkv + h] : 1.f;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const int d = lane + 64 * c;
        if (d < HD) {
          const float n = number(FP8 ? (uint32_t)x[d] : (uint32_t)reinterpret_cast<const uint16_t*>(x)[d]) * scale;
          acc[c] += __builtin_isinf(n) ? n : w * n;   // (also where the probability is too small for 32 bits)
        }
      }
    }
    bool left_one = false;
#pragma unroll
    for (int c = 0; c < NC; ++c) left_one |= lane + 64 * c < HD && !__builtin_isnan(acc[c]);
    nan = __builtin_amdgcn_ballot_w64(left_one) == 0;
  }
  const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
  if (nan) l = __uint_as_float(0x7fc00000u);
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int d = lane + 64 * c;
    if (d >= HD) continue;
    if (split < 0) p.out[(int64_t)row * p.o_st + (int64_t)hq * p.o_sh + d] = f32_to_16<F16>(acc[c] * inv);
    else p.split_o[(((int64_t)split * p.T + row) * p.Hq + hq) * HD + d] = acc[c] * inv;
  }
  // (a sum that is no number must not reach the merge's weights, which would drop the row: its values carry it there)
  if (split >= 0 && lane == 0)
    p.split_lse[((int64_t)split * p.T + row) * p.Hq + hq] = l == 0.f ? -INFINITY : __builtin_isnan(l) ? 0.f : ref + fast_log2(l);
}

// The 16 rows of tile `nt` of a wavefront (accumulators of row m16 and a quarter of its columns in a lane): whether the lane's row
// is finite.  Rows that are not are made again and written here.  `nq` query tokens from row `row0` at position `pos0` on, G
// heads of each from hq0 on.
template <int HD, int TILE, bool FP8, bool F16, int N>
static __device__ __forceinline__ bool finite_or_remade(const PrefillParams& p, const f32x4_t (&acc)[N], float l_tot, int nt, int nq, int G, int g_magic,
                                                        int r, int row0, int h, int hq0, int pos0, int Lk, const WindowTiles& wt, bool sinks_too,
                                                        int v0, int v1, int split) {
  float mark = l_tot * 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e)
#pragma unroll
    for (int i = 0; i < 4; ++i) mark = __builtin_fmaf(acc[e][i], 0.f, mark);
  uint64_t bad = __builtin_amdgcn_ballot_w64(!(mark == 0.f));
  if (__builtin_expect(bad == 0, 1)) return true;
  bad |= bad >> 32;
  bad = (bad | bad >> 16) & 0xffffu;
  for (uint32_t left = (uint32_t)bad; left; left &= left - 1) {
    const int n = 16 * nt + __builtin_ctz(left), i = (n * g_magic) >> 16;   // n / G
    if (i < nq) remake_row<HD, TILE, FP8, F16>(p, r, row0 + i, h, hq0 + n - i * G, pos0 + i, Lk, wt, sinks_too, v0, v1, split);
  }
  return !(bad >> (threadIdx.x & 15) & 1);
}

}  // namespace mi
