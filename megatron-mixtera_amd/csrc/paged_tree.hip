// Attention of drafted tokens over the paged cache (gfx950): the step of speculative decoding.
//
// Every request brings a tree of drafted tokens ("nodes"; a chain is a tree), whose keys and values are already in the
// cache as its last positions: node j of request r sits at position kv_lens[r] - n_r + j.  A node attends to the
// request's whole context (the positions before its nodes) and to the nodes that its row of bits names:
//   out[i] = sum_k P[i][k] V[k],  P[i] = softmax over the visible k of scale * q[i] . K[k].
// A row that sees nothing is zero.  The reference has no such call (its attention takes one new token, or a chain:
// megatron/core/transformer/attention.py:546-600).
//
// Work decomposition.  The (node, query head) pairs that share a KV head are its rows, 16 * NQ of them to a wavefront
// ("part"), one to eight parts to a "group".  The tiles of 16 * NT tokens of all (request, group) pairs are laid end to end
// and a fixed grid of workgroups takes equal spans of that sequence, whatever the mix of lengths; a workgroup's wavefronts
// take the parts of a group and neighbouring KV heads of the same tokens.  A pair within one span writes its result, any other
// leaves normalised fp32 partials and a base-2 log-sum-exp for the merge.  A span touches at most one pair that began
// before it and one that goes on after it, so two slots per workgroup hold all partials.
//
// S^T = K Q^T lands as lane (row m16, g) slot i = token 4g + i, the B operand of O^T += V^T P^T; a pair of 16-token sub-tiles
// makes one product of depth 32 (the products only need the same tokens in the same slots on both sides).  Two kernels: one
// keeps its tiles in registers (any cache; V's operand is built from row loads by byte permutes), one in LDS (below).
//
// Only the tiles that reach past the context look at the bits.  A node's value row may hold infinities or NaN that rows
// which do not see it must not meet, although a product multiplies it by their zeros: such values are taken out of their
// tile and added to the sums of the rows that see them.
//
// The register kernel is bound by memory: 64 requests of 6 nodes over 512-8 192 tokens (24 rows, 8 KV heads of 128, 1.12 GB) took
// it 205 us, 5.4 TB/s.  Loads through buffer descriptors, whose offsets stay in registers: 226 -> 222 us; wavefronts that meet every
// eighth tile, so that none is left to read alone at the end: 222 -> 208 (every tile: 210, and an fp8 cache 455 -> 495 where every
// eighth takes 444); a pair's start counted as a tile: 208 -> 205.
#include <atomic>
#include <type_traits>

#include "mi_capi_internal.h"
#include "mi_common.h"

namespace mi {

struct TreeParams {
  const uint16_t* q;
  int64_t q_st, q_sh;
  const uint8_t* kc;
  const uint8_t* vc;
  int64_t kv_sc;
  int32_t kv_st, kv_sh;
  const int32_t* bt;
  int64_t bt_stride;
  const int32_t* cu_q;
  const int32_t* lens;
  const uint32_t* mask;  // rows of bits, two words for each of the caller's
  int64_t mask_st;       // words between rows
  int32_t mask_words;
  uint16_t* out;
  int64_t o_st, o_sh;
  float* part_o;         // [2 grid][Hkv][rows][HD]
  float* part_lse;       // [2 grid][Hkv][rows]
  int4* pair_info;       // per (request, group), two of them: first and last workgroup, group, first row of q; nodes
  int32_t* pairs;        // how many there are
  const float* k_scale;
  const float* v_scale;
  uint64_t chunk_magic;
  uint32_t g_magic;      // 2^32 / G + 1, 0 for G = 1
  int32_t T, R, r_base, Hq, Hkv, G, chunk, n_chunks, table_cols, grid;
  int32_t last_slice;    // the launch that clears the rows behind the last request
  int32_t share, rows;   // wavefronts that share a KV head, and the rows they take together (a group)
  float scale_log2;
};

// Probabilities of fp16 are multiplied by 2^10 (a row's largest one; the sums are divided by the sum of all, which has the factor too):
// their normal numbers then reach down to e^-16 of the largest, where one of 1 at most would lose bits from 2^-14 on and be gone at 2^-25
// -- what a long context far below one token adds up to.  bf16 has the exponents anyway.
template <bool F16> constexpr float kTreeLift = F16 ? 10.f : 0.f;
constexpr int kTreeRequestsPerLaunch = 2048;  // (their prefix sums lie in LDS)

static __device__ __forceinline__ int tree_div_g(const TreeParams& p, int n) {
  return p.g_magic ? (int)__umulhi((uint32_t)n, p.g_magic) : n;
}
static __device__ __forceinline__ int tree_chunk_of(int tok, uint64_t magic) { return (int)(((uint64_t)(uint32_t)tok * magic) >> 40); }

// A wave-uniform pointer to memory that no kernel writes meanwhile: its loads are scalar.
template <typename T>
static __device__ __forceinline__ const __attribute__((address_space(4))) T* tree_constant(const T* ptr) {
  const uint64_t x = (uint64_t)(uintptr_t)ptr;
  return (const __attribute__((address_space(4))) T*)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) |
                                                      (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}

struct TreeSegment {
  int r, group, part;  // request, which of its groups, and which of its parts (the rows of a wavefront)
  int q_begin, nodes;  // rows of q, nodes of the request
  int len, ctx;        // cached tokens, those before the first node (may be negative: nodes without a position)
  int start, end;      // tokens of the segment
  bool whole;
  int slot, row0;      // partial: its place, and the part's first row in there
};

// Bits of four tokens, node j0 first, of a row of `words` 32-bit words; what lies before node 0 is context.
static __device__ __forceinline__ uint32_t tree_bits(const uint32_t* row, int words, int j0) {
  if (j0 <= -4) return 15u;
  const int j = max(j0, 0), w = j >> 5;
  const uint32_t lo = w < words ? row[w] : 0u, hi = w + 1 < words ? row[w + 1] : 0u;
  const uint32_t bits = (uint32_t)((((uint64_t)hi << 32) | lo) >> (j & 31));
  return j0 < 0 ? (bits << -j0) | ((1u << -j0) - 1u) : bits;
}

// Infinities and NaN among the values of a word (the sign bit of each that is one), the word without them, and, as operands
// of a product with what a row sees of their tokens, their places: an infinity counts 1, a negative one 64, a NaN 4096
// (exact in either type, and 16 of each fit).  The product says what a row's sum meets.
template <bool F16>
static __device__ __forceinline__ uint32_t tree_odd16(uint32_t x) {
  return F16 ? ((x & 0x7c007c00u) + 0x04000400u) & 0x80008000u : ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}
static __device__ __forceinline__ uint32_t tree_odd8(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
template <bool F16>
static __device__ __forceinline__ uint32_t tree_even16(uint32_t x) { return x & ~((tree_odd16<F16>(x) >> 15) * 0xffffu); }
static __device__ __forceinline__ uint32_t tree_even8(uint32_t x) { return x & ~((tree_odd8(x) >> 7) * 0xffu); }
template <bool F16>
static __device__ __forceinline__ uint32_t tree_places(uint32_t w) {
  constexpr uint32_t one = F16 ? 0x3c00u : 0x3f80u, inf = F16 ? 0x7c00u : 0x7f80u, k64 = F16 ? 0x5400u : 0x4280u, k4096 = F16 ? 0x6c00u : 0x4580u;
  auto place = [](uint32_t x) { return (x & 0x7fffu) > inf ? k4096 : x == inf ? one : x == (inf | 0x8000u) ? k64 : 0u; };
  return place(w & 0xffffu) | place(w >> 16) << 16;
}
// four bits as ones
template <bool F16>
static __device__ __forceinline__ uint2 tree_sees(uint32_t b) {
  constexpr uint32_t one = F16 ? 0x3c00u : 0x3f80u;
  return make_uint2((b & 1u ? one : 0u) | (b & 2u ? one << 16 : 0u), (b & 4u ? one : 0u) | (b & 8u ? one << 16 : 0u));
}
static __device__ __forceinline__ float tree_odd_sum(float count) {
  const uint32_t n = (uint32_t)count;
  const float up = n & 63u ? INFINITY : 0.f, down = n >> 6 & 63u ? -INFINITY : 0.f;
  return n >> 12 ? __uint_as_float(0x7fc00000u) : up + down;
}

// SHARE: neighbouring wavefronts take other parts of the same tokens, whose lines then come from memory once and from the
// CU's cache for the others.  Where a request has fewer parts than there are wavefronts, `ways` of them share a part and take every
// `ways`-th tile each; what they have is joined in LDS (`join`).
template <int HD, int NT, int NQ, bool FP8, bool F16, bool SHARE>
static __device__ __forceinline__ void tree_segment(const TreeParams& p, const TreeSegment& s, int h, int lane, int way, int ways, float* join) {
  constexpr int KS = HD / 32, DV = HD / 16, ESZ = FP8 ? 1 : 2, TK = 16 * NT, ROWS = 16 * NQ;
  constexpr int KL = FP8 ? KS / 2 : KS;      // 16-byte loads of a key row and lane
  constexpr int VD = FP8 ? DV / 4 : DV / 2;  // dwords per token and lane of the value operand
  const int m16 = lane & 15, g = lane >> 4;
  const int r = __builtin_amdgcn_readfirstlane(s.r), len = __builtin_amdgcn_readfirstlane(s.len);
  const int start = __builtin_amdgcn_readfirstlane(s.start), end = __builtin_amdgcn_readfirstlane(s.end);
  const int ctx = __builtin_amdgcn_readfirstlane(s.ctx);
  h = __builtin_amdgcn_readfirstlane(h);
  const int last = max(min(end, len) - 1, 0);
  const int step = SHARE ? TK * ways : TK;
  if (SHARE && tree_div_g(p, s.part * ROWS) >= s.nodes) {   // (a part without rows)
    if (ways > 1) {
      __syncthreads();
      __syncthreads();
    }
    return;
  }

  // rows of this lane: row tile nt, row m16
  int q_row[NQ], q_head[NQ];
  bool valid[NQ];
  uint4 qf[NQ][KS];
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    const int n = s.part * ROWS + 16 * nt + m16, qi = tree_div_g(p, n);
    valid[nt] = qi < s.nodes;
    q_row[nt] = s.q_begin + (valid[nt] ? qi : 0);
    q_head[nt] = h * p.G + (n - qi * p.G);
    const uint16_t* row = p.q + (int64_t)q_row[nt] * p.q_st + (int64_t)q_head[nt] * p.q_sh;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) {
      const int d0 = FP8 ? 64 * (kk >> 1) + 16 * g + 8 * (kk & 1) : 32 * kk + 8 * g;  // (16 key bytes to a lane)
      qf[nt][kk] = valid[nt] ? ld16(row + d0) : make_uint4(0, 0, 0, 0);
    }
  }

  const uint8_t* const kbase = p.kc + (int64_t)h * p.kv_sh * ESZ;
  const uint8_t* const vbase = p.vc + (int64_t)h * p.kv_sh * ESZ;
  const int64_t chunk_bytes = p.kv_sc * ESZ;
  const uint32_t tok_bytes = (uint32_t)(p.kv_st * ESZ);
  const uint32_t k_col = 16u * (uint32_t)g, v_col = (uint32_t)(DV * m16 * ESZ);

  // Block-table cursor: the current chunk's entry and the next one's, the one after in flight (requested two chunks before
  // its use), an fp8 cache's scale one chunk ahead.  Table and scales lie in the constant address space: scalar loads, which
  // wait for no tile.  An entry that names no chunk of the cache becomes -1: its tokens are seen by no row, and their loads
  // go to chunk 0.
  const auto* const bt_row = tree_constant(p.bt + (int64_t)(p.r_base + r) * p.bt_stride);
  const int ci_last = tree_chunk_of(last, p.chunk_magic);
  struct Cursor {
    int ci, pc, pc_next, pc_after;
    float sc, sc_next;
  };
  auto entry_load = [&](int ci) { return bt_row[min(ci, ci_last)]; };
  auto entry = [&](int e) { return (uint32_t)e < (uint32_t)p.n_chunks ? e : -1; };
  auto scale_load = [&](const float* scales, int pc) { return tree_constant(scales)[(int64_t)max(pc, 0) * p.Hkv + h]; };
  auto follow = [&](Cursor& c, const float* scales, int ci) {
    if (ci != c.ci) {
      const bool far = SHARE && ci != c.ci + 1;   // (a step over several chunks)
      c.ci = ci;
      c.pc = far ? entry(entry_load(ci)) : c.pc_next;
      c.pc_next = entry(far ? entry_load(ci + 1) : c.pc_after);
      c.pc_after = entry_load(ci + 2);
      if (FP8) {
        c.sc = far ? scale_load(scales, c.pc) : c.sc_next;
        c.sc_next = scale_load(scales, c.pc_next);
      }
    }
  };
  const int begin = SHARE ? start + TK * way : start;
  Cursor kcur, vcur;
  {
    const int ci0 = tree_chunk_of(min(begin, last), p.chunk_magic);
    const int e0 = entry_load(ci0), e1 = entry_load(ci0 + 1), e2 = entry_load(ci0 + 2);
    kcur.ci = ci0;
    kcur.pc = entry(e0);
    kcur.pc_next = entry(e1);
    kcur.pc_after = e2;
    kcur.sc = kcur.sc_next = 1.f;
    vcur = kcur;
    if (FP8) {
      kcur.sc = scale_load(p.k_scale, kcur.pc);
      vcur.sc = scale_load(p.v_scale, kcur.pc);
      kcur.sc_next = scale_load(p.k_scale, kcur.pc_next);
      vcur.sc_next = scale_load(p.v_scale, kcur.pc_next);
    }
  }

  uint4 kf[NT][KL];
  uint32_t vf[NT][4][VD];
  float ksc = 1.f, vsc = 1.f;   // fp8: scales of the staged tiles' chunks
  bool k_page = true;           // whether the staged keys' chunk exists
  // Tiles are read through buffer descriptors that end behind the request's last token: what lies behind arrives as zeros,
  // and so does all of a chunk that the table does not name (its tokens are seen by no row).
  constexpr int kPolicy = SHARE ? 0 : 2;   // (read once they stream past the caches)
  const int k_lane = m16 * tok_bytes + 16 * g;
  int v_lane[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) v_lane[j] = (4 * g + j) * tok_bytes + DV * m16 * ESZ;
  auto tile_of = [&](Cursor& c, const float* scales, const uint8_t* base, int T) {
    const int t0 = min(T, last), ci = tree_chunk_of(t0, p.chunk_magic);
    follow(c, scales, ci);
    const uint32_t left = c.pc < 0 || T > last ? 0u : (uint32_t)min(len - T, TK);
    const uint8_t* at = base + (int64_t)max(c.pc, 0) * chunk_bytes + (int64_t)(t0 - ci * p.chunk) * tok_bytes;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(at), 0, (int)(left ? (left - 1) * (uint32_t)tok_bytes + HD * ESZ : 0u), 0x00020000);
  };
  auto load_k = [&](int T) {
    const auto rs = tile_of(kcur, p.k_scale, kbase, T);
    if (FP8) ksc = kcur.sc;
    k_page = kcur.pc >= 0;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int kk = 0; kk < KL; ++kk)
        kf[u][kk] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(rs, k_lane + 64 * kk, 16 * u * tok_bytes, kPolicy));
  };
  auto load_v = [&](int T) {
    const auto rs = tile_of(vcur, p.v_scale, vbase, T);
    if (FP8) vsc = vcur.sc;
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int soff = 16 * u * tok_bytes;
        if constexpr (VD == 1) {
          vf[u][j][0] = __builtin_amdgcn_raw_buffer_load_b32(rs, v_lane[j], soff, kPolicy);
        } else if constexpr (VD == 3) {
          const auto x = __builtin_amdgcn_raw_buffer_load_b96(rs, v_lane[j], soff, kPolicy);
          vf[u][j][0] = x[0]; vf[u][j][1] = x[1]; vf[u][j][2] = x[2];
        } else {
#pragma unroll
          for (int w = 0; w + 4 <= VD; w += 4) {
            const auto x = __builtin_amdgcn_raw_buffer_load_b128(rs, v_lane[j] + 4 * w, soff, kPolicy);
            vf[u][j][w] = x[0]; vf[u][j][w + 1] = x[1]; vf[u][j][w + 2] = x[2]; vf[u][j][w + 3] = x[3];
          }
          if constexpr (VD % 4 == 2) {
            const auto x = __builtin_amdgcn_raw_buffer_load_b64(rs, v_lane[j] + 4 * (VD - 2), soff, kPolicy);
            vf[u][j][VD - 2] = x[0]; vf[u][j][VD - 1] = x[1];
          }
        }
      }
  };

  // The running maximum starts at a finite lowest value: a row that sees nothing keeps it and a sum of zero.
  float m_run[NQ], l_run[NQ];
  f32x4_t acc[NQ][DV];
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    m_run[nt] = -3e38f;
    l_run[nt] = 0.f;
#pragma unroll
    for (int e = 0; e < DV; ++e) acc[nt][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // fp8: the accumulators are in units of the current value scale (a change of chunk rescales them), so that the
  // probabilities keep their own range: times a small scale they would be subnormal in fp16.
  float unit = 1.f;
  const uint2 ones = make_uint2(ones2<F16>(), ones2<F16>());
  const f32x4_t zero4 = {0.f, 0.f, 0.f, 0.f};

  if (start < end) {
    load_k(begin);
    load_v(begin);
  }
  for (int T = begin; T < end; T += step) {
    // ---- S^T = K Q^T
    const float mul = FP8 ? p.scale_log2 * ksc : p.scale_log2;
    const bool masked = T + TK > min(ctx, end) || !k_page;   // wave-uniform
    const bool page = k_page;
    f32x4_t sc[NQ][NT];
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
      for (int u = 0; u < NT; ++u) sc[nt][u] = zero4;
#pragma unroll
    for (int u = 0; u < NT; ++u) {
#pragma unroll
      for (int kk = 0; kk < KL; ++kk) {
        if constexpr (FP8) {
          const uint2 a0 = fp8x4_to_16x4<F16>(kf[u][kk].x), a1 = fp8x4_to_16x4<F16>(kf[u][kk].y);
          const uint2 b0 = fp8x4_to_16x4<F16>(kf[u][kk].z), b1 = fp8x4_to_16x4<F16>(kf[u][kk].w);
#pragma unroll
          for (int nt = 0; nt < NQ; ++nt) {
            sc[nt][u] = mfma_16x16x32<F16>(make_uint4(a0.x, a0.y, a1.x, a1.y), qf[nt][2 * kk], sc[nt][u]);
            sc[nt][u] = mfma_16x16x32<F16>(make_uint4(b0.x, b0.y, b1.x, b1.y), qf[nt][2 * kk + 1], sc[nt][u]);
          }
        } else {
#pragma unroll
          for (int nt = 0; nt < NQ; ++nt) sc[nt][u] = mfma_16x16x32<F16>(kf[u][kk], qf[nt][kk], sc[nt][u]);
        }
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (!SHARE && !((T - begin) & (8 * TK - 1))) __builtin_amdgcn_s_barrier();
    load_k(T + step);   // (the key registers are free again)
    __builtin_amdgcn_sched_barrier(0);
    if (FP8) {        // a scale may have any sign: the maximum is of the products' own scores
#pragma unroll
      for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][u][i] *= mul;
    }
    uint32_t seen[NQ];   // four bits per sub-tile: what this lane's row sees of its four tokens (masked tiles only)
    if (masked) {
#pragma unroll
      for (int nt = 0; nt < NQ; ++nt) {
        const uint32_t* bits = p.mask + (int64_t)q_row[nt] * p.mask_st;
        seen[nt] = 0;
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          const int t0 = T + 16 * u + 4 * g;
          uint32_t b = page ? tree_bits(bits, p.mask_words, t0 - ctx) & 15u : 0u;
          const int left = end - t0;
          b &= left >= 4 ? 15u : left > 0 ? (1u << left) - 1u : 0u;
          seen[nt] |= b << (4 * u);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(b >> i & 1u)) sc[nt][u][i] = -INFINITY;
        }
      }
    }
    // ---- running maximum and sum (row m16; only the maximum crosses lanes, the sums come from the matrix cores)
    const float pm = FP8 ? 1.f : mul;
    uint2 pf[NQ][NT];
    // (values of a chunk whose scale is zero weigh nothing; the unit stays, since no sum fits one that small)
    const bool weigh = !FP8 || !(fabsf(vsc) < 1e-30f);
    const float unit_new = FP8 && page && weigh ? vsc : unit;
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
      float tmax = -INFINITY;
#pragma unroll
      for (int u = 0; u < NT; ++u) tmax = fmaxf(fmaxf(tmax, fmaxf(sc[nt][u][0], sc[nt][u][1])), fmaxf(sc[nt][u][2], sc[nt][u][3]));
      const float m_new = fmaxf(m_run[nt], rowgroup_max(tmax) * pm);
      const float alpha = fast_exp2(m_run[nt] - m_new);
      m_run[nt] = m_new;
      const float neg = kTreeLift<F16> - m_new;
      f32x4_t sum = zero4;
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const float p0 = fast_exp2(__builtin_fmaf(sc[nt][u][0], pm, neg)), p1 = fast_exp2(__builtin_fmaf(sc[nt][u][1], pm, neg));
        const float p2 = fast_exp2(__builtin_fmaf(sc[nt][u][2], pm, neg)), p3 = fast_exp2(__builtin_fmaf(sc[nt][u][3], pm, neg));
        pf[nt][u] = make_uint2(pack2<F16>(p0, p1), pack2<F16>(p2, p3));
        sum = mfma_16x16x16<F16>(ones, pf[nt][u], sum);
        if (FP8 && !weigh) pf[nt][u] = make_uint2(0, 0);
      }
      l_run[nt] = l_run[nt] * alpha + sum[0];
      const float scale = FP8 ? alpha * (unit / unit_new) : alpha;
      if (__builtin_amdgcn_ballot_w64(scale != 1.f)) {
#pragma unroll
        for (int e = 0; e < DV; ++e) {
          acc[nt][e][0] *= scale; acc[nt][e][1] *= scale; acc[nt][e][2] *= scale; acc[nt][e][3] *= scale;
        }
      }
    }
    unit = unit_new;
    // ---- O^T += V^T P^T
    // value operands of sub-tile u: output column e of every four tokens, one half of a depth-32 product
    auto column = [&](int u, int e) -> uint2 {
      uint32_t x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (FP8) {
          const uint2 w = fp8x4_to_16x4<F16>(vf[u][j][e >> 2]);
          x[j] = (e >> 1) & 1 ? w.y : w.x;
        } else {
          x[j] = vf[u][j][e >> 1];
        }
      }
      return (e & 1) ? make_uint2(high_halves(x[1], x[0]), high_halves(x[3], x[2]))
                     : make_uint2(low_halves(x[1], x[0]), low_halves(x[3], x[2]));
    };
    if (masked) {
      // Infinities and NaN: a product would take them into rows that do not see their token.  Their places times what the
      // rows see say which sums they belong to; then they are zeros.
      auto odd = [](uint32_t x) { return FP8 ? tree_odd8(x) : tree_odd16<F16>(x); };
      uint32_t any = 0;
#pragma unroll
      for (int u = 0; u < NT; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int w = 0; w < VD; ++w) any |= odd(vf[u][j][w]);
      if (__builtin_amdgcn_ballot_w64(any != 0)) {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
#pragma unroll
          for (int e = 0; e < DV; ++e) {
            __builtin_amdgcn_sched_barrier(0);   // (one column at a time: registers)
            const uint2 c = column(u, e), at = make_uint2(tree_places<F16>(c.x), tree_places<F16>(c.y));
#pragma unroll
            for (int nt = 0; nt < NQ; ++nt) {
              const f32x4_t n = mfma_16x16x16<F16>(at, tree_sees<F16>(seen[nt] >> (4 * u)), zero4);
#pragma unroll
              for (int i = 0; i < 4; ++i) acc[nt][e][i] += tree_odd_sum(n[i]);
            }
          }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int w = 0; w < VD; ++w) vf[u][j][w] = FP8 ? tree_even8(vf[u][j][w]) : tree_even16<F16>(vf[u][j][w]);
      }
    }
#pragma unroll
    for (int u = 0; u < NT; u += NT >= 2 ? 2 : 1)
#pragma unroll
      for (int e = 0; e < DV; ++e) {
        if constexpr (NT >= 2) {
          const uint2 a = column(u, e), b = column(u + 1, e);
#pragma unroll
          for (int nt = 0; nt < NQ; ++nt)
            acc[nt][e] = mfma_16x16x32<F16>(make_uint4(a.x, a.y, b.x, b.y),
                                            make_uint4(pf[nt][u].x, pf[nt][u].y, pf[nt][u + 1].x, pf[nt][u + 1].y), acc[nt][e]);
        } else {
          const uint2 a = column(u, e);
#pragma unroll
          for (int nt = 0; nt < NQ; ++nt) acc[nt][e] = mfma_16x16x16<F16>(a, pf[nt][u], acc[nt][e]);
        }
      }
    __builtin_amdgcn_sched_barrier(0);
    load_v(T + step);
    __builtin_amdgcn_sched_barrier(0);
  }

  if (SHARE && ways > 1) {
    // a register of all lanes after the other: the accumulators, the maximum and the sum of every row tile
    constexpr int WORDS = NQ * (4 * DV + 2);
    if (way) {
      float* at = join + lane;
#pragma unroll
      for (int nt = 0; nt < NQ; ++nt) {
#pragma unroll
        for (int e = 0; e < DV; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) at[64 * ((nt * DV + e) * 4 + i)] = acc[nt][e][i] * unit;
        at[64 * (4 * NQ * DV + 2 * nt)] = m_run[nt];
        at[64 * (4 * NQ * DV + 2 * nt + 1)] = l_run[nt];
      }
    }
    __syncthreads();
    if (!way) {
#pragma unroll
      for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
        for (int e = 0; e < DV; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][e][i] *= unit;
      unit = 1.f;
      for (int w = 1; w < ways; ++w) {
        const float* at = join + (size_t)w * 64 * WORDS + lane;
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt) {
          const float m2 = at[64 * (4 * NQ * DV + 2 * nt)], l2 = at[64 * (4 * NQ * DV + 2 * nt + 1)];
          const float m = fmaxf(m_run[nt], m2), a = fast_exp2(m_run[nt] - m), b = fast_exp2(m2 - m);
          m_run[nt] = m;
          l_run[nt] = l_run[nt] * a + l2 * b;
#pragma unroll
          for (int e = 0; e < DV; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[nt][e][i] = acc[nt][e][i] * a + at[64 * ((nt * DV + e) * 4 + i)] * b;
        }
      }
    }
    __syncthreads();   // (the next segment's may come)
    if (way) return;
  }
  // ---- acc[nt][e][i] is element d = DV (4g + i) + e of the row
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    if (!valid[nt]) continue;
    const float l = l_run[nt];
    const float inv = l == 0.f ? 0.f : unit / l;   // (a NaN stays one)
    if (s.whole) {
      uint16_t* o = p.out + (int64_t)q_row[nt] * p.o_st + (int64_t)q_head[nt] * p.o_sh + 4 * DV * g;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[DV / 2];
#pragma unroll
        for (int dw = 0; dw < DV / 2; ++dw) w[dw] = pack2<F16>(acc[nt][2 * dw][i] * inv, acc[nt][2 * dw + 1][i] * inv);
        st_dwords(o + DV * i, w);
      }
    } else {
      const int64_t row = ((int64_t)s.slot * p.Hkv + h) * p.rows + s.row0 + 16 * nt + m16;
      float* o = p.part_o + row * HD + 4 * DV * g;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < DV; e += 2)
          *reinterpret_cast<float2*>(o + DV * i + e) = make_float2(acc[nt][e][i] * inv, acc[nt][e + 1][i] * inv);
      if (g == 0) p.part_lse[row] = l == 0.f ? -INFINITY : m_run[nt] - kTreeLift<F16> + fast_log2(l);
    }
  }
}

// What one request brings: rows of q, nodes, cached tokens.  Whatever the arrays hold, rows stay inside q, no row belongs to two
// requests of a launch (cu_seqlens_q counts as its own running maximum: the number of groups has a place for each) and tokens stay
// inside the block table.
struct TreeRequest {
  int q_begin, nodes, len;
};
static __device__ __forceinline__ int tree_row(const TreeParams& p, int i) { return min(max(p.cu_q[i], 0), p.T); }
static __device__ __forceinline__ int tree_len(const TreeParams& p, int i) {
  return (int)min((int64_t)max(p.lens[i], 0), (int64_t)p.table_cols * p.chunk);
}
// Maximum of this lane's number and those of the lanes before it (none is negative).
static __device__ __forceinline__ int tree_scan_max(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return v;
}

// ------------------------------------------------------------------------------------------------ tiles through LDS
// For 16-bit caches of widths 64 and 128.  Where a request has many rows per KV head the products are the work, and a CU's cache too
// slow a feed; where it has few, calls that do not fill the memory are faster through LDS too (figures at the entry point's rule).  A
// workgroup of WAVES wavefronts takes 32 * WAVES rows of one (request, KV head), and tiles of 32 tokens go straight from memory into
// LDS (buffer loads with the LDS destination).  With eight stages a barrier serves two tiles, and up to six are ahead of the one at work,
// four of them on their way behind a barrier; with four (width 128, four wavefronts) a barrier serves one, two are ahead and one is on
// its way, 32 KB a CU where the register kernel has 64: in calls that fill the memory that one is faster.  The 16-byte pieces of a row lie
// in another order in every row (an exclusive or with the row's number, applied where the loads pick their source), which
// spreads the reads of 16 rows over all banks without padding; the order of a lane's own reads is an exclusive or again.
// Rows behind the request's last token arrive as zeros (the load's descriptor ends there).  With many rows it is bound by the matrix
// cores and LDS reads, which take about as long: 3 trees of 64 nodes and 64 heads of 128 over 40 000-60 000 tokens 358 us, 887 TFLOP/s;
// 16 trees of 25-61 nodes, 32 heads, 111 us (a third of the 256 rows is empty); with few by memory: 64 chains of 6 nodes over 512-8 192
// tokens 211 us, 5.3 TB/s, and 8.7 us for one of 777 tokens.  A tile's scores beside the exponentials of the tile before it, a barrier per
// two tiles and references that move seldom are what the former gained most by.
template <int HD> static __device__ __forceinline__ int tree_swizzle(int row) { return HD == 64 ? (row >> 1) & 7 : row & 15; }
template <int HD, int WAVES> constexpr int tree_stages() {
  constexpr int room = WAVES == 8 ? 131072 : 65536;   // LDS of a workgroup: one or two of them on a CU
  return room / (HD * 128) > 8 ? 8 : room / (HD * 128);
}

template <int HD, int WAVES, bool F16>
static __device__ __forceinline__ void tree_rows_segment(const TreeParams& p, const TreeSegment& s, int h, int lane, int wave, uint8_t* lds) {
  constexpr int KS = HD / 32, DV = HD / 16, NQ = 2, TK = 32, ROWB = 2 * HD, STAGES = tree_stages<HD, WAVES>();
  constexpr int HALF = TK * ROWB, STAGE = 2 * HALF;           // keys, then values
  constexpr int KLOADS = HALF / 1024, LPW = 2 * KLOADS / WAVES;
  static_assert(LPW * WAVES == 2 * KLOADS && (KLOADS % LPW == 0 || LPW % KLOADS == 0), "whole loads per wavefront");
  const int m16 = lane & 15, g = lane >> 4;
  const int len = __builtin_amdgcn_readfirstlane(s.len), ctx = __builtin_amdgcn_readfirstlane(s.ctx);
  const int start = __builtin_amdgcn_readfirstlane(s.start), end = __builtin_amdgcn_readfirstlane(s.end);

  int q_row[NQ], q_head[NQ];
  bool valid[NQ];
  uint4 qf[NQ][KS];
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    const int n = s.part * 32 + 16 * nt + m16, qi = tree_div_g(p, n);
    valid[nt] = qi < s.nodes;
    q_row[nt] = s.q_begin + (valid[nt] ? qi : 0);
    q_head[nt] = h * p.G + (n - qi * p.G);
    const uint16_t* row = p.q + (int64_t)q_row[nt] * p.q_st + (int64_t)q_head[nt] * p.q_sh;
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) qf[nt][kk] = valid[nt] ? ld16(row + 32 * kk + 8 * g) : make_uint4(0, 0, 0, 0);
  }
  const bool idle = tree_div_g(p, s.part * 32) >= s.nodes;   // (a part without rows: loads and barriers only)

  auto uniform64 = [](uint64_t x) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) | (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
  };
  const uint64_t kbase = uniform64((uint64_t)(uintptr_t)(p.kc + (int64_t)h * p.kv_sh * 2)) & 0xffffffffffffull;
  const uint64_t vbase = uniform64((uint64_t)(uintptr_t)(p.vc + (int64_t)h * p.kv_sh * 2)) & 0xffffffffffffull;
  const int64_t chunk_bytes = p.kv_sc * 2;
  const int tok_bytes = p.kv_st * 2;
  const auto* const bt_row = tree_constant(p.bt + (int64_t)(p.r_base + s.r) * p.bt_stride);   // (scalar loads leave the count of the direct loads alone)
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;

  // this wavefront's loads of a tile: which piece of which row each lane fetches
  uint32_t src[LPW];
#pragma unroll
  for (int i = 0; i < LPW; ++i) {
    const int slot = ((wave * LPW + i) % KLOADS) * 64 + lane, row = slot / (HD / 8), piece = slot % (HD / 8);
    src[i] = (uint32_t)row * (uint32_t)tok_bytes + 16u * (uint32_t)(piece ^ tree_swizzle<HD>(row));
  }
  // The next tile to load: its chunk's entry, the next chunk's (requested a chunk ahead), its place in the chunk.  Past the
  // segment's last tile the loads fetch nothing (zeros), and so they do in a chunk that does not exist.
  const int tiles_end = (end + TK - 1) / TK, chunk_tiles = p.chunk / TK, tile_bytes = TK * tok_bytes;
  const int ci_last = tree_chunk_of(max(end - 1, 0), p.chunk_magic);
  int i_tile = start / TK, i_ci = tree_chunk_of(start, p.chunk_magic), i_in = i_tile - i_ci * chunk_tiles, i_stage = 0;
  int pc = bt_row[min(i_ci, ci_last)], pc_next = bt_row[min(i_ci + 1, ci_last)];
  uint32_t missing = 0;   // bit of a tile in flight (its number modulo 32): its chunk does not exist
  auto issue = [&] {
    const bool there = (uint32_t)pc < (uint32_t)p.n_chunks;
    const int64_t off = (int64_t)(there ? pc : 0) * chunk_bytes + i_in * tile_bytes;
    const uint32_t nrec = there && i_tile < tiles_end ? (uint32_t)(min(len - i_tile * TK, TK) - 1) * (uint32_t)tok_bytes + HD * 2 : 0u;
    const uint32_t bit = 1u << (i_tile & 31);
    missing = there ? missing & ~bit : missing | bit;
#pragma unroll
    for (int i = 0; i < LPW; ++i) {
      const int k = wave * LPW + i;
      const uint64_t a = (k < KLOADS ? kbase : vbase) + (uint64_t)off;
      u32x4_t rs;
      rs.x = (uint32_t)a;
      rs.y = (uint32_t)(a >> 32);
      rs.z = nrec;
      rs.w = 0x00020000u;
      const uint32_t m0 = lds0 + (uint32_t)(i_stage * STAGE + 1024 * k);
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(m0), "v"(src[i]), "s"(rs)
                   : "memory", "m0");
    }
    i_stage = i_stage + 1 == STAGES ? 0 : i_stage + 1;
    ++i_tile;
    if (++i_in == chunk_tiles) {
      i_in = 0;
      ++i_ci;
      pc = pc_next;
      pc_next = bt_row[min(i_ci + 1, ci_last)];
    }
  };

  // Softmax: exponentials are taken against a reference per row, which moves only when a probability leaves a window: with
  // bf16 the row's largest goes to 2^-30 when it moves, and 2 is the limit (the exponent's highest bit, looked at in the packed
  // words: 5 instructions where the maximum of the scores takes 20); with fp16 to 2^10 (kTreeLift), and 2^15 is the limit (the
  // largest of the packed words).  Row sums come from the matrix cores.
  constexpr float kHeadroom = F16 ? -kTreeLift<F16> : 30.f, kNoReference = 3e38f;   // (none: any score leaves the window, -inf stays 0)
  float neg[NQ];   // a probability is 2^(score * scale + neg)
  f32x4_t acc[NQ][DV], sum[NQ];
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    neg[nt] = kNoReference;
    sum[nt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < DV; ++e) acc[nt][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  const f32x4_t zero4 = {0.f, 0.f, 0.f, 0.f};
  const uint4 ones = make_uint4(ones2<F16>(), ones2<F16>(), ones2<F16>(), ones2<F16>());
  // this lane's first key piece and value piece within a stage; step kk: ^ 64 kk, column e: ^ 32 e, sub-tile 1: + 16 rows
  const uint32_t k_at = (uint32_t)(m16 * ROWB + ((g ^ tree_swizzle<HD>(m16)) << 4));
  const int v_row = 4 * g + (m16 >> 2);
  const uint32_t v_at = (uint32_t)(HALF + v_row * ROWB + ((((m16 >> 1) & 1) ^ tree_swizzle<HD>(v_row)) << 4) + 8 * (m16 & 1));

  // Probabilities of two scores (of a tile's eight per row tile and lane): chunk c is row tile c >> 2, sub-tile c >> 1 & 1.
  auto chunk = [&](const f32x4_t (&S)[NQ][2], uint4 (&P)[NQ], int c) {
    const int nt = c >> 2, u = c >> 1 & 1, i = 2 * (c & 1);
    const uint32_t w = pack2<F16>(fast_exp2(__builtin_fmaf(S[nt][u][i], p.scale_log2, neg[nt])),
                                  fast_exp2(__builtin_fmaf(S[nt][u][i + 1], p.scale_log2, neg[nt])));
    const int d = c & 3;
    if (d == 0) P[nt].x = w; else if (d == 1) P[nt].y = w; else if (d == 2) P[nt].z = w; else P[nt].w = w;
  };
  // The same in three stages -- scale and subtract, exponential, pack -- of three chunks at a time, so that no instruction
  // waits for the one before it: at position n stage one of chunk n, two of chunk n - 1, three of chunk n - 2.
  float xs[2][2], ps[2][2];   // of chunks n, n - 1
  auto stages = [&](const f32x4_t (&S)[NQ][2], uint4 (&P)[NQ], int n) {
    if (n >= 2 && n < 10) {
      const int c = n - 2, nt = c >> 2, d = c & 3;
      const uint32_t w = pack2<F16>(ps[c & 1][0], ps[c & 1][1]);
      if (d == 0) P[nt].x = w; else if (d == 1) P[nt].y = w; else if (d == 2) P[nt].z = w; else P[nt].w = w;
    }
    if (n >= 1 && n < 9) {
      ps[(n - 1) & 1][0] = fast_exp2(xs[(n - 1) & 1][0]);
      ps[(n - 1) & 1][1] = fast_exp2(xs[(n - 1) & 1][1]);
    }
    if (n < 8) {
      const int nt = n >> 2, u = n >> 1 & 1, i = 2 * (n & 1);
      xs[n & 1][0] = __builtin_fmaf(S[nt][u][i], p.scale_log2, neg[nt]);
      xs[n & 1][1] = __builtin_fmaf(S[nt][u][i + 1], p.scale_log2, neg[nt]);
    }
  };
  auto leaves_window = [&](const uint4 (&P)[NQ]) {
    if constexpr (F16) {
      uint32_t t;
      asm("v_pk_maximum3_f16 %0, %1, %2, %3" : "=v"(t) : "v"(P[0].x), "v"(P[0].y), "v"(P[0].z));
      asm("v_pk_maximum3_f16 %0, %0, %1, %2" : "+v"(t) : "v"(P[0].w), "v"(P[1].x));
      asm("v_pk_maximum3_f16 %0, %0, %1, %2" : "+v"(t) : "v"(P[1].y), "v"(P[1].z));
      asm("v_pk_maximum3_f16 %0, %0, %1, %1" : "+v"(t) : "v"(P[1].w));
      asm("v_pk_add_u16 %0, %0, %1" : "+v"(t) : "v"(0x08000800u));   // (0x7800, 2^15, becomes the sign; infinity and NaN too)
      return __builtin_amdgcn_ballot_w64((t & 0x80008000u) != 0) != 0;
    } else {
      const uint32_t any = (P[0].x | P[0].y | P[0].z | P[0].w) | (P[1].x | P[1].y | P[1].z | P[1].w);
      return __builtin_amdgcn_ballot_w64((any & 0x40004000u) != 0) != 0;
    }
  };
  auto move_reference = [&](const f32x4_t (&S)[NQ][2], uint4 (&P)[NQ]) {
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
      float top = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, S[nt][i >> 2][i & 3]);
      const float to = fminf(neg[nt], __builtin_fmaf(-rowgroup_max(top), p.scale_log2, -kHeadroom));
      const float alpha = fast_exp2(to - neg[nt]);
      neg[nt] = to;
#pragma unroll
      for (int e = 0; e < DV; ++e) {
        acc[nt][e][0] *= alpha; acc[nt][e][1] *= alpha; acc[nt][e][2] *= alpha; acc[nt][e][3] *= alpha;
      }
      sum[nt][0] *= alpha; sum[nt][1] *= alpha; sum[nt][2] *= alpha; sum[nt][3] *= alpha;
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) chunk(S, P, c);
  };
  auto key_piece = [&](const uint8_t* at, int n) {   // sub-tile n & 1, step n >> 1
    return *reinterpret_cast<const uint4*>(at + (k_at ^ (64u * (n >> 1))) + 16 * (n & 1) * ROWB);
  };
  auto value_piece = [&](const uint8_t* at, int e) {
    const uint8_t* v = at + (v_at ^ (32u * e));
    const uint2 a = lds_ld8_tr(v), b = lds_ld8_tr(v + 16 * ROWB);
    return make_uint4(a.x, a.y, b.x, b.y);
  };
  // One column of O^T += V^T P^T.  ODD: its values may be infinities or NaN that not every row sees (`seen`).
  auto column = [&](auto Oc, int e, uint4 v, const uint4 (&P)[NQ], const uint32_t (&seen)[NQ]) {
    if constexpr (decltype(Oc)::value) {
      if (__builtin_amdgcn_ballot_w64((tree_odd16<F16>(v.x) | tree_odd16<F16>(v.y) | tree_odd16<F16>(v.z) | tree_odd16<F16>(v.w)) != 0)) {
        const uint2 lo = make_uint2(tree_places<F16>(v.x), tree_places<F16>(v.y)), hi = make_uint2(tree_places<F16>(v.z), tree_places<F16>(v.w));
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt) {
          const f32x4_t n = mfma_16x16x16<F16>(hi, tree_sees<F16>(seen[nt] >> 4), mfma_16x16x16<F16>(lo, tree_sees<F16>(seen[nt]), zero4));
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][e][i] += tree_odd_sum(n[i]);
        }
        v = make_uint4(tree_even16<F16>(v.x), tree_even16<F16>(v.y), tree_even16<F16>(v.z), tree_even16<F16>(v.w));
      }
    }
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) acc[nt][e] = mfma_16x16x32<F16>(v, P[nt], acc[nt][e]);
  };
  // This wavefront's share of the next tile (PAIRS: the next two) has landed (what it issued after that may be on its way),
  // then everyone's; the tiles two (and three) back are read by nobody any more, and their places are filled.
  constexpr bool PAIRS = STAGES == 8;
  constexpr int FIRST = PAIRS ? STAGES - 3 : STAGES - 2;   // tiles that set out at the start
  auto turn = [&] {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((PAIRS ? STAGES - 6 : STAGES - 4) * LPW) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    issue();
    if (PAIRS) issue();
  };
#define MI_SB() __builtin_amdgcn_sched_barrier(0)

  // (the queries have arrived before any direct load: the compiler waits for them here and not among those)
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
    for (int kk = 0; kk < KS; ++kk) asm volatile("" ::"v"(qf[nt][kk].x), "v"(qf[nt][kk].y), "v"(qf[nt][kk].z), "v"(qf[nt][kk].w));
  __syncthreads();   // (the stages are free: every wavefront has left the segment before)
  if (start < end) {
    // (the values "before the first tile" are zeros: their probabilities are, and zero times a stale value must not be NaN)
    for (int i = lane * 16; i < HALF; i += 1024) *reinterpret_cast<uint4*>(lds + (STAGES - 1) * STAGE + HALF + i) = make_uint4(0, 0, 0, 0);
    for (int i = 0; i < FIRST; ++i) issue();
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((FIRST - 1) * LPW) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  }
  if (idle) {   // (a part without rows)
    for (int T = start; T < end; T += PAIRS ? 2 * TK : TK) turn();
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    return;
  }
  if (start < end) {
    // The stream of a tile: its scores, piece by piece, beside the probabilities of the tile before; then the values of that
    // one.  Pieces come from LDS three ahead of their products, across the barrier and from tile to tile.
    constexpr int NK = 2 * KS, RING = 4, AHEAD = RING - 1;
    static_assert((NK + DV) % RING == 0 && 8 % NK == 0, "the next tile's first pieces follow the last column");
    uint4 fr[RING], P[NQ];
    uint32_t seen[NQ];
    f32x4_t S[NQ][2], Sn[NQ][2];
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) {
      P[nt] = make_uint4(0, 0, 0, 0);
      seen[nt] = 255u;
#pragma unroll
      for (int u = 0; u < 2; ++u) S[nt][u] = f32x4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    }
    int T = start, stage = 0, before = STAGES - 1;
    bool odd_tile = false;
    uint4 Pnone[NQ];   // (stages 0 and 1 pack nothing)
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) fr[n] = key_piece(lds, n);
    stages(S, Pnone, 0);
    stages(S, Pnone, 1);
    auto step = [&](auto Mc) {
      constexpr bool MASK = decltype(Mc)::value;
      const int next = stage + 1 == STAGES ? 0 : stage + 1;
      const uint8_t* const at_k = lds + stage * STAGE;
      const uint8_t* const at_v = lds + before * STAGE;
      const uint8_t* const at_next = lds + next * STAGE;
      auto request = [&](int n) {
        fr[n % RING] = n < NK ? key_piece(at_k, n) : n < NK + DV ? value_piece(at_v, n - NK) : key_piece(at_next, n - NK - DV);
      };
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        request(n + AHEAD);
        MI_SB();
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt) Sn[nt][n & 1] = mfma_16x16x32<F16>(fr[n % RING], qf[nt][n >> 1], n >> 1 ? Sn[nt][n & 1] : zero4);
        MI_SB();
#pragma unroll
        for (int i = 8 / NK * n; i < 8 / NK * (n + 1); ++i) stages(S, P, i + 2);   // (0 and 1 beside the last columns before)
        MI_SB();
      }
      if (leaves_window(P)) move_reference(S, P);
      if (!PAIRS || !odd_tile) turn();
      // what no row of this tile's scores may count
      const bool page = !(missing >> ((T / TK) & 31) & 1u);
      uint32_t sees[NQ];
      if constexpr (MASK) {
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt) {
          const uint32_t* bits = p.mask + (int64_t)q_row[nt] * p.mask_st;
          sees[nt] = 0;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int t0 = T + 16 * u + 4 * g;
            uint32_t b = page ? tree_bits(bits, p.mask_words, t0 - ctx) & 15u : 0u;
            const int left = end - t0;
            b &= left >= 4 ? 15u : left > 0 ? (1u << left) - 1u : 0u;
            sees[nt] |= b << (4 * u);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!(b >> i & 1u)) Sn[nt][u][i] = -INFINITY;
          }
        }
      } else if (!page) {
#pragma unroll
        for (int nt = 0; nt < NQ; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) Sn[nt][u] = f32x4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
      }
#pragma unroll
      for (int e = 0; e < DV; ++e) {
        request(NK + e + AHEAD);
        MI_SB();
        column(Mc, e, fr[(NK + e) % RING], P, seen);
        MI_SB();
        if (e >= DV - 2) stages(Sn, Pnone, e - (DV - 2));
        MI_SB();
      }
#pragma unroll
      for (int nt = 0; nt < NQ; ++nt) {
        sum[nt] = mfma_16x16x32<F16>(ones, P[nt], sum[nt]);
#pragma unroll
        for (int u = 0; u < 2; ++u) S[nt][u] = Sn[nt][u];
        if (MASK) seen[nt] = sees[nt];
      }
      odd_tile = !odd_tile;
      before = stage;
      stage = next;
      T += TK;
    };
    const int open = min(ctx, end);   // every row sees the tokens before
    while (T + TK <= open) step(std::false_type{});
    while (T < end) step(std::true_type{});
#pragma unroll
    for (int n = 2; n < 10; ++n) stages(S, P, n);
    if (leaves_window(P)) move_reference(S, P);
#pragma unroll
    for (int e = 0; e < DV; ++e) {
      MI_SB();   // (one column at a time: registers)
      column(std::true_type{}, e, value_piece(lds + before * STAGE, e), P, seen);
    }
#pragma unroll
    for (int nt = 0; nt < NQ; ++nt) sum[nt] = mfma_16x16x32<F16>(ones, P[nt], sum[nt]);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no load may still be on its way into this workgroup's LDS)
  }
#undef MI_SB

  // ---- acc[nt][e][i] is element d = 16 e + 4 g + i of the row
#pragma unroll
  for (int nt = 0; nt < NQ; ++nt) {
    if (!valid[nt]) continue;
    const float l = sum[nt][0], inv = l == 0.f ? 0.f : 1.f / l;
    if (s.whole) {
      uint16_t* o = p.out + (int64_t)q_row[nt] * p.o_st + (int64_t)q_head[nt] * p.o_sh + 4 * g;
#pragma unroll
      for (int e = 0; e < DV; ++e)
        st8(o + 16 * e, make_uint2(pack2<F16>(acc[nt][e][0] * inv, acc[nt][e][1] * inv), pack2<F16>(acc[nt][e][2] * inv, acc[nt][e][3] * inv)));
    } else {
      const int64_t row = ((int64_t)s.slot * p.Hkv + h) * p.rows + s.row0 + 16 * nt + m16;
      float* o = p.part_o + row * HD + 4 * g;
#pragma unroll
      for (int e = 0; e < DV; ++e)
        *reinterpret_cast<float4*>(o + 16 * e) = make_float4(acc[nt][e][0] * inv, acc[nt][e][1] * inv, acc[nt][e][2] * inv, acc[nt][e][3] * inv);
      if (g == 0) p.part_lse[row] = l == 0.f ? -INFINITY : fast_log2(l) - neg[nt];
    }
  }
}

// The span of this workgroup along the tiles of all (request, group) pairs, as segments one after the other: seg(segment);
// every wavefront walks the same ones.  Up to 64 requests lie in the lanes of every wavefront (no LDS, no barrier), more in
// dynamic LDS: tiles and groups of requests 0 .. i, and where the rows of request i end.  (The entry point has made sure that all tiles together are an int.)
// Clears the rows behind the last request on the way.
constexpr int kTreeStart = 1;   // what a pair's start counts, in tiles
template <int HD, int TK, typename Seg>
static __device__ __forceinline__ void tree_walk(const TreeParams& p, Seg seg) {
  extern __shared__ int32_t tree_lds[];
  int32_t* const cum = tree_lds;
  int32_t* const first = cum + p.R;
  int32_t* const row_end = first + p.R;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const bool in_lanes = p.R <= 64;

  TreeRequest mine{0, 0, 0};   // of request `lane` (in lanes)
  int cum_l = 0, first_l = 0;
  auto scan64 = [&](int base, int before) {   // `before`: where the rows of the requests before `base` end
    const int i = base + lane;
    int n_groups = 0, n_tiles = 0, from = 0, to = 0;
    if (i < p.R) {
      from = tree_row(p, i);
      to = tree_row(p, i + 1);
      mine.len = tree_len(p, i);
    }
    mine.q_begin = max(before, tree_scan_max(from));
    mine.nodes = max(mine.q_begin, tree_scan_max(to)) - mine.q_begin;
    if (i < p.R) {
      n_groups = (int)(((int64_t)mine.nodes * p.G + p.rows - 1) / p.rows);
      n_tiles = max((mine.len + TK - 1) / TK, 1);   // (a request without tokens has a tile in which nothing is seen)
    }
    cum_l = wave_scan(n_groups * n_tiles);
    first_l = wave_scan(n_groups);
  };
  if (in_lanes) {
    scan64(0, 0);
  } else {
    if (wave == 0) {
      int tiles = 0, groups = 0, rows = 0;
      for (int base = 0; base < p.R; base += 64) {
        scan64(base, rows);
        if (base + lane < p.R) {
          cum[base + lane] = tiles + cum_l;
          first[base + lane] = groups + first_l;
          row_end[base + lane] = mine.q_begin + mine.nodes;
        }
        rows = __builtin_amdgcn_readlane(mine.q_begin + mine.nodes, 63);
        tiles += __builtin_amdgcn_readlane(cum_l, 63);
        groups += __builtin_amdgcn_readlane(first_l, 63);
      }
    }
    __syncthreads();
  }
  auto cum_at = [&](int i) { return in_lanes ? __builtin_amdgcn_readlane(cum_l, i) : __builtin_amdgcn_readfirstlane(cum[i]); };
  auto first_at = [&](int i) { return in_lanes ? __builtin_amdgcn_readlane(first_l, i) : __builtin_amdgcn_readfirstlane(first[i]); };
  auto request_at = [&](int i) {
    if (!in_lanes) {
      const int begin = __builtin_amdgcn_readfirstlane(i ? row_end[i - 1] : tree_row(p, 0));
      return TreeRequest{begin, __builtin_amdgcn_readfirstlane(row_end[i]) - begin, tree_len(p, i)};
    }
    return TreeRequest{__builtin_amdgcn_readlane(mine.q_begin, i), __builtin_amdgcn_readlane(mine.nodes, i), __builtin_amdgcn_readlane(mine.len, i)};
  };
  const int total = cum_at(p.R - 1), pairs = first_at(p.R - 1);
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.pairs = pairs;

  // rows behind the last request are zeros
  if (p.last_slice) {
    const TreeRequest end = request_at(p.R - 1);
    const int tq = end.q_begin + end.nodes;
    if (tq < p.T) {
      const int64_t per_row = (int64_t)p.Hq * HD / 8, all = (int64_t)(p.T - tq) * per_row;
      const int64_t step = (int64_t)gridDim.x * gridDim.y * blockDim.x;
      for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x; i < all; i += step) {
        const int64_t row = i / per_row;
        const int e = (int)(i - row * per_row) * 8;
        st16(p.out + (tq + row) * p.o_st + (int64_t)(e / HD) * p.o_sh + e % HD, make_uint4(0, 0, 0, 0));
      }
    }
  }

  // The span: equal shares where the tiles fill the grid (a pair's start counts as one more: its queries, table entries and
  // first tile arrive one trip after the other), otherwise few tiles each -- a span's tiles follow one another, every further
  // span of a pair is one more partial to merge.
  if (total == 0) return;
  const int span = max(1, (int)rintf(__builtin_amdgcn_sqrtf(0.035f * (float)total * __builtin_amdgcn_rcpf((float)pairs))));
  const int extra = total / span >= p.grid ? kTreeStart : 0;
  int t0, t1;
  if (extra) {
    const int all = total + extra * pairs, per = all / p.grid, rem = all - per * p.grid;
    t0 = (int)blockIdx.x * per + min((int)blockIdx.x, rem);
    t1 = t0 + per + ((int)blockIdx.x < rem ? 1 : 0);
  } else {
    t0 = (int)blockIdx.x * span;
    t1 = min(t0 + span, total);
  }
  if (t0 >= t1) return;
  int r;   // the first request whose tiles reach beyond t0
  if (in_lanes) {
    r = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < p.R && cum_l + extra * first_l > t0));
  } else {
    int lo = 0, hi = p.R - 1;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (cum[mid] + extra * first[mid] > t0) hi = mid; else lo = mid + 1;
    }
    r = __builtin_amdgcn_readfirstlane(lo);
  }
  for (; t0 < t1; ++r) {
    const int rb = r ? cum_at(r - 1) + extra * first_at(r - 1) : 0, re = cum_at(r) + extra * first_at(r);
    if (t0 >= re) continue;
    const TreeRequest t = request_at(r);
    const int tiles = max((t.len + TK - 1) / TK, 1) + extra;
    TreeSegment s;
    s.r = r; s.q_begin = t.q_begin; s.nodes = t.nodes; s.len = t.len; s.ctx = t.len - t.nodes;
    while (t0 < t1 && t0 < re) {
      s.group = __builtin_amdgcn_readfirstlane((t0 - rb) / tiles);
      const int tb = t0 - rb - s.group * tiles, te = min(tiles, tb + (t1 - t0));
      if (te <= extra) {
        t0 += te - tb;
        continue;
      }
      const bool begins = tb <= extra, ends = te == tiles;
      s.start = max(tb - extra, 0) * TK;
      s.end = min((te - extra) * TK, t.len);
      s.whole = begins && ends;
      s.slot = 2 * blockIdx.x + (begins ? 1 : 0);
      // (read across the lanes while all of them are on: inside the branch a value that was put aside comes back for lane 0 only)
      const int pair = (r ? first_at(r - 1) : 0) + s.group;
      if (wave == 0 && lane == 0 && blockIdx.y == 0) {
        int4* info = p.pair_info + 2 * (int64_t)pair;
        if (begins) {
          info->x = blockIdx.x;
          info->z = s.group;
          info->w = s.q_begin;
          info[1].x = s.nodes;
        }
        if (ends) info->y = blockIdx.x;
      }
      seg(s);
      t0 += te - tb;
    }
  }
}

template <int HD, int NT, int NQ, bool FP8, bool F16, bool SHARE>
__global__ __launch_bounds__(512, 2) void paged_tree_kernel(TreeParams p) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int heads = (blockDim.x >> 6) / (SHARE ? p.share : 1);   // KV heads of the workgroup
  const int h = blockIdx.y * heads + (SHARE ? wave / p.share : wave), sub = SHARE ? wave % p.share : 0;
  if constexpr (SHARE) {
    // (the wavefronts' pieces of LDS: behind the walk's)
    extern __shared__ int32_t tree_lds[];
    float* const joins = reinterpret_cast<float*>(tree_lds + (p.R <= 64 ? 0 : 3 * p.R));
    tree_walk<HD, 16 * NT>(p, [&](TreeSegment& s) {
      // parts of this group, and how many wavefronts each has
      const int rows = min(s.nodes * p.G - s.group * p.rows, p.rows);
      int ways = p.share;
      while (ways > 1 && (p.share / ways) * 16 * NQ < rows) ways >>= 1;
      const int part = sub / ways, way = sub - part * ways;
      s.part = s.group * p.share + part;
      s.row0 = part * 16 * NQ;
      tree_segment<HD, NT, NQ, FP8, F16, true>(p, s, h, lane, way, ways, joins + (size_t)wave * 64 * NQ * (HD / 4 + 2));
    });
  } else {
    tree_walk<HD, 16 * NT>(p, [&](TreeSegment& s) {
      s.part = s.group;
      s.row0 = 0;
      tree_segment<HD, NT, NQ, FP8, F16, false>(p, s, h, lane, 0, 1, nullptr);
    });
  }
}

template <int HD, int WAVES, bool F16>
__global__ __launch_bounds__(64 * WAVES, 2) void paged_tree_rows_kernel(TreeParams p) {
  __shared__ __attribute__((aligned(1024))) uint8_t stages[tree_stages<HD, WAVES>() * HD * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  tree_walk<HD, 32>(p, [&](TreeSegment& s) {
    s.part = s.group * WAVES + wave;
    s.row0 = wave * 32;
    tree_rows_segment<HD, WAVES, F16>(p, s, blockIdx.y, lane, wave, stages);
  });
}

// Sum of a row's partials, weighted by 2^(lse - max): one workgroup per (request, group), KV head and eight rows or so.  A
// thread owns four neighbouring values of a row; `groups` sets of threads take its partials in turn, eight in flight each.
constexpr int kTreeMergeThreads = 256;
template <bool F16>
__global__ __launch_bounds__(1024) void paged_tree_merge_kernel(TreeParams p, int head_dim, int groups) {
  __shared__ float red[6][1024];
  const int pair = blockIdx.x, h = blockIdx.y;
  if (pair >= *p.pairs) return;
  const int4 info = p.pair_info[2 * pair];
  const int nodes = p.pair_info[2 * pair + 1].x;
  if (info.x == info.y) return;   // written by the streaming kernel
  const int cols = head_dim >> 2, block_rows = kTreeMergeThreads / cols, set = cols * block_rows;
  const int grp = threadIdx.x / set, in = threadIdx.x - grp * set;
  const int row = blockIdx.z * block_rows + in / cols, d = 4 * (in % cols);
  const int n = info.z * p.rows + row, qi = tree_div_g(p, n);
  if (tree_div_g(p, info.z * p.rows + blockIdx.z * block_rows) >= nodes) return;   // (uniform)
  const bool live = grp < groups && row < p.rows && qi < nodes;
  float mx = -INFINITY, den = 0.f;
  float4 num = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float lse, float weight, float4 v) {   // `weight` partials' worth of `v`, relative to 2^lse
    if (lse == -INFINITY) return;                       // (saw nothing)
    const float m = lse > mx || lse != lse ? lse : mx;  // (NaN goes on)
    const float a = fast_exp2(mx - m), b = fast_exp2(lse - m);
    num.x = num.x * a + b * v.x; num.y = num.y * a + b * v.y; num.z = num.z * a + b * v.z; num.w = num.w * a + b * v.w;
    den = den * a + b * weight;
    mx = m;
  };
  if (live)
    for (int w0 = info.x + 8 * grp; w0 <= info.y; w0 += 8 * groups) {
      float lse[8];
      float4 po[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int w = min(w0 + j, info.y);
        const int64_t at = ((int64_t)(2 * w + (w == info.x ? 1 : 0)) * p.Hkv + h) * p.rows + row;
        lse[j] = p.part_lse[at];
        po[j] = *reinterpret_cast<const float4*>(p.part_o + at * head_dim + d);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (w0 + j <= info.y) add(lse[j], 1.f, po[j]);
    }
  if (groups > 1) {
    const int i = threadIdx.x;
    red[0][i] = mx; red[1][i] = den; red[2][i] = num.x; red[3][i] = num.y; red[4][i] = num.z; red[5][i] = num.w;
    __syncthreads();
    if (grp) return;
    for (int g = 1; g < groups; ++g) {
      const int k = g * set + in;
      add(red[0][k], red[1][k], make_float4(red[2][k], red[3][k], red[4][k], red[5][k]));
    }
  }
  if (!live) return;
  const float inv = den == 0.f ? 0.f : 1.f / den;
  uint16_t* o = p.out + (int64_t)(info.w + qi) * p.o_st + (int64_t)(h * p.G + n - qi * p.G) * p.o_sh + d;
  st8(o, make_uint2(pack2<F16>(num.x * inv, num.y * inv), pack2<F16>(num.z * inv, num.w * inv)));
}

// Wavefronts per workgroup (`share` parts of a group times neighbouring KV heads), workgroups along the tiles, rows of a
// group.  Parts share where the average request has more rows than one takes: on average 32 rows of an fp8 cache (4 to 12
// nodes of 4 heads) took 455 us in parts of their own and 523 in shared ones, which read once and convert twice; 36 rows of a 16-bit
// cache in chunks of 48 69 us shared.  `many`: paged_tree_rows_kernel, four wavefronts (two workgroups on a CU) up to the 128 rows they
// take (16 requests of 4 096 tokens: 128 rows 75.5 us), eight beyond (132 rows 91.3, 256 rows 110.6).
struct TreeShape {
  int waves, share, grid, heads, rows;
};
static int64_t tree_mean_rows(int T, int R, int G) { return (int64_t)T * G / R; }
static TreeShape tree_shape(int T, int R, int Hq, int Hkv, int head_dim, bool many) {
  TreeShape s;
  const int64_t mean = tree_mean_rows(T, R, Hq / Hkv);
  if (many) {
    s.heads = 1;
    s.waves = s.share = mean <= 128 ? 4 : 8;
    s.grid = device_cu_count() * (s.waves == 8 ? 1 : 2) / Hkv;
    s.rows = 32 * s.waves;
  } else {
    const int rows = head_dim > 128 ? 16 : 32;
    s.share = mean <= rows ? 1 : mean <= 2 * rows ? 2 : mean <= 4 * rows ? 4 : 8;
    s.heads = 1;
    for (int w = 2; w <= 8 / s.share; ++w)
      if (Hkv % w == 0) s.heads = w;
    s.waves = s.heads * s.share;
    s.grid = device_cu_count() * (8 / s.waves) / (Hkv / s.heads);
    s.rows = rows * s.share;
  }
  if (s.grid < 1) s.grid = 1;
  return s;
}
// More than the default 64 KB of dynamic LDS, once per kernel and device.
template <void (*K)(TreeParams)>
static bool tree_raise_lds() {
  static std::atomic<bool> raised[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return false;
  if (raised[dev].load(std::memory_order_acquire)) return true;
  if (hipFuncSetAttribute((const void*)K, hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024) != hipSuccess) return false;
  raised[dev].store(true, std::memory_order_release);
  return true;
}
static int64_t tree_align(int64_t n) { return (n + 255) & ~(int64_t)255; }
static int64_t tree_most_pairs(int T, int R, int G, int rows) {
  const int64_t n = R < kTreeRequestsPerLaunch ? R : kTreeRequestsPerLaunch;
  return (int64_t)T * G / rows + n;
}

}  // namespace mi

using namespace mi;

static int64_t tree_workspace(const TreeShape& s, int T, int R, int G, int Hkv, int head_dim) {
  const int64_t rows = (int64_t)2 * s.grid * Hkv * s.rows;
  return 256 + tree_align(32 * tree_most_pairs(T, R, G, s.rows)) + tree_align(rows * 4) + rows * head_dim * 4;
}
extern "C" int64_t mi_tree_workspace_bytes(int32_t T, int32_t R, int32_t Hq, int32_t Hkv, int32_t head_dim) {
  if (T <= 0 || R <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || head_dim <= 0) return 0;
  int64_t most = 0;   // (which kernel a call takes depends on the cache as well)
  for (int many = 0; many < 2; ++many) {
    const int64_t n = tree_workspace(tree_shape(T, R, Hq, Hkv, head_dim, many != 0), T, R, Hq / Hkv, Hkv, head_dim);
    if (n > most) most = n;
  }
  return most;
}

extern "C" int mi_paged_tree_attention(
    const void* q, int64_t q_stride_tok, int64_t q_stride_head, const void* k_cache, const void* v_cache,
    int64_t kv_stride_chunk, int64_t kv_stride_tok, int64_t kv_stride_head, int32_t n_chunks, int32_t kv_dtype,
    const float* k_scales, const float* v_scales, const int32_t* block_table, int64_t bt_stride, int32_t table_columns,
    const int32_t* cu_seqlens_q, const int32_t* kv_lens, const int64_t* tree_mask, int64_t mask_stride,
    int32_t mask_words, void* out, int64_t o_stride_tok, int64_t o_stride_head, void* workspace, int64_t workspace_bytes,
    int32_t T, int32_t R, int32_t Hq, int32_t Hkv, int32_t head_dim, int32_t chunk_tokens, float softmax_scale,
    int32_t dtype, void* stream) {
  if (T == 0) return MI_OK;
  if (dtype != MI_DTYPE_BF16 && dtype != MI_DTYPE_FP16)
    return mi_fail(MI_ERR_UNSUPPORTED, "mi_paged_tree_attention: dtype must be MI_DTYPE_BF16 or MI_DTYPE_FP16");
  if (!q || !k_cache || !v_cache || !block_table || !cu_seqlens_q || !kv_lens || !tree_mask || !out)
    return mi_fail(MI_ERR_NULL, "mi_paged_tree_attention: null pointer argument");
  if (T < 0 || R <= 0 || Hq <= 0 || Hkv <= 0 || Hq % Hkv || Hkv > 65535)
    return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: need T >= 0, R > 0 and Hq a multiple of Hkv");
  const int G = Hq / Hkv;
  if (G > 64) return mi_fail(MI_ERR_UNSUPPORTED, "mi_paged_tree_attention: at most 64 query heads per KV head");
  if ((int64_t)T * G >= (int64_t)1 << 31 || (int64_t)T * G / 16 + R >= (int64_t)1 << 31)
    return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: too many rows");
  const bool fp8 = kv_dtype == MI_KV_FP8_E4M3;
  if (!fp8 && kv_dtype != MI_KV_16BIT) return mi_fail(MI_ERR_UNSUPPORTED, "mi_paged_tree_attention: unknown kv_dtype");
  if (head_dim != 64 && head_dim != 96 && head_dim != 128 && head_dim != 192 && head_dim != 256)
    return mi_fail(MI_ERR_UNSUPPORTED, "mi_paged_tree_attention: head_dim must be 64, 96, 128, 192 or 256");
  if (fp8 && head_dim != 64 && head_dim != 128)
    return mi_fail(MI_ERR_UNSUPPORTED, "mi_paged_tree_attention: an fp8 cache needs head_dim 64 or 128");
  if (fp8 && (!k_scales || !v_scales)) return mi_fail(MI_ERR_NULL, "mi_paged_tree_attention: an fp8 cache needs both scale arrays");
  if (chunk_tokens <= 0 || chunk_tokens % 16)
    return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: chunk size must be a positive multiple of 16");
  // (a tile's number has 32 bits, also that of the one a wavefront asks for behind the last: up to 512 tokens on)
  if (n_chunks <= 0 || table_columns <= 0 || (int64_t)table_columns * chunk_tokens > 0x7ffff000)
    return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: need a cache, and a block table of at most 2^31 - 4096 tokens a row");
  if (table_columns >= 1 << 24)   // (the 64-bit product with the reciprocal that finds a chunk)
    return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: a block table has fewer than 2^24 columns");
  if ((int64_t)table_columns * chunk_tokens * chunk_tokens >= (int64_t)1 << 40)   // (the reciprocal's own rounding)
    return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: tokens a row times chunk size must stay below 2^40");
  if (mask_words < 1 || mask_words > 4 || mask_stride < mask_words)
    return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: a row of the mask has 1 to 4 words");
  const int esz = fp8 ? 1 : 2;
  if (((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15)
    return mi_fail(MI_ERR_ALIGN, "mi_paged_tree_attention: q/k/v/out must be 16-byte aligned");
  if ((q_stride_tok | q_stride_head | o_stride_tok | o_stride_head) % 8 ||
      ((kv_stride_chunk | kv_stride_tok | kv_stride_head) * esz) % 16)
    return mi_fail(MI_ERR_ALIGN, "mi_paged_tree_attention: strides must keep rows 16-byte aligned");
  if (kv_stride_tok < 0 || kv_stride_head < 0 || kv_stride_head > 0x7fffffff || kv_stride_tok * (int64_t)chunk_tokens * esz >= (int64_t)1 << 31)
    return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: one chunk must span less than 2 GiB");
  if (!(softmax_scale > 0.f)) return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: softmax_scale must be positive");
  if (!workspace || workspace_bytes < mi_tree_workspace_bytes(T, R, Hq, Hkv, head_dim))
    return mi_fail(MI_ERR_WORKSPACE, "mi_paged_tree_attention: workspace too small (see mi_tree_workspace_bytes)");
  if ((uintptr_t)workspace & 15) return mi_fail(MI_ERR_ALIGN, "mi_paged_tree_attention: workspace must be 16-byte aligned");

  // Through LDS wherever that kernel has the cache's form (16 requests of 4 096 tokens, 8 KV heads of 128, us: 8 rows 68.7 -> 51.0,
  // 32 rows 86.8 -> 55.1, 64 rows 90.9 -> 60.4; one of 800, 20 rows: 19.5 -> 14.3), but for
  // - few rows of width 64, where its steps cost more than the loads (16 of 3 000 tokens, 12 rows, 32 KV heads: 73.9 and 95.9;
  //   16 of 4 096, 16 rows, 8 heads: 36.4 and 36.2; 64 of 2 000, 21 rows: 24.8 and 17.4);
  // - few rows of width 128 in a call that fills the memory, as far as the host knows (not the lengths): eight heads of a token then
  //   lie beside one another in a workgroup of the register kernel.  Registers and LDS, us: 64 requests of 2 000 tokens, 32 heads, 3 rows
  //   313 and 364, 12 rows 314 and 371; 128 of 1 000, 8 heads, 12 rows 97 and 106; 16 of 4 096, 16 heads, 3 rows 92 and 106; in short
  //   contexts the other way about (128 of 300, 8 heads, 12 rows 43.6 and 41.6).  With more rows to fewer heads LDS: 64 of 2 000,
  //   8 heads, 12 rows 103.0 and 100.5, 24 rows 119 and 101; 4 heads, 3 rows 52.3 and 49.1.  Level at 3 rows and fewer from some 256
  //   requests times heads on (16 of 1 000, 16 heads 30.7 and 31.9; 8 of them 22.7 and 23.0, 4 with 24 heads over 4 096 44.0 and 40.1).
  const int64_t mean = tree_mean_rows(T, R, G);
  const bool flood = head_dim == 128 && Hkv % 8 == 0 && 80 * (mean > 3 ? mean : 3) <= (int64_t)R * Hkv;
  const bool many = !fp8 && chunk_tokens % 32 == 0 && ((head_dim == 128 && !flood) || (head_dim == 64 && mean >= 16));
  const TreeShape shape = tree_shape(T, R, Hq, Hkv, head_dim, many);
  const bool f16 = dtype == MI_DTYPE_FP16;
  TreeParams p;
  p.q = (const uint16_t*)q; p.q_st = q_stride_tok; p.q_sh = q_stride_head;
  p.kc = (const uint8_t*)k_cache; p.vc = (const uint8_t*)v_cache;
  p.kv_sc = kv_stride_chunk; p.kv_st = (int32_t)kv_stride_tok; p.kv_sh = (int32_t)kv_stride_head;
  p.bt = block_table; p.bt_stride = bt_stride;
  p.mask = (const uint32_t*)tree_mask; p.mask_st = 2 * mask_stride; p.mask_words = 2 * mask_words;
  p.out = (uint16_t*)out; p.o_st = o_stride_tok; p.o_sh = o_stride_head;
  uint8_t* ws = (uint8_t*)workspace;
  const int64_t rows = (int64_t)2 * shape.grid * Hkv * shape.rows;
  p.pairs = (int32_t*)ws;
  p.pair_info = (int4*)(ws + 256);
  ws += 256 + tree_align(32 * tree_most_pairs(T, R, G, shape.rows));
  p.part_lse = (float*)ws;
  p.part_o = (float*)(ws + tree_align(rows * 4));
  p.k_scale = k_scales; p.v_scale = v_scales;
  p.chunk_magic = (((uint64_t)1 << 40) + chunk_tokens - 1) / chunk_tokens;
  p.g_magic = G == 1 ? 0u : (uint32_t)(((uint64_t)1 << 32) / G + 1);
  p.T = T; p.Hq = Hq; p.Hkv = Hkv; p.G = G; p.chunk = chunk_tokens; p.n_chunks = n_chunks; p.table_cols = table_columns;
  p.grid = shape.grid; p.share = shape.share; p.rows = shape.rows; p.scale_log2 = softmax_scale * 1.4426950408889634f;
  hipStream_t st = (hipStream_t)stream;
  const dim3 grid(shape.grid, Hkv / shape.heads), block(64 * shape.waves);
  const bool wide = head_dim > 128;
  // tokens of a tile: 32, 16 of wide heads, 64 of an fp8 cache with narrow ones (what the registers hold in flight); a tile
  // lies in one chunk
  const int nt = wide || chunk_tokens % 32 ? 1 : fp8 && head_dim == 64 && chunk_tokens % 64 == 0 ? 4 : 2;
  const int tile = many ? 32 : 16 * nt;
  if (tree_most_pairs(T, R, G, shape.rows) * ((int64_t)table_columns * chunk_tokens / tile + 2) >= (int64_t)1 << 31)
    return mi_fail(MI_ERR_SHAPE, "mi_paged_tree_attention: rows per KV head times the tokens of a table row must stay below some 2^36");
  for (int r0 = 0; r0 < R; r0 += kTreeRequestsPerLaunch) {
    p.r_base = r0;
    p.R = R - r0 < kTreeRequestsPerLaunch ? R - r0 : kTreeRequestsPerLaunch;
    p.cu_q = cu_seqlens_q + r0; p.lens = kv_lens + r0;
    p.last_slice = r0 + p.R == R;
    // (the walk's arrays; where parts share, what the wavefronts of a part join: 64 lanes' registers each)
    const size_t walk = p.R <= 64 ? 0 : (size_t)p.R * 3 * sizeof(int32_t);
    const size_t lds = walk + (!many && shape.share > 1 ? (size_t)shape.waves * 64 * (shape.rows / shape.share / 16) * (head_dim / 4 + 2) * sizeof(float) : 0);
#define MI_TREE_ONE(HD_, NT_, NQ_, FP8_, F16_, SHARE_)                                                                 \
    do {                                                                                                               \
      if (SHARE_ && lds > 65536 && !tree_raise_lds<paged_tree_kernel<HD_, NT_, NQ_, FP8_, F16_, SHARE_>>())            \
        return mi_fail(MI_ERR_LAUNCH, "mi_paged_tree_attention: cannot raise the dynamic LDS limit");                  \
      hipLaunchKernelGGL((paged_tree_kernel<HD_, NT_, NQ_, FP8_, F16_, SHARE_>), grid, block, lds, st, p);             \
    } while (0)
#define MI_TREE(HD_, NT_, NQ_, FP8_)                                                                                   \
    do {                                                                                                               \
      if (f16 && p.share > 1) MI_TREE_ONE(HD_, NT_, NQ_, FP8_, true, true);                                            \
      else if (f16) MI_TREE_ONE(HD_, NT_, NQ_, FP8_, true, false);                                                     \
      else if (p.share > 1) MI_TREE_ONE(HD_, NT_, NQ_, FP8_, false, true);                                             \
      else MI_TREE_ONE(HD_, NT_, NQ_, FP8_, false, false);                                                             \
    } while (0)
#define MI_TREE_16(HD_)                                                                                                \
    do {                                                                                                               \
      if (nt == 1) MI_TREE(HD_, 1, 2, false);                                                                          \
      else MI_TREE(HD_, 2, 2, false);                                                                                  \
    } while (0)
#define MI_TREE_8(HD_)                                                                                                 \
    do {                                                                                                               \
      if (nt == 1) MI_TREE(HD_, 1, 2, true);                                                                           \
      else MI_TREE(HD_, 2, 2, true);                                                                                   \
    } while (0)
#define MI_TREE_ROWS(HD_, W_)                                                                                          \
    do {                                                                                                               \
      if (f16) hipLaunchKernelGGL((paged_tree_rows_kernel<HD_, W_, true>), grid, block, lds, st, p);                   \
      else hipLaunchKernelGGL((paged_tree_rows_kernel<HD_, W_, false>), grid, block, lds, st, p);                      \
    } while (0)
    if (many && shape.waves == 4) {
      if (head_dim == 64) MI_TREE_ROWS(64, 4);
      else MI_TREE_ROWS(128, 4);
    } else if (many) {
      if (head_dim == 64) MI_TREE_ROWS(64, 8);
      else MI_TREE_ROWS(128, 8);
    } else if (fp8 && nt == 4) MI_TREE(64, 4, 2, true);
    else if (fp8 && head_dim == 64) MI_TREE_8(64);
    else if (fp8) MI_TREE_8(128);
    else if (head_dim == 64) MI_TREE_16(64);
    else if (head_dim == 96) MI_TREE_16(96);
    else if (head_dim == 128) MI_TREE(128, 1, 2, false);
    else if (head_dim == 192) MI_TREE(192, 1, 1, false);
    else MI_TREE(256, 1, 1, false);
#undef MI_TREE_ROWS
#undef MI_TREE_8
#undef MI_TREE_16
#undef MI_TREE
#undef MI_TREE_ONE
    // (thread sets per row: for the partials that a request is expected to be cut into)
    const int cols = head_dim / 4, block_rows = kTreeMergeThreads / cols;
    const int64_t pairs = tree_most_pairs(T, p.R, G, shape.rows);
    const int groups = shape.grid / pairs > 16 ? 4 : shape.grid / pairs > 8 ? 2 : 1;
    const dim3 mgrid((unsigned)pairs, Hkv, (shape.rows + block_rows - 1) / block_rows), mblock(groups > 1 ? groups * cols * block_rows : kTreeMergeThreads);
    if (f16) hipLaunchKernelGGL((paged_tree_merge_kernel<true>), mgrid, mblock, 0, st, p, head_dim, groups);
    else hipLaunchKernelGGL((paged_tree_merge_kernel<false>), mgrid, mblock, 0, st, p, head_dim, groups);
  }
  return mi_check_launch("mi_paged_tree_attention");
}
