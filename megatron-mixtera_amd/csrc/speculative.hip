// Verification of drafted tokens and the move of the accepted nodes' cache rows (gfx950).
//
// Every request brings a tree of drafted tokens (see paged_tree.hip for the attention over it): row i of the logits is
// the target's view of what follows node i, parents[i] the node (inside the request) that token i was drafted after.
//
// Verification walks each tree from its root.  With p the target's distribution at a node (softmax of logits /
// temperature over the values that reach `cut`), the node's children are tried in order:
//   * draft probabilities q (the distribution that the children were drawn from, one row per node): a child with token t is
//     accepted where u q(t) < p_j(t), and after a rejection p_{j+1} = (p_j - q)+, normalised.  Written out this is
//       p_j = (p - c_j q)+ / n_j,   c_0 = 0, n_0 = 1,   c_{j+1} = c_j + n_j,   n_{j+1} = sum (p - c_{j+1} q)+,
//     so a node needs two numbers besides p and q, however often it was rejected;
//   * without them (tokens that the draft chose rather than drew): accepted where u < p_j(t), and a rejected token leaves
//     the distribution;
//   * greedy: accepted where t is the largest logit's index.
// The first accepted child is the next node; where there is none the request's last token is drawn from what is left by an
// inverse CDF in vocabulary order, so that the tokens are distributed as the target's own draws would be.
//
// Tokens are whole numbers picked at borders of long sums, so exponentials and sums are 64-bit: one rounding of a 32-bit
// cumulative sum (6e-8) is as wide as the whole share of many a token of a 128 k vocabulary.  The exponential is a table of
// 2^(i/128) in LDS and a polynomial of degree 4 (relative error 1e-15).  Where the rows' sums only scale what is compared (draft
// probabilities: what a rejection leaves is a sum of its own) they take a form of 6e-10 (add_exps); where the rejected tokens are
// taken off them a difference has to be as exact as its terms, and they take the 64-bit form.
//
// One launch for all rows (issue-bound), one workgroup per request for the walk, one launch for what a rejection leaves of the last
// node's row, one workgroup per request for the draw: the last three are chains of dependent loads.  us, vocabulary 128 256, bf16:
// 5 nodes, draft probabilities 4.3 + 4.6 + 3.8 + 8.0; 64 chains of 6: 35.0 + 6.7 + 13.5 + 13.3, without draft probabilities 49.1 + 5.1 +
// 13.0 (the draw); 671 nodes in 16 trees under a cut, no draft probabilities 32.6 + 9.6 + 7.2; 716 nodes in 16 trees, draft
// probabilities 61.1 + 299 + 7.7 + 12.6 (the walk sums a row for every rejected child that has a further sibling, on one CU); greedy
// over 270 rows of 32 003 fp32 logits 9.2 + 4.1.
#include <type_traits>

#include "mi_capi_internal.h"
#include "mi_common.h"

namespace mi {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyNodes = 1024;    // nodes of a request that are looked at: what the walk holds in LDS
constexpr int kVerifyMostParts = 64;
constexpr int kVerifyPart = 8192;     // elements of a part, at most (whose weights the draw's threads hold, eight each)

struct VerifyPartial {   // of one part of a row
  double sum;            // of exp(x - max); greedy: unused
  float max;
  int32_t index;         // greedy: the first place of the maximum
};
struct VerifyState {     // what the walk hands the draw
  double c;              // weights are (p - c q)+; 0: no child of the last node was rejected, q is not read
  double sum;            // the last node's row: sum of exp(x - top)
  float top;
  int32_t row;           // -1: the request is empty
  int32_t tested;        // whether its children were tried (a path of max_path nodes: no)
  int32_t pad;
};

struct VerifyParams {
  const uint8_t* logits; int64_t stride;   // bytes between rows
  const uint8_t* draft; int64_t draft_stride; int32_t draft_dtype;
  const int64_t* tokens;
  const int32_t* parents;
  const int32_t* cu;
  const float* uniform;
  const float* cut;
  int64_t* out_tokens; int32_t* out_rows; int32_t* out_counts;
  VerifyPartial* partial;    // [T][parts]
  double* residual;          // [R][parts]
  VerifyState* state;        // [R]
  int32_t* removed;          // [T]: the tokens that a request's last node's rejected children took out, -1: none
  int32_t T, R, V, max_path, parts, part;   // part: elements, a multiple of 8
  float inv_temperature; int32_t scaled;
};

constexpr double kLog2e = 1.4426950408889634074;

// The table of 2^(i / 128), filled by the workgroup.
static __device__ __forceinline__ void fill_exp_table(double* table) {
  for (int i = threadIdx.x; i < 128; i += blockDim.x) table[i] = exp2(i * (1.0 / 128));
}
constexpr double kExpMagic = 1.5 * 35184372088832.0;   // 1.5 2^45: an addition rounds to multiples of 1/128
// e^d for d <= 0 (NaN: 0)
static __device__ __forceinline__ double table_exp(const double* table, double d) {
  const double t = fmax(d * kLog2e, -2000.0);
  const double u = t + kExpMagic;
  const double r = (t - (u - kExpMagic)) * 0.69314718055994530942;
  const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, u);
  double y = __builtin_fma(r, 1.0 / 24, 1.0 / 6);
  y = __builtin_fma(r, y, 0.5);
  y = __builtin_fma(r, y, 1.0);
  y = __builtin_fma(r, y, 1.0);
  return __builtin_ldexp(table[k & 127] * y, k >> 7);
}
// The same for long sums, two thirds of the instructions: nothing below e^-690, whose place e^-690 takes.
static __device__ __forceinline__ void table_exp_parts(const double* table, double d, double& scale, double& y) {
  constexpr double kLn2 = 0.69314718055994530942;
  d = fmax(d, -690.0);
  const double u = __builtin_fma(d, kLog2e, kExpMagic);
  const double r = __builtin_fma(d, kLog2e, kExpMagic - u);
  const int k = (int)(uint32_t)__builtin_bit_cast(uint64_t, u);
  y = __builtin_fma(r, kLn2 * kLn2 * kLn2 * kLn2 / 24, kLn2 * kLn2 * kLn2 / 6);
  y = __builtin_fma(r, y, kLn2 * kLn2 / 2);
  y = __builtin_fma(r, y, kLn2);
  y = __builtin_fma(r, y, 1.0);
  scale = __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, table[k & 127]) + ((uint64_t)(uint32_t)(k >> 7) << 52));
}

static __device__ __forceinline__ float load_element(const uint8_t* row, int dtype, int i) {
  if (dtype == 0) return reinterpret_cast<const float*>(row)[i];
  const uint16_t x = reinterpret_cast<const uint16_t*>(row)[i];
  return dtype == 1 ? bf16_to_f32(x) : to_f32<true>(x);
}

// Eight elements e0 .. e0 + 7 of a row: a 16-byte line or two where they are aligned and inside, which `fetch` sends for
// and `values` waits for; otherwise one by one, `fill` outside [0, V).
template <int DT>
struct VerifyLine {
  uint4 a, b;
  bool whole;
  __device__ __forceinline__ void fetch(const uint8_t* row, int e0, int V) {
    const uint8_t* at = row + (int64_t)e0 * (DT == 0 ? 4 : 2);
    whole = e0 >= 0 && e0 + 8 <= V && !((uintptr_t)at & 15);
    if (whole) {
      a = ld16(at);
      if constexpr (DT == 0) b = ld16(at + 16);
    }
  }
  __device__ __forceinline__ void values(const uint8_t* row, int e0, int V, float fill, float (&x)[8]) const {
    if (whole) {
      if constexpr (DT == 0) {
        x[0] = __uint_as_float(a.x); x[1] = __uint_as_float(a.y); x[2] = __uint_as_float(a.z); x[3] = __uint_as_float(a.w);
        x[4] = __uint_as_float(b.x); x[5] = __uint_as_float(b.y); x[6] = __uint_as_float(b.z); x[7] = __uint_as_float(b.w);
      } else {
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[2 * j] = lo_to_f32<DT == 2>(w[j]);
          x[2 * j + 1] = hi_to_f32<DT == 2>(w[j]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = e0 + j >= 0 && e0 + j < V ? load_element(row, DT, e0 + j) : fill;
    }
  }
};
// The same of a type that is known at run time.
struct VerifyAnyLine {
  VerifyLine<0> line;
  __device__ __forceinline__ void fetch(const uint8_t* row, int dtype, int e0, int V) {
    if (dtype == 0) {
      line.fetch(row, e0, V);
    } else {
      VerifyLine<1> l;
      l.whole = false;
      l.fetch(row, e0, V);
      line.a = l.a;
      line.whole = l.whole;
    }
  }
  __device__ __forceinline__ void values(const uint8_t* row, int dtype, int e0, int V, float fill, float (&x)[8]) const {
    if (dtype == 0) {
      line.values(row, e0, V, fill, x);
    } else if (dtype == 1) {
      const VerifyLine<1> l{line.a, line.b, line.whole};
      l.values(row, e0, V, fill, x);
    } else {
      const VerifyLine<2> l{line.a, line.b, line.whole};
      l.values(row, e0, V, fill, x);
    }
  }
};

// A row of logits cut into parts of `part` elements.  Parts are counted from the last 16-byte line at or before the row's
// first element, so that the groups of eight are aligned whatever the row's own address: element e lies at place e + shift.
template <int DT>
struct VerifyRow {
  const uint8_t* row;
  int shift;
  float cut;
  __device__ __forceinline__ VerifyRow(const VerifyParams& p, int i) {
    row = p.logits + (int64_t)i * p.stride;
    shift = (int)((uintptr_t)row & 15) / (DT == 0 ? 4 : 2);
    cut = p.cut ? p.cut[i] : -INFINITY;
  }
  // a logit as the sampler sees it: times the reciprocal of the temperature, rounded to the logits' type; -inf: left out
  __device__ __forceinline__ float finish(const VerifyParams& p, float x) const {
    if (p.scaled) {
      x *= p.inv_temperature;
      // (the sampler's fp32 product, rounded to fp16 by another instruction: in one, v_fma_mixlo_f16, it would be rounded once,
      // and 6.6 % of fp16's numbers over 0.6 come out a step lower, some of them below a cut that they made)
      if (DT == 2) asm("" : "+v"(x));
      if (DT != 0) x = to_f32<DT == 2>(f32_to_16<DT == 2>(x));
    }
    return x < cut ? -INFINITY : x;
  }
  __device__ __forceinline__ float at(const VerifyParams& p, int e) const { return finish(p, load_element(row, DT, e)); }
};

// One step of a sum over the lanes: the value of the lane that DPP control CTRL names, 0 where there is none or MASK leaves
// the lane's row of 16 out.
template <int CTRL, int MASK>
static __device__ __forceinline__ double dpp_f64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, MASK, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, MASK, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Inclusive sums over the lanes: inside the rows of 16, then the last of a row to the next one, of two rows to the next two.
static __device__ __forceinline__ double wave_scan_f64(double x) {
  x += dpp_f64<0x111, 0xf>(x);
  x += dpp_f64<0x112, 0xf>(x);
  x += dpp_f64<0x114, 0xf>(x);
  x += dpp_f64<0x118, 0xf>(x);
  x += dpp_f64<0x142, 0xa>(x);
  x += dpp_f64<0x143, 0xc>(x);
  return x;
}
static __device__ __forceinline__ double read_lane_f64(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, lane), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
static __device__ __forceinline__ double wave_sum_f64(double x) { return read_lane_f64(wave_scan_f64(x), 63); }
template <int CTRL, int MASK>
static __device__ __forceinline__ float dpp_max_f32(float x) {   // (-inf where there is no lane)
  return fmaxf(x, __int_as_float(__builtin_amdgcn_update_dpp((int)0xff800000u, __float_as_int(x), CTRL, MASK, 0xf, false)));
}
static __device__ __forceinline__ float wave_max_f32(float x) {
  x = dpp_max_f32<0x111, 0xf>(x);
  x = dpp_max_f32<0x112, 0xf>(x);
  x = dpp_max_f32<0x114, 0xf>(x);
  x = dpp_max_f32<0x118, 0xf>(x);
  x = dpp_max_f32<0x142, 0xa>(x);
  x = dpp_max_f32<0x143, 0xc>(x);
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Sum of e^(x - top) over eight logits, `top` among the row's wavefront, |top| < kNarrow: the exponent's whole 128ths and what
// is left of them come from 32-bit products (a whole number below 2^23 beside its fraction), 2^(whole/128) from the table, the
// fraction's own e^. as 1 + a 32-bit polynomial of at most 0.0027: 6e-10 of a weight at most, a hundredth of half a step of the
// uniform numbers that it meets, in two thirds of the 64-bit form's time.
constexpr float kNarrow = 16384.f;
static __device__ __forceinline__ void add_exps(const double* table, const float (&x)[8], float low, float top, int whole, bool few, double& sum, double& rest) {
  constexpr double kStep = kLog2e * 128, kLn = 0.69314718055994530942 / 128;
  constexpr float kHigh = (float)kStep, kLow = (float)(kStep - (double)kHigh);
  float magic = 12582912.f, second = (float)(kLn * kLn / 2);   // (1.5 2^23; both stay in registers)
  asm("" : "+v"(magic), "+v"(second));
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (few && !__builtin_amdgcn_ballot_w64(x[j] > -INFINITY)) continue;
    const float v = __builtin_amdgcn_fmed3f(x[j], low, top);   // (NaN: low)
    const float u = __builtin_fmaf(v, kHigh, magic);
    float r = __builtin_fmaf(v, kHigh, -(u - magic));
    r = __builtin_fmaf(v, kLow, r);
    const int k = (int)__float_as_uint(u) - whole;
    const float y = r * __builtin_fmaf(r, __builtin_fmaf(r, (float)(kLn * kLn * kLn / 6), second), (float)kLn);
    const uint64_t t = __builtin_bit_cast(uint64_t, table[k & 127]);
    const uint32_t hi = (uint32_t)(t >> 32) + ((uint32_t)(k & ~127) << 13);
    const double w = __builtin_bit_cast(double, (uint64_t)hi << 32 | (uint32_t)t);
    sum += w;
    rest = __builtin_fma(w, (double)y, rest);
  }
}

// Maximum and sum of exponentials (greedy: maximum and its first place) of one part of one row, which the threads hold in
// registers: all loads are on their way before the first value is used.  Scaling and cut keep the order of logits, so that the
// largest of eight says whether any of them counts.  Bound by the rate at which vector instructions issue (some 27 a logit, 11 of
// them for its exponential): 384 rows of 128 256 bf16 logits 35.0 us, 2.8 TB/s; 671 rows of which a cut leaves 50 logits each 32.6 us,
// 5.3 TB/s.  With 64-bit exponentials the former took 47.5 us, and 52 with a running maximum per thread; without the looks at eights and
// at single elements under a cut the latter took 45.6.  The 64-bit form is what a call without draft probabilities needs (64 chains of
// 6, the whole call: 51.3 -> 62.2 us, their rows 49.1; under a cut, which leaves few exponentials, 30.7 and 30.4).
constexpr int kVerifyLines = kVerifyPart / (8 * kVerifyThreads);
template <int DT, bool GREEDY>
__global__ __launch_bounds__(kVerifyThreads) void verify_rows_kernel(VerifyParams p) {
  __shared__ double table[128];
  __shared__ double sums[4];
  __shared__ float tops[4];
  __shared__ int places[4];
  const int part = blockIdx.y, row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const VerifyRow<DT> rd(p, row);
  const int begin = part * p.part - rd.shift, end = min(begin + p.part, p.V), mine = begin + 8 * (int)threadIdx.x;
  VerifyLine<DT> lines[kVerifyLines];
#pragma unroll
  for (int i = 0; i < kVerifyLines; ++i)
    if (mine + 8 * kVerifyThreads * i < end) lines[i].fetch(rd.row, mine + 8 * kVerifyThreads * i, p.V);
  if (!GREEDY) fill_exp_table(table);
  float top = -INFINITY, line_top[kVerifyLines];
  int place = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < kVerifyLines; ++i) {
    const int e0 = mine + 8 * kVerifyThreads * i;
    line_top[i] = -INFINITY;
    if (e0 >= end) continue;
    float v[8];
    lines[i].values(rd.row, e0, p.V, -INFINITY, v);
    if constexpr (GREEDY) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((v[j] > top || place == 0x7fffffff) && e0 + j >= 0 && e0 + j < p.V && v[j] == v[j]) {
          top = v[j];
          place = e0 + j;
        }
    } else {
      const float m = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
      line_top[i] = rd.finish(p, m);
      top = fmaxf(top, line_top[i]);
    }
  }
  const float wave_top = wave_max_f32(top);
  if (lane == 0) tops[wave] = wave_top;
  __syncthreads();   // (the table, too)
  const float all = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  const bool narrow = !GREEDY && __builtin_amdgcn_readfirstlane(p.draft && fabsf(all) < kNarrow);
  if constexpr (GREEDY) {
    int best = top == all ? place : 0x7fffffff;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) best = min(best, __shfl_xor(best, d, 64));
    if (lane == 0) places[wave] = best;
  } else {
    double s0 = 0, s1 = 0;
    const bool plain = !p.scaled && !p.cut, few = p.cut != nullptr;
    const float power = narrow ? rintf(all * (float)kLog2e) : 0.f;   // the narrow form's sums are relative to 2^power
    const int whole = 0x4b400000 + 128 * (int)power;
#pragma unroll
    for (int i = 0; i < kVerifyLines; ++i) {
      if (!__builtin_amdgcn_ballot_w64(line_top[i] > -INFINITY)) continue;   // (a cut leaves few)
      const int e0 = mine + 8 * kVerifyThreads * i;
      float v[8];
      if (e0 < end) {
        lines[i].values(rd.row, e0, p.V, -INFINITY, v);
        if (!plain)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = rd.finish(p, v[j]);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = -INFINITY;
      }
      if (narrow) {
        add_exps(table, v, all - 690.f, all, whole, few, s0, s1);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if (few && !__builtin_amdgcn_ballot_w64(v[j] > -INFINITY)) continue;
          double scale, y;
          table_exp_parts(table, (double)v[j] - (double)all, scale, y);
          s0 = v[j] > -INFINITY ? __builtin_fma(scale, y, s0) : s0;
        }
      }
    }
    const double s = wave_sum_f64(s0 + s1);
    if (lane == 0) sums[wave] = s;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    VerifyPartial o{0, all, 0x7fffffff};
    if constexpr (GREEDY) {
      o.index = min(min(places[0], places[1]), min(places[2], places[3]));
    } else {
      o.sum = sums[0] + sums[1] + sums[2] + sums[3];
      if (narrow) o.sum *= table_exp(table, (double)rintf(all * (float)kLog2e) * 0.69314718055994530942 - (double)all);
    }
    p.partial[(int64_t)row * p.parts + part] = o;
  }
}

// Sum over the workgroup, in every thread.
static __device__ __forceinline__ double block_sum(double x, double* scratch) {
  x = wave_sum_f64(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = x;
  __syncthreads();
  double s = 0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) s += scratch[w];
  return s;
}

// This thread's share of the sum of (p - c q)+ over the places [0, places) from `first` on of a row; MINUS false: c is 0, q is not read.
// (Two or four lines ahead of their use took more registers and as much time.)
template <int DT, bool MINUS>
static __device__ __forceinline__ double left_over(const VerifyParams& p, const VerifyRow<DT>& rd, const double* table, int row,
                                                   int first, int places, int threads, float top, double sum, double c) {
  const uint8_t* qr = p.draft + (int64_t)row * p.draft_stride;
  const double inv = 1.0 / sum;
  const int begin = first - rd.shift, end = min(begin + places, p.V);
  double s = 0;
  for (int e0 = begin + 8 * (int)threadIdx.x; e0 < end; e0 += 8 * threads) {
    VerifyLine<DT> px;
    VerifyAnyLine qx;
    px.fetch(rd.row, e0, p.V);
    if (MINUS) qx.fetch(qr, p.draft_dtype, e0, p.V);
    float x[8], y[8] = {};
    px.values(rd.row, e0, p.V, -INFINITY, x);
    if (MINUS) qx.values(qr, p.draft_dtype, e0, p.V, 0.f, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float v = rd.finish(p, x[j]);
      double scale, z;
      table_exp_parts(table, (double)v - (double)top, scale, z);
      const double w = v > -INFINITY ? scale * inv : 0.0;
      s += fmax(__builtin_fma(w, z, -c * (double)y[j]), 0.0);
    }
  }
  return s;
}

// The walk of one request's tree, one workgroup each.  A chain of dependent steps: parents and tokens, the logits that they name
// (beside the partial sums of all the request's rows), then LDS only, but for draft probabilities after a rejection: what is left of
// the row, by the one workgroup, for each that has a further sibling.  4.6 us for 5 nodes, 9.6 for 16 trees of 25-61 nodes without
// draft probabilities, 299 with them.
constexpr int kWalkThreads = 1024;
enum { kGreedy = 0, kTarget = 1, kDraft = 2 };
template <int DT, int MODE>
__global__ __launch_bounds__(kWalkThreads) void verify_walk_kernel(VerifyParams p) {
  __shared__ double table[128];
  __shared__ double scratch[kWalkThreads / 64];
  __shared__ double prob[kVerifyNodes], sum_s[kVerifyNodes];
  __shared__ float top_s[kVerifyNodes], q_s[kVerifyNodes];
  __shared__ int32_t parent[kVerifyNodes], token[kVerifyNodes], after[kVerifyNodes];   // after: the next node; draft: the first child
  __shared__ int32_t sibling[MODE == kDraft ? kVerifyNodes : 1];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
  const int begin = min(max(p.cu[r], 0), p.T), n = min(min(max(p.cu[r + 1], begin), p.T) - begin, kVerifyNodes);
  int32_t* const rows = p.out_rows + (int64_t)r * p.max_path;
  int64_t* const out = p.out_tokens + (int64_t)r * p.max_path;
  for (int i = tid; i < p.max_path; i += kWalkThreads) {
    rows[i] = -1;
    out[i] = -1;
  }
  if (n <= 0) {
    if (tid == 0) {
      p.out_counts[r] = 0;
      p.state[r] = VerifyState{0, 0, 0.f, -1, 0, 0};
    }
    return;
  }
  // a node to a thread: its parent, its token, what the parent's row says about it -- on their way during the sums below
  static_assert(kVerifyNodes == kWalkThreads, "a node to a thread");
  int up = -1;
  int64_t drafted = -1;
  if (tid < n) {
    up = p.parents[begin + tid];
    drafted = p.tokens[begin + tid];
    if (tid == 0 || up < 0 || up >= tid) up = -1;
  }
  const bool inside = drafted >= 0 && drafted < p.V;
  const float chance = MODE == kTarget && tid < n ? p.uniform[begin + tid] : 0.f;
  float said = -INFINITY, q = 0.f;
  if (MODE != kGreedy && up >= 0 && inside) {
    said = VerifyRow<DT>(p, begin + up).at(p, (int)drafted);
    if (MODE == kDraft) q = load_element(p.draft + (int64_t)(begin + up) * p.draft_stride, p.draft_dtype, (int)drafted);
  }
  fill_exp_table(table);
  __syncthreads();
  // maximum and sum of a row: a wavefront each, a part to a lane
  static_assert(kVerifyMostParts == 64, "a part to a lane");
  constexpr int kWaves = kWalkThreads / 64, kAhead = 4;
  for (int i0 = tid >> 6; i0 < n; i0 += kAhead * kWaves) {
    VerifyPartial parts[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kWaves;
      parts[k] = VerifyPartial{0, -INFINITY, 0x7fffffff};
      if (i < n && lane < p.parts) parts[k] = p.partial[(int64_t)(begin + i) * p.parts + lane];
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kWaves;
      if (i >= n) break;
      const VerifyPartial& part = parts[k];
      const float top = wave_max_f32(part.max);
      if (MODE == kGreedy) {
        int best = part.max == top ? part.index : 0x7fffffff;
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) best = min(best, __shfl_xor(best, d, 64));
        if (lane == 0) token[i] = best;   // (of the row, here)
      } else {
        const double s = wave_sum_f64(part.max > -INFINITY ? part.sum * table_exp(table, (double)part.max - (double)top) : 0.0);
        if (lane == 0) {
          top_s[i] = top;
          sum_s[i] = s;
        }
      }
    }
  }
  if (tid < n) {
    after[tid] = 0x7fffffff;
    parent[tid] = up;
  }
  __syncthreads();
  if (MODE == kGreedy) {
    if (up >= 0 && inside && drafted == token[up]) atomicMin(&after[up], tid);   // (a row of NaN has no place: 2^31 - 1)
  } else if (tid < n) {
    token[tid] = inside ? (int)drafted : -1;
    prob[tid] = up >= 0 && inside && sum_s[up] > 0 ? table_exp(table, (double)said - (double)top_s[up]) / sum_s[up] : 0.0;
    q_s[tid] = q;
  }
  __syncthreads();
  if (MODE == kTarget) {
    // a token that an earlier sibling had has left the distribution
    bool again = false;
    double before = 0;
    const int i = tid, tok = inside ? (int)drafted : -1, most = (tid & ~63) < n ? min(n, (tid | 63) + 1) : 0;   // (one count of turns for the wavefront)
#pragma unroll 8
    for (int j = 1; j < most; ++j) again |= (parent[j] == up) & (token[j] == tok) & (j < i);
    __syncthreads();
    if (again && up >= 0) prob[i] = 0;
    __syncthreads();
    if (i < n) p.removed[begin + i] = again ? -1 : tok;
#pragma unroll 8
    for (int j = 1; j < most; ++j) before = __builtin_fma(prob[j], (parent[j] == up) & (j < i) ? 1.0 : 0.0, before);   // (a load a turn, no branch)
    // (what rounding takes below zero is nothing: no token is accepted on it)
    if (up >= 0 && (double)chance * fmax(1.0 - before, 0.0) < prob[i]) atomicMin(&after[up], i);
    __syncthreads();
  }
  if (MODE != kDraft) {
    if (tid == 0) {
      int at = 0, count = 1;
      rows[0] = begin;
      while (count < p.max_path && after[at] < n) {
        const int next = after[at];
        out[count - 1] = token[MODE == kGreedy ? at : next];   // (an accepted token is its parent's largest logit)
        at = next;
        rows[count++] = begin + at;
      }
      p.out_counts[r] = count;
      if (MODE == kGreedy) out[count - 1] = token[at] == 0x7fffffff ? 0 : token[at];
      else p.state[r] = VerifyState{0, sum_s[at], top_s[at], begin + at, count < p.max_path, 0};
    }
    return;
  }
  // Draft probabilities: the rejections of a node's earlier children decide what a later one is held against.
  if (tid < n) {
    int next = 0x7fffffff;
    if (up >= 0) atomicMin(&after[up], tid);
#pragma unroll 8
    for (int j = (tid & ~63) + 1; j < n; ++j) next = min(next, (parent[j] == up) & (j > tid) ? j : 0x7fffffff);
    sibling[tid] = up >= 0 && next < n ? next : -1;
  }
  __syncthreads();
  int at = 0, count = 1;
  double c = 0;
  if (tid == 0) rows[0] = begin;
  while (count < p.max_path) {
    double left = 1;
    int child = after[at] < n ? after[at] : -1;
    while (child >= 0) {
      const double of = q_s[child], w = prob[child] - c * of;
      if ((double)p.uniform[begin + child] * left * of < w) break;
      c += left;
      child = sibling[child];
      if (child >= 0) {   // (what is left matters to a sibling; the draw makes its own sum)
        const VerifyRow<DT> rd(p, begin + at);
        left = block_sum(left_over<DT, true>(p, rd, table, begin + at, 0, p.V + rd.shift, kWalkThreads, top_s[at], sum_s[at], c), scratch);
      }
    }
    if (child < 0) break;
    at = child;
    c = 0;
    if (tid == 0) {
      out[count - 1] = token[at];
      rows[count] = begin + at;
    }
    ++count;
  }
  if (tid == 0) {
    p.out_counts[r] = count;
    p.state[r] = VerifyState{c, sum_s[at], top_s[at], begin + at, count < p.max_path, 0};   // (c is 0 where max_path ended it)
  }
}

// Draft probabilities: what is left of one part of the last node's distribution, sum (p - c q)+.  Where nothing was rejected that is
// the part's own sum, which the draw's weights need with their own 64 bits: the rows' sums are good to 6e-10 here.
template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_left_kernel(VerifyParams p) {
  __shared__ double table[128];
  __shared__ double scratch[kVerifyThreads / 64];
  const int part = blockIdx.y, r = blockIdx.x;
  const VerifyState st = p.state[r];
  fill_exp_table(table);   // (the state is on its way)
  __syncthreads();
  if (st.row < 0) return;
  const VerifyRow<DT> rd(p, st.row);
  const int first = part * p.part;
  double mine;   // (the row of a node without children may hold anything)
  if (st.c != 0) mine = left_over<DT, true>(p, rd, table, st.row, first, p.part, kVerifyThreads, st.top, st.sum, st.c);
  else mine = left_over<DT, false>(p, rd, table, st.row, first, p.part, kVerifyThreads, st.top, st.sum, 0.0);
  const double s = block_sum(mine, scratch);
  if (threadIdx.x == 0) p.residual[(int64_t)r * p.parts + part] = s;
}

// The draw of a request's last token: the part that holds it (every wavefront, a part to a lane), then the place inside the
// part, whose weights the threads hold.  Three trips to memory one after the other and two scans; 8.0 us for one request, 13.3 for 64
// (with the parts' sums in one thread and the weights in LDS 24.6 and 24.8).
constexpr int kDrawThreads = 1024;
static_assert(kVerifyPart == 8 * kDrawThreads, "eight places to a thread");
template <int DT, int MODE>
__global__ __launch_bounds__(kDrawThreads) void verify_draw_kernel(VerifyParams p) {
  constexpr int kWaves = kDrawThreads / 64;
  __shared__ double table[128];
  __shared__ unsigned long long gone_s[kVerifyMostParts];
  __shared__ double run[kWaves];
  __shared__ uint32_t gone[MODE == kTarget ? kVerifyPart / 32 : 1];
  __shared__ int found[2];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const VerifyState st = p.state[r];
  const int begin = min(max(p.cu[r], 0), p.T), n = min(min(max(p.cu[r + 1], begin), p.T) - begin, kVerifyNodes);
  fill_exp_table(table);   // (the state is on its way)
  if (MODE == kTarget)
    for (int i = tid; i < kVerifyPart / 32; i += kDrawThreads) gone[i] = 0;
  if (tid < kVerifyMostParts) gone_s[tid] = 0;
  if (tid == 0) {
    found[0] = 0x7fffffff;
    found[1] = -1;
  }
  __syncthreads();
  if (st.row < 0) return;
  const int node = st.row - begin, count = p.out_counts[r];
  const float uniform = p.uniform[begin];
  const VerifyRow<DT> rd(p, st.row);
  const double inv = 1.0 / st.sum;
  auto chance = [&](float x) { return table_exp(table, (double)x - (double)st.top) * inv; };
  double whole = 0;
  if (lane < p.parts) {
    const VerifyPartial q = p.partial[(int64_t)st.row * p.parts + lane];
    if (q.max > -INFINITY) whole = q.sum * chance(q.max);
  }
  double mass = whole;
  if (MODE == kDraft) mass = lane < p.parts ? p.residual[(int64_t)r * p.parts + lane] : 0.0;
  // tokens that the rejected children took out: each once
  auto removed = [&](auto f) {
    if (MODE != kTarget || !st.tested) return;
    for (int i = node + 1 + tid; i < n; i += kDrawThreads)
      if (p.parents[begin + i] == node && p.removed[begin + i] >= 0) f(p.removed[begin + i]);
  };
  if (MODE == kTarget && st.tested) {
    // (in multiples of 2^-60, so that their order does not matter; below 1e-13 of a part's mass its own sum and theirs are
    // rounding, and a part that lost everything must keep nothing)
    removed([&](int tok) { atomicAdd(&gone_s[(tok + rd.shift) / p.part], (unsigned long long)(chance(rd.at(p, tok)) * 0x1p60 + 0.5)); });
    __syncthreads();
    const double kept = whole - (double)gone_s[lane] * 0x1p-60;
    mass = gone_s[lane] && !(kept > whole * 1e-13) ? 0.0 : kept;
  }
  mass = fmax(mass, 0.0);
  double sums = wave_scan_f64(mass), total = read_lane_f64(sums, 63);
  // Rejections that leave nothing (a target equal to the draft's, or smaller everywhere that it is kept, up to rounding):
  // the last token comes from the target itself.
  bool nothing = !(total > 1e-13);
  if (nothing) {
    mass = whole;
    sums = wave_scan_f64(mass);
    total = read_lane_f64(sums, 63);
  }
  const double want = (double)uniform * total;
  const uint64_t beyond = __builtin_amdgcn_ballot_w64(sums > want && mass > 0.0);
  const uint64_t some = __builtin_amdgcn_ballot_w64(mass > total * 1e-18);   // (the sum's own rounding: the last part that has any)
  uint64_t alive = __builtin_amdgcn_ballot_w64(mass > 0.0);                  // parts that have not been looked through in vain
  int part = beyond ? __builtin_ctzll(beyond) : some ? 63 - __builtin_clzll(some) : 0, token = 0;
  double rest = beyond ? want - read_lane_f64(sums - mass, part) : want;
  const uint8_t* qr = MODE == kDraft ? p.draft + (int64_t)st.row * p.draft_stride : nullptr;
  // Once, but for a part whose mass was rounding after all: then the next part's first token, or the last one before.  (All
  // wavefronts hold the same masses and go the same way.)
  for (;;) {
    const int first = part * p.part - rd.shift;
    const bool minus = MODE == kDraft && st.c != 0 && !nothing;
    if (MODE == kTarget && !nothing) {
      removed([&](int tok) {
        const int i = tok - first;
        if (i >= 0 && i < p.part) atomicOr(&gone[i >> 5], 1u << (i & 31));
      });
      __syncthreads();
    }
    double weight[8], mine = 0;
    const int at = 8 * tid;
#pragma unroll
    for (int j = 0; j < 8; ++j) weight[j] = 0;
    if (at < p.part) {
      VerifyLine<DT> px;
      VerifyAnyLine qx;
      px.fetch(rd.row, first + at, p.V);
      if (minus) qx.fetch(qr, p.draft_dtype, first + at, p.V);
      float x[8], y[8];
      px.values(rd.row, first + at, p.V, -INFINITY, x);
      if (minus) qx.values(qr, p.draft_dtype, first + at, p.V, 0.f, y);
      const uint32_t out = MODE == kTarget ? gone[at >> 5] >> (at & 31) : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        double w = chance(rd.finish(p, x[j]));
        if (minus) w = fmax(w - st.c * (double)y[j], 0.0);
        if (MODE == kTarget && (out >> j & 1)) w = 0;
        weight[j] = w;
        mine += w;
      }
    }
    const double upto = wave_scan_f64(mine);
    if (lane == 63) run[wave] = upto;
    __syncthreads();
    double sum = upto - mine;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += w < wave ? run[w] : 0.0;
    int last = -1, place = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      sum += weight[j];
      if (weight[j] > 0) {
        last = at + j;
        if (sum > rest && place == 0x7fffffff) place = at + j;
      }
    }
    if (place != 0x7fffffff) atomicMin(&found[0], place);
    if (last >= 0) atomicMax(&found[1], last);
    __syncthreads();
    if (found[1] >= 0) {
      token = first + (found[0] != 0x7fffffff ? found[0] : found[1]);
      break;
    }
    alive &= ~((uint64_t)1 << part);
    if (!alive && !nothing) {
      nothing = true;
      alive = __builtin_amdgcn_ballot_w64(whole > 0.0);
      part = -1;
    }
    if (!alive) break;   // (no logit reaches the cut: token 0)
    const uint64_t above = part < 0 ? alive : part < 63 ? alive >> (part + 1) << (part + 1) : 0;
    rest = above ? -1.0 : INFINITY;
    part = above ? __builtin_ctzll(above) : 63 - __builtin_clzll(alive);
    // (nothing was found, by nobody: `found` is as it was)
    if (MODE == kTarget) {
      for (int i = tid; i < kVerifyPart / 32; i += kDrawThreads) gone[i] = 0;
      __syncthreads();
    }
  }
  if (tid == 0) p.out_tokens[(int64_t)r * p.max_path + count - 1] = token;
}

// ------------------------------------------------------------------------------------------------ the cache afterwards
struct KeepParams {
  uint8_t* kc; uint8_t* vc;
  int64_t layer_bytes, chunk_bytes; int64_t tok_bytes;
  const float* k_scale; const float* v_scale; int64_t scale_layer;
  const int32_t* bt; int64_t bt_stride;
  const int32_t* rows; int64_t rows_stride;
  const int32_t* counts; const int32_t* cu; const int32_t* lens;
  int32_t* new_lens;
  int32_t columns, chunk, n_chunks, table_cols, units, units_per_head, Hkv;
};

constexpr int kKeepBatch = 64;   // path entries whose places lie in LDS at a time
constexpr int kKeepLoads = 8;    // rows in flight per thread

// One workgroup per request, layer and cache: the accepted nodes' rows move to where the path puts them.  A path rises, so
// node path[i] >= i lies at or behind its place i, and a place never lies on a node that a later entry still needs:
// a thread reads a few rows of its 16-byte column, then writes them, from the front of the path to its end.
// Bound by the launch and three dependent trips: 4.5 us for one request's 32 layers, 9.0 for 64 requests' (28.6 MB read and written, 4.3 us at 6.7 TB/s).
template <bool FP8>
__global__ __launch_bounds__(256) void kv_keep_kernel(KeepParams p) {
  __shared__ int src_chunk[kKeepBatch], dst_chunk[kKeepBatch];   // -1: nothing moves
  __shared__ int src_pos[kKeepBatch], dst_pos[kKeepBatch];
  const int r = blockIdx.x, layer = blockIdx.y, tid = threadIdx.x;
  const bool value = blockIdx.z != 0;
  const int begin = p.cu[r], n = max(p.cu[r + 1] - begin, 0), len = p.lens[r];
  const int count = min(max(p.counts[r], 0), p.columns);
  if (layer == 0 && !value && tid == 0) p.new_lens[r] = len - n + count;
  uint8_t* const cache = (value ? p.vc : p.kc) + (int64_t)layer * p.layer_bytes;
  const float* const scale = FP8 ? (value ? p.v_scale : p.k_scale) + (int64_t)layer * p.scale_layer : nullptr;
  const int64_t first = (int64_t)len - n, most = (int64_t)p.table_cols * p.chunk;
  for (int base = 1; base < count; base += kKeepBatch) {
    __syncthreads();
    const int m = min(kKeepBatch, count - base);
    int any = 0;
    if (tid < m) {
      const int i = base + tid, node = p.rows[(int64_t)r * p.rows_stride + i] - begin;
      const int64_t from = first + node, to = first + i;
      int a = -1, b = -1;
      if (node >= 0 && node < n && node != i && from >= 0 && from < most && to >= 0 && to < most) {
        a = p.bt[(int64_t)r * p.bt_stride + from / p.chunk];
        b = p.bt[(int64_t)r * p.bt_stride + to / p.chunk];
        if ((uint32_t)a >= (uint32_t)p.n_chunks || (uint32_t)b >= (uint32_t)p.n_chunks) a = b = -1;
      }
      src_chunk[tid] = a;
      dst_chunk[tid] = b;
      src_pos[tid] = (int)(from % p.chunk);
      dst_pos[tid] = (int)(to % p.chunk);
      any = a >= 0;
    }
    if (!__syncthreads_or(any)) continue;
    for (int u = tid; u < p.units; u += blockDim.x) {
      const int head = FP8 ? u / p.units_per_head : 0;
      for (int i0 = 0; i0 < m; i0 += kKeepLoads) {
        uint4 x[kKeepLoads];
#pragma unroll
        for (int j = 0; j < kKeepLoads; ++j)
          if (i0 + j < m && src_chunk[i0 + j] >= 0)
            x[j] = ld16(cache + src_chunk[i0 + j] * p.chunk_bytes + src_pos[i0 + j] * p.tok_bytes + 16 * u);
#pragma unroll
        for (int j = 0; j < kKeepLoads; ++j) {
          if (i0 + j >= m || src_chunk[i0 + j] < 0) continue;
          const int a = src_chunk[i0 + j], b = dst_chunk[i0 + j];
          uint4 y = x[j];
          if (FP8 && a != b) {   // another chunk, another scale: e4m3 of value * scale / scale, saturating; NaN stays NaN
            const float f = scale[(int64_t)a * p.Hkv + head] / scale[(int64_t)b * p.Hkv + head];
            auto moved = [&](float x, uint32_t code) {
              const float v = x * f;
              return v == v ? f32_to_e4m3_sat(v) : (code & 0x80u) | 0x7fu;
            };
            uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const f32x2_t lo = fp8x2_lo_to_f32(w[k]), hi = fp8x2_hi_to_f32(w[k]);
              w[k] = moved(lo.x, w[k]) | moved(lo.y, w[k] >> 8) << 8 | moved(hi.x, w[k] >> 16) << 16 | moved(hi.y, w[k] >> 24) << 24;
            }
            y = make_uint4(w[0], w[1], w[2], w[3]);
          }
          st16(cache + b * p.chunk_bytes + dst_pos[i0 + j] * p.tok_bytes + 16 * u, y);
        }
      }
    }
  }
}

static int64_t align256(int64_t n) { return (n + 255) & ~(int64_t)255; }

// Parts of a row: enough workgroups to fill the chip, no fewer than 2 048 elements each, no more than kVerifyPart.
static void verify_parts(int T, int V, int* parts, int* part) {
  const int64_t places = (int64_t)V + 7;   // (with the shift of a row that does not start at a 16-byte line)
  int64_t n = (places + kVerifyPart - 1) / kVerifyPart;
  const int64_t wish = 2048 / (T > 0 ? T : 1) + 1;
  if (n < wish) n = wish;
  if (n > places / 2048 + 1) n = places / 2048 + 1;
  if (n > kVerifyMostParts) n = kVerifyMostParts;
  const int64_t size = ((places + n - 1) / n + 7) & ~(int64_t)7;
  *part = (int)size;
  *parts = (int)((places + size - 1) / size);
}

}  // namespace mi

using namespace mi;

extern "C" int64_t mi_verify_workspace_bytes(int32_t T, int32_t R, int32_t vocab) {
  if (T < 0 || R <= 0 || vocab <= 0 || vocab > kVerifyMostParts * kVerifyPart - 8) return 0;
  int parts, part;
  verify_parts(T, vocab, &parts, &part);
  return align256((int64_t)T * parts * sizeof(VerifyPartial)) + align256((int64_t)R * parts * sizeof(double)) +
         align256((int64_t)R * sizeof(VerifyState)) + align256((int64_t)T * sizeof(int32_t));
}

template <int DT>
static void launch_verify(const VerifyParams& p, int mode, hipStream_t st) {
  const dim3 grid(p.T, p.parts), block(kVerifyThreads);
  if (mode == kGreedy) {
    if (p.T) hipLaunchKernelGGL((verify_rows_kernel<DT, true>), grid, block, 0, st, p);
    hipLaunchKernelGGL((verify_walk_kernel<DT, kGreedy>), dim3(p.R), dim3(kWalkThreads), 0, st, p);
    return;
  }
  if (p.T) hipLaunchKernelGGL((verify_rows_kernel<DT, false>), grid, block, 0, st, p);
  if (mode == kTarget) {
    hipLaunchKernelGGL((verify_walk_kernel<DT, kTarget>), dim3(p.R), dim3(kWalkThreads), 0, st, p);
    hipLaunchKernelGGL((verify_draw_kernel<DT, kTarget>), dim3(p.R), dim3(kDrawThreads), 0, st, p);
  } else {
    hipLaunchKernelGGL((verify_walk_kernel<DT, kDraft>), dim3(p.R), dim3(kWalkThreads), 0, st, p);
    hipLaunchKernelGGL((verify_left_kernel<DT>), dim3(p.R, p.parts), block, 0, st, p);
    hipLaunchKernelGGL((verify_draw_kernel<DT, kDraft>), dim3(p.R), dim3(kDrawThreads), 0, st, p);
  }
}

extern "C" int mi_verify_drafted_tokens(const void* logits, int64_t stride_row, int32_t logits_dtype, int32_t T,
                                        int32_t vocab, const int64_t* tokens, const int32_t* parents,
                                        const int32_t* cu_seqlens_q, int32_t R, int32_t max_path, int32_t greedy,
                                        const void* draft_probs, int64_t draft_stride_row, int32_t draft_dtype,
                                        const float* uniform, float temperature, const float* cut,
                                        int64_t* out_tokens, int32_t* out_rows, int32_t* out_counts, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
  if (R == 0) return MI_OK;
  if (!cu_seqlens_q || !out_tokens || !out_rows || !out_counts)
    return mi_fail(MI_ERR_NULL, "mi_verify_drafted_tokens: null pointer argument");
  if (T > 0 && (!logits || !tokens || !parents)) return mi_fail(MI_ERR_NULL, "mi_verify_drafted_tokens: null pointer argument");
  if (T < 0 || R < 0 || max_path < 1)
    return mi_fail(MI_ERR_SHAPE, "mi_verify_drafted_tokens: need T >= 0, R >= 0 and max_path >= 1");
  if (vocab <= 0 || stride_row < vocab || vocab > kVerifyMostParts * kVerifyPart - 8)
    return mi_fail(MI_ERR_SHAPE, "mi_verify_drafted_tokens: need 0 < vocab <= 524280 and a row stride of at least vocab");
  if (logits_dtype < 0 || logits_dtype > 2 || draft_dtype < 0 || draft_dtype > 2)
    return mi_fail(MI_ERR_UNSUPPORTED, "mi_verify_drafted_tokens: logits and draft_probs must be fp32 (0), bf16 (1) or fp16 (2)");
  if (greedy && (draft_probs || cut)) return mi_fail(MI_ERR_SHAPE, "mi_verify_drafted_tokens: a greedy call takes neither draft_probs nor cut");
  if (!greedy && T > 0 && !uniform) return mi_fail(MI_ERR_NULL, "mi_verify_drafted_tokens: sampling needs one uniform number per row");
  if (!greedy && !(temperature > 0.f)) return mi_fail(MI_ERR_SHAPE, "mi_verify_drafted_tokens: temperature must be positive");
  if (draft_probs && draft_stride_row < vocab)
    return mi_fail(MI_ERR_SHAPE, "mi_verify_drafted_tokens: draft_probs need a row stride of at least vocab");
  const int esz = logits_dtype ? 2 : 4, dsz = draft_dtype ? 2 : 4;
  if (((uintptr_t)logits & (esz - 1)) || ((uintptr_t)draft_probs & (dsz - 1)))
    return mi_fail(MI_ERR_ALIGN, "mi_verify_drafted_tokens: rows must be aligned to their elements");
  if (!workspace || workspace_bytes < mi_verify_workspace_bytes(T, R, vocab))
    return mi_fail(MI_ERR_WORKSPACE, "mi_verify_drafted_tokens: workspace smaller than mi_verify_workspace_bytes()");
  if ((uintptr_t)workspace & 15) return mi_fail(MI_ERR_ALIGN, "mi_verify_drafted_tokens: the workspace must be 16-byte aligned");
  VerifyParams p;
  p.logits = (const uint8_t*)logits; p.stride = stride_row * esz;
  p.draft = (const uint8_t*)draft_probs; p.draft_stride = draft_stride_row * dsz; p.draft_dtype = draft_dtype;
  p.tokens = tokens; p.parents = parents; p.cu = cu_seqlens_q; p.uniform = uniform; p.cut = cut;
  p.out_tokens = out_tokens; p.out_rows = out_rows; p.out_counts = out_counts;
  p.T = T; p.R = R; p.V = vocab; p.max_path = max_path;
  verify_parts(T, vocab, &p.parts, &p.part);
  uint8_t* ws = (uint8_t*)workspace;
  p.partial = (VerifyPartial*)ws;
  ws += align256((int64_t)T * p.parts * sizeof(VerifyPartial));
  p.residual = (double*)ws;
  ws += align256((int64_t)R * p.parts * sizeof(double));
  p.state = (VerifyState*)ws;
  ws += align256((int64_t)R * sizeof(VerifyState));
  p.removed = (int32_t*)ws;
  p.scaled = !greedy && temperature != 1.f;
  p.inv_temperature = greedy ? 1.f : 1.f / temperature;
  const int mode = greedy ? kGreedy : draft_probs ? kDraft : kTarget;
  hipStream_t st = (hipStream_t)stream;
  if (logits_dtype == 0) launch_verify<0>(p, mode, st);
  else if (logits_dtype == 1) launch_verify<1>(p, mode, st);
  else launch_verify<2>(p, mode, st);
  return mi_check_launch("mi_verify_drafted_tokens");
}

extern "C" int mi_kv_keep_accepted(void* k_cache, void* v_cache, int64_t kv_stride_layer, int64_t kv_stride_chunk,
                                   int64_t kv_stride_tok, int32_t layers, int32_t n_chunks, int32_t chunk_tokens,
                                   int32_t Hkv, int32_t head_dim, int32_t elem_bytes, const float* k_scales,
                                   const float* v_scales, int64_t scale_stride_layer, const int32_t* block_table,
                                   int64_t bt_stride, int32_t table_columns, const int32_t* rows, int64_t rows_stride,
                                   int32_t columns, const int32_t* counts, const int32_t* cu_seqlens_q,
                                   const int32_t* kv_lens, int32_t* new_kv_lens, int32_t R, void* stream) {
  if (R == 0) return MI_OK;
  if (!k_cache || !block_table || !rows || !counts || !cu_seqlens_q || !kv_lens || !new_kv_lens)
    return mi_fail(MI_ERR_NULL, "mi_kv_keep_accepted: null pointer argument");
  if (R < 0 || layers <= 0 || layers > 65535 || n_chunks <= 0 || chunk_tokens <= 0 || Hkv <= 0 || head_dim <= 0 || columns < 0 || table_columns <= 0)
    return mi_fail(MI_ERR_SHAPE, "mi_kv_keep_accepted: bad sizes");
  if (elem_bytes != 1 && elem_bytes != 2) return mi_fail(MI_ERR_UNSUPPORTED, "mi_kv_keep_accepted: elements of 1 or 2 bytes");
  const bool fp8 = k_scales || v_scales;
  if (fp8 && (elem_bytes != 1 || !k_scales || !v_scales || !v_cache))
    return mi_fail(MI_ERR_SHAPE, "mi_kv_keep_accepted: scales belong to both caches of bytes");
  if (elem_bytes == 1 && !fp8) return mi_fail(MI_ERR_NULL, "mi_kv_keep_accepted: a cache of bytes needs k_scales and v_scales");
  const int64_t row = (int64_t)Hkv * head_dim * elem_bytes;
  if (row % 16 || (fp8 && head_dim % 16))
    return mi_fail(MI_ERR_ALIGN, "mi_kv_keep_accepted: token rows (of an fp8 cache: heads) must be whole 16-byte pieces");
  if ((((uintptr_t)k_cache | (uintptr_t)v_cache) & 15) || ((kv_stride_layer | kv_stride_chunk | kv_stride_tok) * elem_bytes) % 16)
    return mi_fail(MI_ERR_ALIGN, "mi_kv_keep_accepted: caches and strides must keep rows 16-byte aligned");
  KeepParams p;
  p.kc = (uint8_t*)k_cache; p.vc = (uint8_t*)v_cache;
  p.layer_bytes = kv_stride_layer * elem_bytes; p.chunk_bytes = kv_stride_chunk * elem_bytes; p.tok_bytes = kv_stride_tok * elem_bytes;
  p.k_scale = k_scales; p.v_scale = v_scales; p.scale_layer = scale_stride_layer;
  p.bt = block_table; p.bt_stride = bt_stride; p.rows = rows; p.rows_stride = rows_stride; p.counts = counts;
  p.cu = cu_seqlens_q; p.lens = kv_lens; p.new_lens = new_kv_lens;
  p.columns = columns; p.chunk = chunk_tokens; p.n_chunks = n_chunks; p.table_cols = table_columns;
  p.units = (int)(row / 16); p.units_per_head = head_dim * elem_bytes / 16; p.Hkv = Hkv;
  const dim3 grid(R, layers, v_cache ? 2 : 1), block(p.units <= 64 ? 64 : p.units <= 128 ? 128 : 256);
  hipStream_t st = (hipStream_t)stream;
  if (fp8) hipLaunchKernelGGL((kv_keep_kernel<true>), grid, block, 0, st, p);
  else hipLaunchKernelGGL((kv_keep_kernel<false>), grid, block, 0, st, p);
  return mi_check_launch("mi_kv_keep_accepted");
}
