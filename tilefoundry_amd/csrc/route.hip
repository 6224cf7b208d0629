// The choice of experts: scores, a bias for the choice, groups, top k, weights.
#include "host_common.h"
#include "decode_common.h"
#include "tf_mx4.h"

using namespace tfd;
using namespace tfd_host;

namespace {

// ---------------------------------------------------------------------------
// A wave per row; lane l holds experts l, l + 64, ...  Scores and choices are
// 64-bit: biased scores of different experts lie as close as an f32 rounding often
// enough to settle a choice by it.  Groups: a power of two of lanes per group walks
// it for its two best choices; a group's rank is the number of groups before it.
// Picks: k rounds of a wave's best (value, then lower index) of the lanes' sorted
// choices, as integers in their order: the upper halves' maximum almost always leaves
// one lane, the lower halves and the index settle the rest.  Reductions stay in registers
// (DPP and lane swaps).
// Bound: at one row the launch and the chain of k wave maxima, at thousands of rows the
// 64-bit exponentials' and the rounds' VALU operations; the logits are read once.  256
// experts, 8 picks: one row 4.1 us, 4,001 rows in 8 groups 9.5 us.
// ---------------------------------------------------------------------------
constexpr double kNone = -__builtin_huge_val();

__device__ __forceinline__ uint32_t lo32(double v) {
  return (uint32_t)__builtin_bit_cast(uint64_t, v);
}
__device__ __forceinline__ uint32_t hi32(double v) {
  return (uint32_t)(__builtin_bit_cast(uint64_t, v) >> 32);
}
__device__ __forceinline__ double both(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double from_lane_d(double v, int lane) {
  return both(__builtin_amdgcn_readlane(lo32(v), lane), __builtin_amdgcn_readlane(hi32(v), lane));
}

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  v = max(v, dpp_u<kDppXor1>(v));
  v = max(v, dpp_u<kDppXor2>(v));
  v = max(v, dpp_u<kDppHalfMirror>(v));
  v = max(v, dpp_u<kDppMirror>(v));
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(b[0], b[1]);
}
template <int kCtrl>
__device__ __forceinline__ double dpp_d(double v) {
  return both(dpp_u<kCtrl>(lo32(v)), dpp_u<kCtrl>(hi32(v)));
}
__device__ __forceinline__ double wave_sum_d(double v) {
  v += dpp_d<kDppXor1>(v);
  v += dpp_d<kDppXor2>(v);
  v += dpp_d<kDppHalfMirror>(v);
  v += dpp_d<kDppMirror>(v);
  const auto l = __builtin_amdgcn_permlane16_swap(lo32(v), lo32(v), false, false);
  const auto h = __builtin_amdgcn_permlane16_swap(hi32(v), hi32(v), false, false);
  v = both(l[0], h[0]) + both(l[1], h[1]);
  const auto m = __builtin_amdgcn_permlane32_swap(lo32(v), lo32(v), false, false);
  const auto n = __builtin_amdgcn_permlane32_swap(hi32(v), hi32(v), false, false);
  return both(m[0], n[0]) + both(m[1], n[1]);
}
__device__ __forceinline__ double xor_d(double v, int mask) {
  return both(__shfl_xor(lo32(v), mask, kWave), __shfl_xor(hi32(v), mask, kWave));
}

// A double as an integer in the doubles' order (no NaN comes here; -0 before +0 is put
// right by adding a zero).
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v + 0.0);
  return b >> 63 ? ~b : b | (1ull << 63);
}

template <int kPer>
__global__ __launch_bounds__(kBlock) void k_route_experts(TfdRouteArgs a) {
  __shared__ double c_s[kWavesPerBlock][kPer * kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int row = blockIdx.x * kWavesPerBlock + wave;
  if (row >= a.rows) return;
  const int E = a.experts;
  double l[kPer], s[kPer], c[kPer];
  // every load before a use (past the experts: the last one again)
  float v[kPer], bias[kPer];
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) bias[j] = a.bias[min(lane + kWave * j, E - 1)];
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) bias[j] = 0.f;
  }
  const int64_t first = (int64_t)row * a.ldl;
  if (a.type == TFD_TYPE_F32) {
    const float* p = (const float*)a.logits + first;
#pragma unroll
    for (int j = 0; j < kPer; ++j) v[j] = p[min(lane + kWave * j, E - 1)];
  } else {
    const uint16_t* p = (const uint16_t*)a.logits + first;
    uint16_t h[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) h[j] = p[min(lane + kWave * j, E - 1)];
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      v[j] = a.type == TFD_TYPE_BF16 ? bf2f(h[j]) : (float)__builtin_bit_cast(_Float16, h[j]);
  }
  float top = -__builtin_huge_valf();
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const bool in = lane + kWave * j < E && v[j] == v[j];
    l[j] = in ? (double)v[j] : kNone;                // NaN: as masked
    top = fmaxf(top, (float)l[j]);
  }
  if (a.score == TFD_SCORE_SOFTMAX) {
    const double m = (double)wave_max(top);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      // equal to the largest: one, infinities too; masked: nothing
      s[j] = l[j] == kNone ? 0.0 : l[j] == m ? 1.0 : exp(l[j] - m);
      sum += s[j];
    }
    // (the largest's is one: a sum of zero has nothing to share)
    const double all = wave_sum_d(sum), inv = all > 0.0 ? 1.0 / all : 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) s[j] *= inv;
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) s[j] = 1.0 / (1.0 + exp(-l[j]));
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const double b = (double)bias[j];
    c[j] = l[j] == kNone || b != b ? kNone : s[j] + b;
  }
  if (a.kept_groups < a.groups) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) c_s[wave][lane + kWave * j] = c[j];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int per = E / a.groups;
    int sh = 0;                                      // of lanes per group
    while ((2 << sh) * a.groups <= kWave) ++sh;
    const int L = 1 << sh, g = lane >> sh;
    double b1 = kNone, b2 = kNone;
    if (g < a.groups)
      for (int i = lane & (L - 1); i < per; i += L) {
        const double v = c_s[wave][g * per + i];
        b2 = fmax(b2, fmin(b1, v));
        b1 = fmax(b1, v);
      }
    for (int d = 1; d < L; d *= 2) {
      const double o1 = xor_d(b1, d), o2 = xor_d(b2, d);
      b2 = fmax(fmin(b1, o1), fmax(b2, o2));
      b1 = fmax(b1, o1);
    }
    // a group with one expert that can be chosen ranks by it alone
    const double best = a.group_top == 2 && b2 != kNone ? b1 + b2 : b1;
    int rank = 0;
    for (int h = 0; h < a.groups; ++h) {
      const double v = from_lane_d(best, h << sh);
      rank += v > best || (v == best && h < g);
    }
    const uint64_t kept = __ballot(g < a.groups && rank < a.kept_groups);
    // an expert's group: e + 1/2 over `per` lies at least 1/1024 from a whole number, and f32's
    // error under 512 * 2^-22
    const float inv = __builtin_amdgcn_rcpf((float)per);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = lane + kWave * j, group = (int)(((float)e + 0.5f) * inv);
      if (e < E && !((kept >> (group << sh)) & 1)) c[j] = kNone;
    }
  }
  // each lane's keys, largest first (neighbours change places only where the second is
  // larger: equal ones stay by their ids); the scores wait in LDS for the picks
  uint64_t key[kPer];
  int id[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    key[j] = ordered(c[j]);
    id[j] = lane + kWave * j;
    c_s[wave][id[j]] = s[j];
  }
#pragma unroll
  for (int i = kPer - 1; i > 0; --i)
#pragma unroll
    for (int j = 0; j < i; ++j) {
      const bool swap = key[j + 1] > key[j];
      const uint64_t k0 = key[j], k1 = key[j + 1];
      const int i0 = id[j], i1 = id[j + 1];
      key[j] = swap ? k1 : k0, key[j + 1] = swap ? k0 : k1;
      id[j] = swap ? i1 : i0, id[j + 1] = swap ? i0 : i1;
    }
  const uint64_t none = ordered(kNone);
  int my_id = -1;
  for (int r = 0; r < a.k; ++r) {
    const uint32_t hi = (uint32_t)(key[0] >> 32), lo = (uint32_t)key[0];
    const uint32_t mh = __builtin_amdgcn_readfirstlane(wave_max_u(hi));
    // nothing left that can be chosen (no finite value shares this half)
    if (mh == (uint32_t)(none >> 32)) break;
    uint64_t who = __ballot(hi == mh);
    if (__popcll(who) > 1) {
      const uint32_t ml = wave_max_u(hi == mh ? lo : 0u);
      who = __ballot(hi == mh && lo == ml);
      if (__popcll(who) > 1) {
        // the same value: the lowest id (as the largest of complements)
        const bool in = (who >> lane) & 1;
        const uint32_t other = ~(uint32_t)id[0];
        const uint32_t mi = wave_max_u(in ? other : 0u);
        who = __ballot(in && other == mi);
      }
    }
    const int owner = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(who));
    const int pick = __builtin_amdgcn_readlane(id[0], owner);
    if (lane == owner) {
#pragma unroll
      for (int j = 0; j + 1 < kPer; ++j) key[j] = key[j + 1], id[j] = id[j + 1];
      key[kPer - 1] = none;
    }
    if (lane == r) my_id = pick;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  const double my_s = my_id >= 0 ? c_s[wave][my_id] : 0.0;
  const double total = wave_sum_d(my_s);
  if (lane < a.k + a.shared) {
    double w = my_s * (double)a.scale;
    if (a.renormalise) w = total > 0.0 ? my_s / total * (double)a.scale : 0.0;
    const bool extra = lane >= a.k;
    a.weights[(int64_t)row * a.ld + lane] = extra ? 1.f : (float)w;
    a.ids[(int64_t)row * a.ld + lane] = extra ? E + lane - a.k : my_id;
  }
}

// Threads of one launch, in whole blocks, have 32 bits.
constexpr int kMaxRows = kWavesPerBlock * (int)((((int64_t)1 << 32) - kBlock) / kBlock);

}  // namespace

extern "C" int tfd_route_experts(const TfdRouteArgs* args, void* stream) {
  if (!args) return fail(kBadArg, "route_experts: null args");
  const TfdRouteArgs& a = *args;
  if (a.type != TFD_TYPE_F32 && a.type != TFD_TYPE_BF16 && a.type != TFD_TYPE_F16)
    return fail(kBadArg, "route_experts: type %d", a.type);
  if (a.score != TFD_SCORE_SOFTMAX && a.score != TFD_SCORE_SIGMOID)
    return fail(kBadArg, "route_experts: score %d", a.score);
  if (a.experts < 1 || a.experts > TFD_ROUTE_MAX_EXPERTS || a.rows < 0 || a.rows > kMaxRows)
    return fail(kBadShape, "route_experts: rows=%d (0..%d) experts=%d (1..%d)", a.rows, kMaxRows,
                a.experts, TFD_ROUTE_MAX_EXPERTS);
  if (a.groups < 1 || a.groups > kWave || a.experts % a.groups || a.kept_groups < 1 ||
      a.kept_groups > a.groups || (a.group_top != 1 && a.group_top != 2))
    return fail(kBadShape, "route_experts: %d experts in %d groups, %d kept by their best %d",
                a.experts, a.groups, a.kept_groups, a.group_top);
  if (a.k < 1 || a.shared < 0 || a.k > kWave || a.shared > kWave - a.k ||
      a.k > a.kept_groups * (a.experts / a.groups))
    return fail(kBadShape, "route_experts: k=%d shared=%d of %d experts that stay", a.k, a.shared,
                a.kept_groups * (a.experts / a.groups));
  if (!(a.scale > 0.f) || a.scale > 3.402823466e38f)
    return fail(kBadArg, "route_experts: scale must be positive and finite");
  if (a.rows == 0) return 0;
  if (!a.logits || !a.weights || !a.ids) return fail(kBadArg, "route_experts: null pointer");
  if ((a.rows > 1 && a.ldl < a.experts) || a.ld < a.k + a.shared)
    return fail(kBadArg, "route_experts: ldl=%lld ld=%d", (long long)a.ldl, a.ld);
  if ((uintptr_t)a.logits % (a.type == TFD_TYPE_F32 ? 4 : 2) || (uintptr_t)a.bias % 4)
    return fail(kBadArg, "route_experts: logits or bias not aligned to its elements");
  const int grid = (a.rows + kWavesPerBlock - 1) / kWavesPerBlock;
  hipStream_t s = (hipStream_t)stream;
  const int per = (a.experts + kWave - 1) / kWave;
  if (per <= 1) k_route_experts<1><<<grid, kBlock, 0, s>>>(a);
  else if (per <= 2) k_route_experts<2><<<grid, kBlock, 0, s>>>(a);
  else if (per <= 4) k_route_experts<4><<<grid, kBlock, 0, s>>>(a);
  else k_route_experts<8><<<grid, kBlock, 0, s>>>(a);
  return launched("route_experts");
}
