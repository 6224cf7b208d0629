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
// Picks: k rounds of a wave's best (value, then lower index).
// Bound: at one row the chain of k wave reductions, at thousands of rows the
// 64-bit exponentials and reductions' VALU operations; the logits themselves are
// read once.
// ---------------------------------------------------------------------------
constexpr double kNone = -__builtin_huge_val();

__device__ __forceinline__ double xor_d(double v, int mask) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __shfl_xor((uint32_t)b, mask, kWave);
  const uint32_t hi = __shfl_xor((uint32_t)(b >> 32), mask, kWave);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double from_lane_d(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)b, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ float logit(const TfdRouteArgs& a, int64_t at) {
  if (a.type == TFD_TYPE_F32) return ((const float*)a.logits)[at];
  const uint16_t b = ((const uint16_t*)a.logits)[at];
  if (a.type == TFD_TYPE_BF16) return bf2f(b);
  return (float)__builtin_bit_cast(_Float16, b);
}

template <int kPer>
__global__ __launch_bounds__(kBlock) void k_route_experts(TfdRouteArgs a) {
  __shared__ double c_s[kWavesPerBlock][kPer * kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int row = blockIdx.x * kWavesPerBlock + wave;
  if (row >= a.rows) return;
  const int E = a.experts;
  double l[kPer], s[kPer], c[kPer];
  double m = kNone;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + kWave * j;
    const float v = e < E ? logit(a, (int64_t)row * a.ldl + e) : -__builtin_huge_valf();
    l[j] = v != v ? kNone : (double)v;               // NaN: as masked
    m = fmax(m, l[j]);
  }
  if (a.score == TFD_SCORE_SOFTMAX) {
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) m = fmax(m, xor_d(m, d));
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      // equal to the largest: one, infinities too; masked: nothing
      s[j] = l[j] == kNone ? 0.0 : l[j] == m ? 1.0 : exp(l[j] - m);
      sum += s[j];
    }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) sum += xor_d(sum, d);
#pragma unroll
    for (int j = 0; j < kPer; ++j) s[j] = sum > 0.0 ? s[j] / sum : 0.0;
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) s[j] = 1.0 / (1.0 + exp(-l[j]));
  }
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = lane + kWave * j;
    const double b = a.bias && e < E ? (double)a.bias[e] : 0.0;
    c[j] = l[j] == kNone || b != b ? kNone : s[j] + b;
  }
  if (a.kept_groups < a.groups) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) c_s[wave][lane + kWave * j] = c[j];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const int per = E / a.groups;
    int L = 1;                                       // lanes per group
    while (2 * L * a.groups <= kWave) L *= 2;
    const int g = lane / L;
    double b1 = kNone, b2 = kNone;
    if (g < a.groups)
      for (int i = lane % L; i < per; i += L) {
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
      const double v = from_lane_d(best, h * L);
      rank += v > best || (v == best && h < g);
    }
    const uint64_t kept = __ballot(g < a.groups && rank < a.kept_groups);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = lane + kWave * j;
      if (e < E && !((kept >> (e / per * L)) & 1)) c[j] = kNone;
    }
  }
  double my_s = 0.0, total = 0.0;
  int my_id = -1;
  for (int r = 0; r < a.k; ++r) {
    // this lane's best, then the wave's: the larger choice, equal ones the lower id
    double bc = c[0], bs = s[0];
    int bi = lane;
#pragma unroll
    for (int j = 1; j < kPer; ++j)
      if (c[j] > bc) {
        bc = c[j];
        bs = s[j];
        bi = lane + kWave * j;
      }
#pragma unroll
    for (int d = 1; d < kWave; d *= 2) {
      const double oc = xor_d(bc, d);
      const int oi = __shfl_xor(bi, d, kWave);
      if (oc > bc || (oc == bc && oi < bi)) {
        bc = oc;
        bi = oi;
      }
    }
    if (bc == kNone) break;                          // nothing left that can be chosen
    const int owner = bi & (kWave - 1);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
      if (bi == lane + kWave * j) {
        bs = s[j];
        c[j] = kNone;
      }
    bs = from_lane_d(bs, __builtin_amdgcn_readfirstlane(owner));
    total += bs;
    if (lane == r) {
      my_s = bs;
      my_id = bi;
    }
  }
  if (lane < a.k + a.shared) {
    double w = my_s * (double)a.scale;
    if (a.renormalise) w = total > 0.0 ? my_s / total * (double)a.scale : 0.0;
    const bool extra = lane >= a.k;
    a.weights[(int64_t)row * a.ld + lane] = extra ? 1.f : (float)w;
    a.ids[(int64_t)row * a.ld + lane] = extra ? E + lane - a.k : my_id;
  }
}

}  // namespace

extern "C" int tfd_route_experts(const TfdRouteArgs* args, void* stream) {
  if (!args) return fail(kBadArg, "route_experts: null args");
  const TfdRouteArgs& a = *args;
  if (a.type != TFD_TYPE_F32 && a.type != TFD_TYPE_BF16 && a.type != TFD_TYPE_F16)
    return fail(kBadArg, "route_experts: type %d", a.type);
  if (a.score != TFD_SCORE_SOFTMAX && a.score != TFD_SCORE_SIGMOID)
    return fail(kBadArg, "route_experts: score %d", a.score);
  if (a.experts < 1 || a.experts > TFD_ROUTE_MAX_EXPERTS || a.rows < 0)
    return fail(kBadShape, "route_experts: rows=%d experts=%d (1..%d)", a.rows, a.experts,
                TFD_ROUTE_MAX_EXPERTS);
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
