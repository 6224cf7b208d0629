// Beam search: the best candidates of all beams' next tokens, and rows moved to the rows that
// continue them.
#include "host_common.h"
#include "decode_common.h"
#include "tf_search.h"
#include "tf_mx4.h"

using namespace tfd;
using namespace tfd_host;

namespace {

constexpr int kMaxBeams = TFD_BEAM_MAX;
constexpr double kNone = -__builtin_huge_val();

// A logit and its token as one integer in the order of choice: the larger logit, then the
// lower token.  0: no candidate (NaN, -inf).
__device__ __forceinline__ uint64_t key_of(float x, int token) {
  if (!(x > -__builtin_huge_valf())) return 0;
  const uint32_t b = __float_as_uint(x + 0.f);     // (-0 as +0)
  const uint32_t o = b >> 31 ? ~b : b | 0x80000000u;
  return ((uint64_t)o << 32) | (uint32_t)~token;
}
__device__ __forceinline__ float logit_of(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ int token_of(uint64_t key) { return (int)~(uint32_t)key; }

template <int kCtrl>
__device__ __forceinline__ uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, 0xF, 0xF, false);
}
__device__ __forceinline__ double pair_d(uint32_t lo, uint32_t hi) {
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
template <int kCtrl>
__device__ __forceinline__ double dpp_d(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return pair_d(dpp_u<kCtrl>((uint32_t)b), dpp_u<kCtrl>((uint32_t)(b >> 32)));
}
// Sums and conjunctions over a wave, in registers (DPP and lane swaps).
__device__ __forceinline__ double wave_sum_d(double v) {
  v += dpp_d<kDppXor1>(v);
  v += dpp_d<kDppXor2>(v);
  v += dpp_d<kDppHalfMirror>(v);
  v += dpp_d<kDppMirror>(v);
  uint64_t b = __builtin_bit_cast(uint64_t, v);
  const auto l = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false);
  const auto h = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false,
                                                  false);
  v = pair_d(l[0], h[0]) + pair_d(l[1], h[1]);
  b = __builtin_bit_cast(uint64_t, v);
  const auto m = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false);
  const auto n = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false,
                                                  false);
  return pair_d(m[0], n[0]) + pair_d(m[1], n[1]);
}
__device__ __forceinline__ uint32_t wave_and(uint32_t v) {
  v &= dpp_u<kDppXor1>(v);
  v &= dpp_u<kDppXor2>(v);
  v &= dpp_u<kDppHalfMirror>(v);
  v &= dpp_u<kDppMirror>(v);
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  v = a[0] & a[1];
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return __builtin_amdgcn_readfirstlane(b[0] & b[1]);
}

constexpr float kLog2e = 1.44269502162933349609375f;

// 2^(d log2 e) for d <= 0 to about an f32's last bit: log2 e in two parts.
__device__ __forceinline__ float exp_neg(float d) {
  constexpr float kLo = 1.92596303e-8f;
  return __builtin_amdgcn_exp2f(fmaf(d, kLog2e, d * kLo));
}

__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);     // (-0 as +0)
  return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float float_of(uint32_t o) {
  return __uint_as_float(o >> 31 ? o & 0x7fffffffu : ~o);
}

// The largest of three, NaN left out (written out: fmaxf first makes its operands quiet).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

// The largest t that at least k of the lanes' values reach (0: fewer are above 0), bit by bit
// below the bits that all share; it may stop short where exactly k do.
template <int kN>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&v)[kN], int k) {
  uint32_t all = v[0], any = v[0];
#pragma unroll
  for (int i = 1; i < kN; ++i) all &= v[i], any |= v[i];
  all = wave_and(all), any = ~wave_and(~any);
  uint32_t t = 0;
  if (all == any) return all;                // (all equal)
  const uint32_t top = 0x80000000u >> __builtin_clz(all ^ any);
  t = any & ~(2 * top - 1);
#pragma unroll 1
  for (uint32_t bit = top; bit; bit >>= 1) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i) n += __popcll(__ballot(v[i] >= (t | bit)));
    if (n < k) continue;
    t |= bit;
    if (n == k) break;
  }
  return t;
}

// A lane's place behind the n before, of the lanes of `who`.
__device__ __forceinline__ int placed_at(uint64_t who, int n) {
  return n + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32),
                                            __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
}

struct BeamPlan {
  int per, chunks;       // values of a lane, chunks (of a wave) of a row
};

// What a wave holds of its chunk's candidates: values by fours (each four consecutive tokens)
// in which one reaches the bound, and those that do.
constexpr int kFours = 128, kNear = 128, kAtOnce = 8;
typedef float f4 __attribute__((ext_vector_type(4)));
struct alignas(16) Near {
  float x[4 * kFours];
  uint64_t near[kNear + kAtOnce];
  int token[kFours];
};
// Up to so many beams the bound comes from the lanes' best values: that leaves
// 64 ln(64 / (64 - beams)) fours, 30 of 24 beams; above it from all fours' best, which leaves as
// many as there are beams, for one ballot a four and bit.
constexpr int kFewBeams = 24;

// What a wave's chunk of a row leaves: its largest logit, the sum of exp(x - that), and its
// `beams` largest keys in falling order (0 where there are fewer).
struct ChunkSum {
  double sum;
  float top;
  int pad;
};

template <int kType>
__device__ __forceinline__ float logit_at(const void* p, int64_t i) {
  if (kType == TFD_TYPE_F32) return ((const float*)p)[i];
  if (kType == TFD_TYPE_BF16) return bf2f(((const bf16*)p)[i]);
  return (float)__builtin_bit_cast(_Float16, ((const uint16_t*)p)[i]);
}

// ---------------------------------------------------------------------------
// A wave per chunk of a row, its values in registers, no barrier.  The beams-th largest of
// the lanes' best values bounds the chunk's beams-th largest from below: what reaches it,
// hardly more than `beams` values, goes through LDS to be ranked by counting.  Four values at a
// time are tested by their largest and moved together.  Where more do than LDS holds (equal
// logits), the places are filled one by one, from memory.
// ---------------------------------------------------------------------------
template <int kType, int kPer, bool kVec>
__global__ __launch_bounds__(kBlock, kPer == 64 ? 4 : kPer == 32 ? 6 : 8)
void k_beam_scan(TfdBeamArgs a, int chunks, int waves, ChunkSum* __restrict__ sums,
                 uint64_t* __restrict__ lists) {
  constexpr float kInf = __builtin_huge_valf();
  constexpr int kQuads = kPer / 4;
  __shared__ Near near_s[kWavesPerBlock];
  const int lane = threadIdx.x & (kWave - 1);
  const int in_block = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int w = blockIdx.x * kWavesPerBlock + in_block;
  if (w >= waves) return;
  const int row = w / chunks, chunk = w % chunks;
  if (a.done && a.done[row]) return;               // (its lists are not read)
  Near& mine_s = near_s[in_block];
  const int c0 = chunk * kWave * kPer, K = a.beams;
  const int64_t base = (int64_t)row * a.ldl;
  float x[kPer];
  // a lane's values come in runs of kRun, 16 bytes of memory
  constexpr int kRun = kType == TFD_TYPE_F32 ? 4 : 8;
  auto at = [&](int j) { return c0 + (j / kRun) * kRun * kWave + kRun * lane + j % kRun; };
  auto put_run = [&](int j, const u32x4& v) {
#pragma unroll
    for (int e = 0; e < kRun; ++e) {
      if (kType == TFD_TYPE_F32) x[j + e] = __uint_as_float(v[e % 4]);
      else if (kType == TFD_TYPE_BF16) x[j + e] = e % 2 ? bf_hi(v[e / 2]) : bf_lo(v[e / 2]);
      else x[j + e] = (float)__builtin_bit_cast(_Float16, (uint16_t)(v[e / 2] >> (16 * (e % 2))));
    }
  };
  const bool whole = c0 + kWave * kPer <= a.vocab;
  if (kVec && whole) {
    constexpr int kSize = kType == TFD_TYPE_F32 ? 4 : 2;
    const uint8_t* const p = (const uint8_t*)a.logits + (base + c0) * kSize + lane * 16;
#pragma unroll
    for (int j = 0; j < kPer; j += kRun)
      put_run(j, __builtin_nontemporal_load((g_u32x4*)(p + j * kWave * kSize)));
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      x[j] = logit_at<kType>(a.logits, base + min(at(j), a.vocab - 1));
      if (at(j) >= a.vocab) x[j] = -kInf;
    }
  }
  // Largest of four, of the lane, of the wave, and the sum of 2^(x log2 e + c), c = -m log2 e
  // rounded: one fused multiply-add a value, and what c's rounding left out (exactly fma's remainder) is
  // put right in the sum.  log2 e as one f32 is 1.3e-8 of x - m off: 1.1e-7 of a sum over
  // 4,096 equal values, half of an f32's last place at one, where the scores that go out
  // are themselves f32 of at least ln 4096.
  float top4[kQuads], best, m;
  auto tops = [&] {
    best = -kInf;
#pragma unroll
    for (int q = 0; q < kQuads; ++q)
      top4[q] = max3(max3(x[4 * q], x[4 * q + 1], x[4 * q + 2]), x[4 * q + 3], -kInf);
#pragma unroll
    for (int q = 0; q < kQuads; q += 2) best = max3(best, top4[q], top4[q + 1]);
    m = wave_max(best);
  };
  auto added = [&](auto term) {
    double sum = 0.0;
#pragma unroll
    for (int q = 0; q < kQuads; ++q) {
      float e[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[i] = term(x[4 * q + i]);
      sum += (double)((e[0] + e[1]) + (e[2] + e[3]));
    }
    return wave_sum_d(sum);
  };
  tops();
  const float c = -m * kLog2e;
  double sum = added([&](float v) { return __builtin_amdgcn_exp2f(fmaf(v, kLog2e, c)); }) *
               (double)__builtin_amdgcn_exp2f(-fmaf(m, kLog2e, c));
  // NaN or +inf among the values, none above -inf, or a reference so large that its remainder
  // is: with the first two put in their places (NaN as -inf, +inf as the largest number),
  // differences first
  if (!(fabsf(m) <= 1048576.f && sum < 1e30)) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      asm volatile("" : "+v"(x[j]));         // (or it is done for every chunk, to be chosen from)
      x[j] = fminf(fmaxf(x[j], -kInf), 3.402823466e38f);
    }
    tops();
    const float ref = m == -kInf ? 0.f : m;
    sum = added([&](float v) { return exp_neg(v - ref); });
  }
  uint32_t t;
  if (K <= kFewBeams) {
    t = kth_largest<1>({best > -kInf ? order_of(best) : 0u}, K);
  } else {
    uint32_t o[kQuads];
#pragma unroll
    for (int q = 0; q < kQuads; ++q) o[q] = top4[q] > -kInf ? order_of(top4[q]) : 0u;
    t = kth_largest(o, K);
  }
  // the fours that reach it (t 0: every one that has a candidate)
  const float bound = t ? float_of(t) : -3.402823466e38f;
  int fours = 0;
#pragma unroll
  for (int q = 0; q < kQuads; ++q) {
    const uint64_t who = __ballot(top4[q] >= bound);
    if (!who) continue;
    const int place = placed_at(who, fours);
    if (top4[q] >= bound && place < kFours) {
      *reinterpret_cast<f4*>(mine_s.x + 4 * place) =
          f4{x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]};
      mine_s.token[place] = at(4 * q);
    }
    fours += __popcll(who);
  }
  auto wrote = [] {                          // (this wave's LDS operations run in order)
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  };
  wrote();
  uint64_t* const list = lists + (int64_t)w * K;
  int n = fours <= kFours ? 0 : kNear + 1;
  for (int i = lane; n <= kNear && i - lane < 4 * fours; i += kWave) {
    const float v = i < 4 * fours ? mine_s.x[i] : -kInf;
    const uint64_t who = __ballot(v >= bound);
    const int place = placed_at(who, n);
    if (v >= bound && place < kNear) mine_s.near[place] = key_of(v, mine_s.token[i / 4] + i % 4);
    n += __popcll(who);
  }
  if (n <= kNear) {
    if (lane < kAtOnce) mine_s.near[n + lane] = 0;
    wrote();
    for (int i = lane; i < n; i += kWave) {
      const uint64_t k = mine_s.near[i];
      int r = 0;
      for (int j = 0; j < n; j += kAtOnce)
#pragma unroll
        for (int e = 0; e < kAtOnce; ++e) r += mine_s.near[j + e] > k;
      if (r < K) list[r] = k;
    }
    if (n + lane < K) list[n + lane] = 0;          // (beams <= 64)
  } else {
    uint64_t last = ~0ull;
#pragma unroll 1
    for (int r = 0; r < K; ++r) {
      uint64_t mine = 0;
#pragma unroll 1
      for (int i = c0 + lane; i < min(c0 + kWave * kPer, a.vocab); i += kWave) {
        const uint64_t k = key_of(fminf(fmaxf(logit_at<kType>(a.logits, base + i), -kInf),
                                        3.402823466e38f), i);
        if (k < last && k > mine) mine = k;
      }
      for (int d = 1; d < kWave; d *= 2) {
        const uint64_t o = __shfl_xor((unsigned long long)mine, d, kWave);
        mine = o > mine ? o : mine;
      }
      if (lane == 0) list[r] = mine;               // (more than beams candidates are there)
      last = mine;
    }
  }
  if (lane == 0) sums[w] = ChunkSum{sum, m, 0};
}

// ---------------------------------------------------------------------------
// A block per group.  Candidates in order: rank, then the lower row, then the key.  A wave's
// beams-th best list head bounds the group's beams-th best candidate from below; what reaches
// the largest such bound is collected and ranked by counting by one wave, after another bound
// where there are many.  If more does than the buffer holds (thousands of equal ranks), the
// places are filled one by one instead.  A thread holds the first keys of a list from the start
// on, so that few loads wait for others.  Bound by latency: 6.7 us for 4 beams of 151,936 logits
// (4.5 of them until the lists, which other dies wrote, have come), 11.8 for 16 of 16.
// ---------------------------------------------------------------------------
constexpr int kMerge = 1024, kMergeWaves = kMerge / kWave, kFound = 2048;
constexpr int kHeldKeys = 4, kHeldSums = 3, kFewHeads = 32;

struct Cand {
  double rank;
  uint64_t key;
  int beam;
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
  return (a.rank > b.rank) |
         ((a.rank == b.rank) & ((a.beam < b.beam) | ((a.beam == b.beam) & (a.key > b.key))));
}

// n ^ p.  Halves of whole numbers by products and a root, which are exact where the result is a
// whole number (pow is off in its last place there, and orders equal ranks).
__device__ __forceinline__ double length_power(int n, double p) {
  const double twice = 2.0 * p;
  if (twice != floor(twice)) return pow((double)n, p);
  double y = (int)twice & 1 ? sqrt((double)n) : 1.0, b = n;
  for (int k = (int)twice / 2; k; k /= 2, b *= b)
    if (k & 1) y *= b;
  return y;
}

__global__ __launch_bounds__(kMerge) void k_beam_merge(TfdBeamArgs a, int chunks,
                                                       const ChunkSum* __restrict__ sums,
                                                       const uint64_t* __restrict__ lists) {
  __shared__ double add_s[kMaxBeams], size_s[kMaxBeams];
  __shared__ float top_s[kMaxBeams];
  __shared__ uint8_t done_s[kMaxBeams];
  __shared__ int length_s[kMaxBeams];
  __shared__ uint32_t bound_s[kMergeWaves];
  __shared__ double found_rank[kFound];
  __shared__ uint64_t found_key[kFound];
  __shared__ uint8_t found_beam[kFound];
  __shared__ uint32_t head_s[kMerge];
  __shared__ Cand wave_s[kMergeWaves];
  __shared__ int n_s, heads_s;
  __shared__ float least_s;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int K = a.beams, row0 = blockIdx.x * K, n_lists = K * chunks;
  const uint64_t* const mine = lists + (int64_t)row0 * chunks * K;
  uint64_t held[kHeldKeys];
#pragma unroll
  for (int i = 0; i < kHeldKeys; ++i)
    held[i] = mine[(int64_t)min(tid, n_lists - 1) * K + min(i, K - 1)];
  if (tid == 0) n_s = heads_s = 0;
  // value = add + (logit - top), rank = value / size (the difference first: an infinite logit
  // stands as 3.4e38); a row that offers nothing has add NaN.  Divided, as the definition says: a
  // product with the reciprocal orders ranks that are equal (-3 of length 3, -2 of 2) otherwise.
  for (int b = wave; b < K; b += kMergeWaves) {
    const int row = row0 + b;
    const ChunkSum* const t = sums + (int64_t)row * chunks;
    ChunkSum c[kHeldSums];
#pragma unroll
    for (int i = 0; i < kHeldSums; ++i) c[i] = t[min(lane + i * kWave, chunks - 1)];
    const float score = a.scores[row];
    const int length = a.lengths ? a.lengths[row] : 0;
    const bool over = a.done && a.done[row], none = !(fabsf(score) < __builtin_huge_valf());
    const double size =
        a.penalty == 0.0 ? 1.0 : length_power(max(length + (over ? 0 : 1), 1), a.penalty);
    double lse = 0.0;
    float m = -__builtin_huge_valf();
    if (!over) {
#pragma unroll
      for (int i = 0; i < kHeldSums; ++i) m = fmaxf(m, c[i].top);
      for (int i = lane + kHeldSums * kWave; i < chunks; i += kWave) m = fmaxf(m, t[i].top);
      m = wave_max(m);
      // (an f32 exponential: the largest chunk's is exactly one)
      double s = 0.0;
#pragma unroll
      for (int i = 0; i < kHeldSums; ++i)
        if (c[i].sum > 0.0 && lane + i * kWave < chunks)
          s += c[i].sum * (double)exp_neg(c[i].top - m);
      for (int i = lane + kHeldSums * kWave; i < chunks; i += kWave)
        if (t[i].sum > 0.0) s += t[i].sum * (double)exp_neg(t[i].top - m);
      lse = log(wave_sum_d(s));
    }
    if (lane == 0) {
      top_s[b] = m;
      done_s[b] = over;
      length_s[b] = length;
      add_s[b] = none ? __builtin_nan("") : (double)score - lse;
      size_s[b] = size;
    }
  }
  __syncthreads();
  auto value_of = [&](const Cand& c) {
    return done_s[c.beam] ? add_s[c.beam]
                          : add_s[c.beam] + ((double)logit_of(c.key) - (double)top_s[c.beam]);
  };
  // entry i of a row's list, whose key (as far as there is one) is `key`; a finished row's
  // only candidate lies in its first list
  auto with_key = [&](int list, int i, uint64_t key) {
    Cand c;
    c.beam = list / chunks;
    c.key = !done_s[c.beam] ? key
            : list == c.beam * chunks && i == 0 ? key_of(0.f, a.eos) : 0;
    c.rank = c.key ? value_of(c) : kNone;
    if (a.penalty != 0.0) c.rank /= size_s[c.beam];
    if (!(c.rank > kNone)) c.key = 0, c.rank = kNone;
    return c;
  };
  auto cand = [&](int list, int i) { return with_key(list, i, mine[(int64_t)list * K + i]); };
  double best = tid < n_lists ? with_key(tid, 0, held[0]).rank : kNone;
  for (int l = tid + kMerge; l < n_lists; l += kMerge) best = fmax(best, cand(l, 0).rank);
  // in f32, rounded down: a bound all the same
  const uint32_t head = best > kNone ? order_of(__double2float_rd(best)) : 0u;
  const uint32_t t = kth_largest<1>({head}, K);
  if (lane == 0) bound_s[wave] = t;
  __syncthreads();
  uint32_t top = bound_s[0];
#pragma unroll
  for (int w = 1; w < kMergeWaves; ++w) top = max(top, bound_s[w]);
  // the threads' heads that reach it; where they are many, they bound it once more (every wave for
  // itself)
  const uint64_t reach = __ballot(head >= max(top, 1u));
  if (reach) {
    int at = 0;
    if (lane == 0) at = atomicAdd(&heads_s, __popcll(reach));
    at = placed_at(reach, __builtin_amdgcn_readfirstlane(at));
    if (head >= max(top, 1u)) head_s[at] = head;
  }
  __syncthreads();
  const int heads = heads_s;
  auto again = [&](auto& v) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(v) / 4); ++i)
      v[i] = lane + i * kWave < heads ? head_s[lane + i * kWave] : 0u;
    top = max(top, kth_largest(v, K));
  };
  if (heads > 4 * kWave) {
    uint32_t v[kMergeWaves];
    again(v);
  } else if (heads > kWave) {
    uint32_t v[4];
    again(v);
  } else if (heads > kFewHeads) {
    uint32_t v[1];
    again(v);
  }
  const double bound = top ? (double)float_of(top) : kNone;
  auto collect = [&](const Cand& c) {
    if (!c.key || c.rank < bound) return false;
    const int at = atomicAdd(&n_s, 1);
    if (at < kFound) found_rank[at] = c.rank, found_key[at] = c.key, found_beam[at] = c.beam;
    return true;
  };
  auto walk = [&](int l, int from) {         // kHeldKeys at a time: each load would be waited for
    bool more = true;
    for (int i0 = from; more && i0 < K; i0 += kHeldKeys) {
      uint64_t keys[kHeldKeys];
#pragma unroll
      for (int i = 0; i < kHeldKeys; ++i) keys[i] = mine[(int64_t)l * K + min(i0 + i, K - 1)];
#pragma unroll
      for (int i = 0; i < kHeldKeys; ++i)
        if (more && i0 + i < K) more = collect(with_key(l, i0 + i, keys[i]));
    }
  };
  if (tid < n_lists) {
    bool more = true;
#pragma unroll
    for (int i = 0; i < kHeldKeys; ++i)
      if (more && i < K) more = collect(with_key(tid, i, held[i]));
    if (more) walk(tid, kHeldKeys);
  }
  for (int l = tid + kMerge; l < n_lists; l += kMerge) walk(l, 0);
  __syncthreads();
  int n = n_s;
  auto put = [&](int place, const Cand& c) {
    const int row = row0 + c.beam, at = row0 + place;
    const bool over = done_s[c.beam];
    const int token = token_of(c.key), len = length_s[c.beam];
    a.parents[at] = row;
    a.tokens[at] = token;
    a.scores_out[at] = (float)value_of(c);
    a.lengths_out[at] = len + (over ? 0 : 1);
    a.done_out[at] = over || token == a.eos;
  };
  auto put_none = [&](int place) {
    const int at = row0 + place;
    a.parents[at] = at;
    a.tokens[at] = -1;
    a.scores_out[at] = -__builtin_huge_valf();
    a.lengths_out[at] = length_s[place];
    a.done_out[at] = done_s[place];
  };
  // many (a row far ahead of the others, whose lists' first keys are fewer than the beams): the
  // beams-th best of them bounds them again, and what reaches that moves to the front
  if (n > kWave && n <= kFound) {
    if (wave == 0) {
      auto bounded = [&](auto& v) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(v) / 4); ++i) {
          const int j = lane + i * kWave;
          v[i] = j < n ? order_of(__double2float_rd(found_rank[j])) : 0u;
        }
        least_s = float_of(kth_largest(v, K));
      };
      if (n <= 4 * kWave) {
        uint32_t v[4];
        bounded(v);
      } else if (n <= 16 * kWave) {
        uint32_t v[16];
        bounded(v);
      } else {
        uint32_t v[kFound / kWave];
        bounded(v);
      }
    }
    __syncthreads();
    const double least = (double)least_s;
    Cand kept[kFound / kMerge];
#pragma unroll
    for (int i = 0; i < kFound / kMerge; ++i) {
      const int j = min(tid + i * kMerge, n - 1);
      kept[i] = Cand{found_rank[j], found_key[j], found_beam[j]};
      if (tid + i * kMerge >= n || kept[i].rank < least) kept[i].key = 0;
    }
    if (tid == 0) n_s = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kFound / kMerge; ++i) {
      if (!kept[i].key) continue;
      const int at = atomicAdd(&n_s, 1);
      found_rank[at] = kept[i].rank, found_key[at] = kept[i].key, found_beam[at] = kept[i].beam;
    }
    __syncthreads();
    n = n_s;
  }
  if (n <= kWave) {                          // a candidate per lane of one wave
    if (wave > 0) return;
    const Cand c = lane < n ? Cand{found_rank[lane], found_key[lane], found_beam[lane]} : Cand{};
    int r = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) r += better(Cand{found_rank[j], found_key[j], found_beam[j]}, c);
    if (lane < n && r < K) put(r, c);
    if (lane >= n && lane < K) put_none(lane);
    return;
  }
  if (n <= kFound) {
    for (int i = tid; i < n; i += kMerge) {
      const Cand c{found_rank[i], found_key[i], found_beam[i]};
      int r = 0;
      for (int j = 0; j < n; ++j) r += better(Cand{found_rank[j], found_key[j], found_beam[j]}, c);
      if (r < K) put(r, c);
    }
    return;                                  // (more than K)
  }
  Cand last{__builtin_huge_val(), ~0ull, -1};
  for (int place = 0; place < K; ++place) {
    Cand top{kNone, 0, kMaxBeams};
    for (int l = tid; l < n_lists; l += kMerge)
      for (int i = 0; i < K; ++i) {
        const Cand c = cand(l, i);
        if (!c.key || better(top, c)) break;
        if (better(last, c)) {
          top = c;
          break;
        }
      }
    for (int d = 1; d < kWave; d *= 2) {
      Cand o;
      o.rank = __shfl_xor(top.rank, d, kWave);
      o.key = __shfl_xor((unsigned long long)top.key, d, kWave);
      o.beam = __shfl_xor(top.beam, d, kWave);
      if (better(o, top)) top = o;
    }
    if (lane == 0) wave_s[wave] = top;
    __syncthreads();
    top = wave_s[0];
    for (int w = 1; w < kMergeWaves; ++w)
      if (better(wave_s[w], top)) top = wave_s[w];
    __syncthreads();
    if (tid == 0) put(place, top);           // (more than K candidates are there)
    last = top;
  }
}

// Chunks as long as leave some waves for every compute unit and, for a group, no more lists
// than the merging block has threads; longer where there are many waves all the same.  The scan
// takes the same either way (8 beams of 4 groups over 248,320 f32 logits 10.9 us by 32 values a
// lane, 11.0 by 64; 16 of 16 over 100,352 in bf16 20.4 and 20.5, 15 of them as its loads take), the
// merge gains by fewer lists (11.7 and 10.9; 14.7 and 12.9).
BeamPlan beam_plan(int rows, int beams, int vocab) {
  BeamPlan p;
  p.per = 8;
  auto chunks = [&] { return (vocab + kWave * p.per - 1) / (kWave * p.per); };
  while (p.per < 32 && ((int64_t)rows * chunks() > 2048 || beams * chunks() > kMerge)) p.per *= 2;
  if (p.per == 32 && ((int64_t)rows * chunks() > 8192 || beams * chunks() > kMerge)) p.per = 64;
  p.chunks = chunks();
  return p;
}

bool beam_shape(int groups, int beams, int vocab) {
  return groups >= 0 && groups <= 65535 && beams >= 1 && beams <= kMaxBeams && vocab >= 1 &&
         vocab <= TFD_BEAM_MAX_VOCAB &&
         (int64_t)groups * beams * ((vocab + 1023) / 1024) < (1 << 23);
}

// ---------------------------------------------------------------------------
// Reorder.  A thread owns one place of all rows of a group: it reads every row that
// another one becomes before it writes any, so nothing has to be kept twice.  Rows that stay
// are neither read (but by others) nor written.  A wave knows the moves by itself -- lane b
// holds row b's parent, a 64-bit mask the rows that move -- and finds its tensor by a
// ballot, so nothing waits for a barrier.  Bound by memory: 8 rows in groups of 4 of 30 states of
// 2 MiB and as many windows of 48 KiB, 5 rows moved from 4, 106 us, 6 from 6 148, all from all 190:
// 5.2 to 5.5 TB/s.  A block that took four pieces in turn, the next one's loads behind the stores
// of the last, was a sixth slower.
// ---------------------------------------------------------------------------
constexpr int kUnits = 4;                    // small units per thread

__host__ __device__ inline int state_unit(const void* base, int64_t row_bytes) {
  const uint64_t both = (uint64_t)(uintptr_t)base | (uint64_t)row_bytes;
  return both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : both % 2 == 0 ? 2 : 1;
}

// The moves' sources, as many as there are, or their stores.
template <typename T, int kN, int kMoves, bool kStore>
__device__ __forceinline__ void each_move(T (&v)[kMoves][kN], T* p, int64_t units, int64_t u0,
                                          uint64_t moved, int from) {
#pragma unroll
  for (int i = 0; i < kMoves; ++i) {
    if (moved) {
      const int to = (int)__builtin_ctzll(moved);
      moved &= moved - 1;
      T* const row = p + (kStore ? to : __builtin_amdgcn_readlane(from, to)) * units;
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        const int64_t u = u0 + k * kBlock;
        if (!kStore) v[i][k] = row[min(u, units - 1)];
        else if (u < units) row[u] = v[i][k];
      }
    }
  }
}

template <typename T, int kN, int kMoves>
__device__ __forceinline__ void move_rows(uint8_t* base, int64_t row_bytes, int64_t block,
                                          uint64_t moved, int from) {
  const int64_t units = row_bytes / (int64_t)sizeof(T);
  const int64_t u = block * (kBlock * kN) + threadIdx.x;
  T* const p = reinterpret_cast<T*>(base);
  T v[kMoves][kN];
  each_move<T, kN, kMoves, false>(v, p, units, u, moved, from);
  each_move<T, kN, kMoves, true>(v, p, units, u, moved, from);
}

template <int kMoves>
__global__ __launch_bounds__(kBlock, kMoves <= 4 ? 8 : kMoves <= 16 ? 5 : 1)
void k_reorder(const TfdState* __restrict__ states, int n, const int* __restrict__ parents,
               int beams, int* err) {
  const int lane = threadIdx.x & (kWave - 1), first = blockIdx.y * beams;
  int from = lane;
  if (lane < beams) from = parents[first + lane] - first;
  const int64_t block = blockIdx.x;
  int t = -1;
  for (int i = 0; i < n; i += kWave)
    t += __popcll(__ballot(i + lane < n && states[min(i + lane, n - 1)].first_block <= block));
  if (from < 0 || from >= beams) {
    if (lane < beams) raise_error(err, TFD_ERR_ROW_RANGE);
    from = lane;
  }
  const uint64_t moved = __ballot(from != lane);
  if (!moved) return;
  const TfdState st = states[__builtin_amdgcn_readfirstlane(t)];
  const int64_t at = block - st.first_block;
  uint8_t* const base = (uint8_t*)st.base + first * st.row_bytes;
  const int unit = state_unit(st.base, st.row_bytes);
  if (unit == 16) move_rows<u32x4, 1, kMoves>(base, st.row_bytes, at, moved, from);
  else if (unit == 4)
    move_rows<uint32_t, kUnits, kMoves>(base, st.row_bytes, at, moved, from);
  else if (unit == 2)
    move_rows<uint16_t, kUnits, kMoves>(base, st.row_bytes, at, moved, from);
  else
    move_rows<uint8_t, kUnits, kMoves>(base, st.row_bytes, at, moved, from);
}

}  // namespace

extern "C" {

int64_t tfd_beam_work_bytes(int groups, int beams, int vocab) {
  if (!beam_shape(groups, beams, vocab)) return 0;
  const BeamPlan p = beam_plan(groups * beams, beams, vocab);
  return (int64_t)groups * beams * p.chunks * ((int64_t)sizeof(ChunkSum) + 8 * beams);
}

int tfd_beam_select(const TfdBeamArgs* args, void* stream) {
  if (!args) return fail(kBadArg, "beam_select: null args");
  const TfdBeamArgs& a = *args;
  if (a.type != TFD_TYPE_F32 && a.type != TFD_TYPE_BF16 && a.type != TFD_TYPE_F16)
    return fail(kBadArg, "beam_select: type %d", a.type);
  if (!beam_shape(a.groups, a.beams, a.vocab))
    return fail(kBadShape, "beam_select: groups=%d beams=%d (1..%d) vocab=%d", a.groups, a.beams,
                kMaxBeams, a.vocab);
  if (a.eos < -1 || a.eos >= a.vocab)
    return fail(kBadArg, "beam_select: eos %d outside -1..%d", a.eos, a.vocab - 1);
  if (!(a.penalty >= 0.0) || a.penalty > 100.0)
    return fail(kBadArg, "beam_select: penalty must lie in 0..100");
  if (a.groups == 0) return 0;
  if (!a.logits || !a.scores || !a.parents || !a.tokens || !a.scores_out || !a.lengths_out ||
      !a.done_out)
    return fail(kBadArg, "beam_select: null pointer");
  const int rows = a.groups * a.beams, size = a.type == TFD_TYPE_F32 ? 4 : 2;
  if ((rows > 1 && a.ldl < a.vocab) || (uintptr_t)a.logits % size)
    return fail(kBadArg, "beam_select: ldl=%lld, logits aligned to their elements",
                (long long)a.ldl);
  if (!a.work || (uintptr_t)a.work % 16 ||
      a.work_bytes < tfd_beam_work_bytes(a.groups, a.beams, a.vocab))
    return fail(kBadArg, "beam_select: work of %lld bytes", (long long)a.work_bytes);
  const BeamPlan p = beam_plan(rows, a.beams, a.vocab);
  ChunkSum* const sums = (ChunkSum*)a.work;
  uint64_t* const lists = (uint64_t*)(sums + (int64_t)rows * p.chunks);
  const bool vec = a.ldl * size % 16 == 0 && (uintptr_t)a.logits % 16 == 0;
  const int waves = rows * p.chunks;
  const unsigned grid = (unsigned)((waves + kWavesPerBlock - 1) / kWavesPerBlock);
  auto s = (hipStream_t)stream;
#define TFD_SCAN(T, P)                                                                   \
  if (vec) k_beam_scan<T, P, true><<<grid, kBlock, 0, s>>>(a, p.chunks, waves, sums, lists); \
  else k_beam_scan<T, P, false><<<grid, kBlock, 0, s>>>(a, p.chunks, waves, sums, lists);
#define TFD_SCAN_TYPE(T)                         \
  {                                              \
    if (p.per == 8) { TFD_SCAN(T, 8) }           \
    else if (p.per == 16) { TFD_SCAN(T, 16) }    \
    else if (p.per == 32) { TFD_SCAN(T, 32) }    \
    else { TFD_SCAN(T, 64) }                     \
  }
  if (a.type == TFD_TYPE_F32) TFD_SCAN_TYPE(TFD_TYPE_F32)
  else if (a.type == TFD_TYPE_BF16) TFD_SCAN_TYPE(TFD_TYPE_BF16)
  else TFD_SCAN_TYPE(TFD_TYPE_F16)
#undef TFD_SCAN_TYPE
#undef TFD_SCAN
  k_beam_merge<<<a.groups, kMerge, 0, s>>>(a, p.chunks, sums, lists);
  return launched("beam_select");
}

int64_t tfd_state_blocks(const void* base, int64_t row_bytes) {
  if (row_bytes <= 0) return 0;
  const int unit = state_unit(base, row_bytes);
  const int64_t per = (int64_t)kBlock * (unit == 16 ? 16 : kUnits * unit);
  return (row_bytes + per - 1) / per;
}

int tfd_reorder_states(const TfdState* states, int n, int64_t blocks, const int32_t* parents,
                       int groups, int beams, int32_t* err, void* stream) {
  if (n < 0 || groups < 0 || groups > 65535 || beams < 1 || beams > kMaxBeams || blocks < 0 ||
      blocks >= (1ll << 24))
    return fail(kBadShape, "reorder_states: n=%d groups=%d beams=%d (1..%d) blocks=%lld", n, groups,
                beams, kMaxBeams, (long long)blocks);
  if (n == 0 || groups == 0 || blocks == 0) return 0;
  if (!states || !parents) return fail(kBadArg, "reorder_states: null pointer");
  const dim3 grid((unsigned)blocks, groups);
  auto s = (hipStream_t)stream;
#define TFD_MOVES(M) k_reorder<M><<<grid, kBlock, 0, s>>>(states, n, parents, beams, err)
  if (beams <= 4) TFD_MOVES(4);
  else if (beams <= 16) TFD_MOVES(16);
  else if (beams <= 32) TFD_MOVES(32);
  else TFD_MOVES(64);
#undef TFD_MOVES
  return launched("reorder_states");
}

}  // extern "C"
