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

__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return ((uint64_t)hi << 32) | lo;
}
__device__ __forceinline__ double lane_d(double v, int lane) {
  return __builtin_bit_cast(double, lane_u64(__builtin_bit_cast(uint64_t, v), lane));
}
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) v += __shfl_xor(v, d, kWave);
  return v;
}

// exp(x) for x <= 0 to about an f32's last bit: the product with log2 e in two parts.
__device__ __forceinline__ float exp_neg(float x) {
  constexpr float kHi = 1.44269502162933349609375f, kLo = 1.92596303e-8f;
  const float t = x * kHi;
  const float rest = fmaf(x, kHi, -t) + x * kLo;
  const float e = __builtin_amdgcn_exp2f(t);
  return x < -100.f ? 0.f : fmaf(e, rest * 0.69314718055994530942f, e);
}

struct BeamPlan {
  int per, chunks;       // values of a thread, chunks of a row
};
constexpr int kScan = 256;

// What a row's chunk leaves: its largest logit, the sum of exp(x - that), and its `beams`
// largest keys in falling order (0 where there are fewer).
struct ChunkSum {
  double sum;
  float top;
  int pad;
};

// ---------------------------------------------------------------------------
// A block per chunk of a row, its values in registers.  The beams-th largest of the threads'
// best keys bounds the chunk's beams-th largest from below; what reaches it -- in at most
// `beams` threads -- is collected and ranked by counting.
// ---------------------------------------------------------------------------
template <int kType>
__device__ __forceinline__ float logit_at(const void* p, int64_t i) {
  float v;
  if (kType == TFD_TYPE_F32) v = ((const float*)p)[i];
  else if (kType == TFD_TYPE_BF16) v = bf2f(((const bf16*)p)[i]);
  else v = (float)__builtin_bit_cast(_Float16, ((const uint16_t*)p)[i]);
  return v;
}

template <int kType, int kPer, bool kVec>
__global__ __launch_bounds__(kScan) void k_beam_scan(TfdBeamArgs a, int chunks,
                                                     ChunkSum* __restrict__ sums,
                                                     uint64_t* __restrict__ lists) {
  constexpr int kWaves = kScan / kWave;
  __shared__ uint64_t best_s[kScan];
  __shared__ uint64_t found_s[kMaxBeams * kPer];
  __shared__ float top_s[kWaves];
  __shared__ double sum_s[kWaves];
  __shared__ uint64_t bound_s;
  __shared__ int n_s;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int row = blockIdx.x / chunks, chunk = blockIdx.x % chunks;
  if (a.done && a.done[row]) return;               // (its lists are not read)
  const int c0 = chunk * kScan * kPer, K = a.beams;
  const int64_t base = (int64_t)row * a.ldl;
  float x[kPer];
  auto at = [&](int j) { return c0 + (j / 4) * 4 * kScan + 4 * tid + j % 4; };
  if (kVec) {
#pragma unroll
    for (int j = 0; j < kPer; j += 4) {
      const int i = min(at(j), a.vocab - 4);       // (vocab % 4 == 0)
      if (kType == TFD_TYPE_F32) {
        const u32x4 v = *(g_u32x4*)((const float*)a.logits + base + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[j + e] = __uint_as_float(v[e]);
      } else {
        const uint64_t v = *(const uint64_t*)((const uint16_t*)a.logits + base + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint16_t h = (uint16_t)(v >> (16 * e));
          x[j + e] = kType == TFD_TYPE_BF16 ? bf2f(h) : (float)__builtin_bit_cast(_Float16, h);
        }
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < kPer; ++j) x[j] = logit_at<kType>(a.logits, base + min(at(j), a.vocab - 1));
  }
  float top = -__builtin_huge_valf();
  int where = 0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    if (x[j] > 3.402823466e38f) x[j] = 3.402823466e38f;      // (NaN stays)
    if (at(j) >= a.vocab) x[j] = -__builtin_huge_valf();
    if (x[j] > top) top = x[j], where = j;
  }
  const uint64_t best = key_of(top, at(where));
  if (tid == 0) n_s = 0, bound_s = 0;
  best_s[tid] = best;
  const float wt = wave_max(top);
  if (lane == 0) top_s[wave] = wt;
  __syncthreads();
  float m = top_s[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, top_s[w]);
  double sum = 0.0;
#pragma unroll
  for (int j = 0; j < kPer; ++j) sum += x[j] > -__builtin_huge_valf() ? exp_neg(x[j] - m) : 0.f;
  sum = wave_sum_d(sum);
  if (lane == 0) sum_s[wave] = sum;
  int rank = 0;
  for (int i = 0; i < kScan; i += 2) rank += (best_s[i] > best) + (best_s[i + 1] > best);
  if (best && rank == K - 1) bound_s = best;
  __syncthreads();
  const uint64_t bound = bound_s;
  if (best && best >= bound) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const uint64_t k = key_of(x[j], at(j));
      if (k && k >= bound) found_s[atomicAdd(&n_s, 1)] = k;
    }
  }
  __syncthreads();
  const int n = n_s;
  uint64_t* const list = lists + (int64_t)blockIdx.x * K;
  for (int i = tid; i < n; i += kScan) {
    const uint64_t k = found_s[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += found_s[j] > k;
    if (r < K) list[r] = k;
  }
  for (int i = n + tid; i < K; i += kScan) list[i] = 0;
  if (tid == 0) {
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) t += sum_s[w];
    sums[blockIdx.x] = ChunkSum{t, m, 0};
  }
}

// ---------------------------------------------------------------------------
// A block per group.  Candidates in order: rank, then the lower row, then the key.  A wave's
// beams-th best list head bounds the group's beams-th best candidate from below; what reaches
// the largest such bound is collected and ranked by counting.  If more than the buffer holds
// does (thousands of equal ranks), the places are filled one by one instead.
// ---------------------------------------------------------------------------
constexpr int kMerge = 512, kMergeWaves = kMerge / kWave, kFound = 2048;

struct Cand {
  double rank;
  uint64_t key;
  int beam;
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
  if (a.rank != b.rank) return a.rank > b.rank;
  if (a.beam != b.beam) return a.beam < b.beam;
  return a.key > b.key;
}

__global__ __launch_bounds__(kMerge) void k_beam_merge(TfdBeamArgs a, int chunks,
                                                       const ChunkSum* __restrict__ sums,
                                                       const uint64_t* __restrict__ lists) {
  __shared__ double add_s[kMaxBeams], div_s[kMaxBeams];
  __shared__ float top_s[kMaxBeams];
  __shared__ double bound_s[kMergeWaves];
  __shared__ double found_rank[kFound];
  __shared__ uint64_t found_key[kFound];
  __shared__ uint8_t found_beam[kFound];
  __shared__ Cand wave_s[kMergeWaves];
  __shared__ int n_s;
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  const int K = a.beams, row0 = blockIdx.x * K;
  if (tid == 0) n_s = 0;
  // value = add + (logit - top), rank = value / div (the difference first: an infinite logit
  // stands as 3.4e38); a row that offers nothing has add NaN
  for (int b = wave; b < K; b += kMergeWaves) {
    const int row = row0 + b;
    const float score = a.scores[row];
    const bool over = a.done && a.done[row], none = !(fabsf(score) < __builtin_huge_valf());
    double lse = 0.0;
    float m = -__builtin_huge_valf();
    if (!over) {
      const ChunkSum* const t = sums + (int64_t)row * chunks;
      for (int c = lane; c < chunks; c += kWave) m = fmaxf(m, t[c].top);
      m = wave_max(m);
      double s = 0.0;
      for (int c = lane; c < chunks; c += kWave)
        if (t[c].top > -__builtin_huge_valf()) s += t[c].sum * exp((double)t[c].top - (double)m);
      lse = log(wave_sum_d(s));
    }
    if (lane == 0) {
      const int len = (a.lengths ? a.lengths[row] : 0) + (over ? 0 : 1);
      top_s[b] = m;
      add_s[b] = none ? __builtin_nan("") : (double)score - lse;
      div_s[b] = a.penalty == 0.f ? 1.0 : pow((double)max(len, 1), (double)a.penalty);
    }
  }
  __syncthreads();
  const int n_lists = K * chunks;
  auto value_of = [&](const Cand& c) {
    return add_s[c.beam] + ((double)logit_of(c.key) - (double)top_s[c.beam]);
  };
  // entry i of a row's list; a finished row's only candidate lies in its first list
  auto cand = [&](int list, int i) {
    Cand c;
    c.beam = list / chunks;
    const int row = row0 + c.beam;
    c.rank = kNone;
    c.key = 0;
    if (a.done && a.done[row]) {
      if (list % chunks == 0 && i == 0) {
        c.key = key_of(0.f, a.eos);
        c.rank = add_s[c.beam] / div_s[c.beam];
      }
    } else {
      c.key = lists[((int64_t)row * chunks + list % chunks) * K + i];
      if (c.key) c.rank = value_of(c) / div_s[c.beam];
    }
    if (c.key && !(c.rank > kNone)) c.key = 0, c.rank = kNone;
    return c;
  };
  double best = kNone;
  for (int l = tid; l < n_lists; l += kMerge) best = fmax(best, cand(l, 0).rank);
  int rank = 0;
  for (int i = 0; i < kWave; ++i) {
    const double o = lane_d(best, i);
    rank += o > best || (o == best && i < lane);
  }
  const uint64_t who = __ballot(rank == K - 1);
  if (lane == 0) bound_s[wave] = lane_d(best, (int)__builtin_ctzll(who));
  __syncthreads();
  double bound = bound_s[0];
  for (int w = 1; w < kMergeWaves; ++w) bound = fmax(bound, bound_s[w]);
  for (int l = tid; l < n_lists; l += kMerge)
    for (int i = 0; i < K; ++i) {
      const Cand c = cand(l, i);
      if (!c.key || c.rank < bound) break;
      const int at = atomicAdd(&n_s, 1);
      if (at < kFound) found_rank[at] = c.rank, found_key[at] = c.key, found_beam[at] = c.beam;
    }
  __syncthreads();
  const int n = n_s;
  auto put = [&](int place, const Cand& c) {
    const int row = row0 + c.beam, at = row0 + place;
    const bool over = a.done && a.done[row];
    const int token = token_of(c.key), len = a.lengths ? a.lengths[row] : 0;
    a.parents[at] = row;
    a.tokens[at] = token;
    a.scores_out[at] = over ? a.scores[row] : (float)value_of(c);
    a.lengths_out[at] = len + (over ? 0 : 1);
    a.done_out[at] = over || token == a.eos;
  };
  auto put_none = [&](int place) {
    const int at = row0 + place;
    a.parents[at] = at;
    a.tokens[at] = -1;
    a.scores_out[at] = -__builtin_huge_valf();
    a.lengths_out[at] = a.lengths ? a.lengths[at] : 0;
    a.done_out[at] = a.done ? a.done[at] : 0;
  };
  if (n <= kFound) {
    for (int i = tid; i < n; i += kMerge) {
      const Cand c{found_rank[i], found_key[i], found_beam[i]};
      int r = 0;
      for (int j = 0; j < n; ++j) r += better(Cand{found_rank[j], found_key[j], found_beam[j]}, c);
      if (r < K) put(r, c);
    }
    for (int i = n + tid; i < K; i += kMerge) put_none(i);
    return;
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

BeamPlan beam_plan(int rows, int vocab) {
  BeamPlan p;
  p.per = 4;
  while (p.per < 32 && (int64_t)rows * ((vocab + kScan * p.per - 1) / (kScan * p.per)) > 1024)
    p.per *= 2;
  p.chunks = (vocab + kScan * p.per - 1) / (kScan * p.per);
  return p;
}

bool beam_shape(int groups, int beams, int vocab) {
  return groups >= 0 && groups <= 65535 && beams >= 1 && beams <= kMaxBeams && vocab >= 1 &&
         vocab <= TFD_BEAM_MAX_VOCAB &&
         (int64_t)groups * beams * ((vocab + 1023) / 1024) < (1 << 24);
}

// ---------------------------------------------------------------------------
// Reorder.  A thread owns one place of all rows of a group: it reads every row that
// another one becomes before it writes any, so nothing has to be kept twice.  Rows that stay
// are neither read (but by others) nor written.
// ---------------------------------------------------------------------------
constexpr int kUnits = 4;                    // small units per thread

__host__ __device__ inline int state_unit(const void* base, int64_t row_bytes) {
  const uint64_t both = (uint64_t)(uintptr_t)base | (uint64_t)row_bytes;
  return both % 16 == 0 ? 16 : both % 4 == 0 ? 4 : both % 2 == 0 ? 2 : 1;
}
inline int64_t state_blocks(const void* base, int64_t row_bytes) {
  const int64_t per = kBlock * (state_unit(base, row_bytes) == 16 ? 1 : kUnits) *
                      (int64_t)state_unit(base, row_bytes);
  return (row_bytes + per - 1) / per;
}

template <typename T, int kN, int kBeams>
__device__ __forceinline__ void move_rows(uint8_t* base, int64_t row_bytes, int64_t unit0,
                                          const int* from_s, int beams) {
  const int64_t units = row_bytes / (int64_t)sizeof(T);
  T* const p = reinterpret_cast<T*>(base);
  T v[kBeams][kN];
#pragma unroll
  for (int b = 0; b < kBeams; ++b) {
    const int from = b < beams ? __builtin_amdgcn_readfirstlane(from_s[b]) : b;
    if (from != b) {
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        const int64_t u = min(unit0 + k * kBlock + (int64_t)threadIdx.x, units - 1);
        v[b][k] = p[from * units + u];
      }
    }
  }
#pragma unroll
  for (int b = 0; b < kBeams; ++b) {
    const int from = b < beams ? __builtin_amdgcn_readfirstlane(from_s[b]) : b;
    if (from != b) {
#pragma unroll
      for (int k = 0; k < kN; ++k) {
        const int64_t u = unit0 + k * kBlock + (int64_t)threadIdx.x;
        if (u < units) p[b * units + u] = v[b][k];
      }
    }
  }
}

template <int kBeams>
__global__ __launch_bounds__(kBlock) void k_reorder(const TfdState* __restrict__ states, int n,
                                                    const int* __restrict__ parents, int beams,
                                                    int* err) {
  __shared__ int from_s[kBeams];
  const int g = blockIdx.y;
  if ((int)threadIdx.x < beams) {
    const int first = g * beams, from = parents[first + threadIdx.x];
    const bool in = from >= first && from < first + beams;
    if (!in) raise_error(err, TFD_ERR_ROW_RANGE);
    from_s[threadIdx.x] = in ? from - first : (int)threadIdx.x;
  }
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (states[mid].first_block <= (int64_t)blockIdx.x) lo = mid;
    else hi = mid;
  }
  const TfdState t = states[lo];
  __syncthreads();
  const int64_t block = (int64_t)blockIdx.x - t.first_block;
  uint8_t* const base = (uint8_t*)t.base + g * beams * t.row_bytes;
  const int unit = state_unit(t.base, t.row_bytes);
  if (unit == 16) move_rows<u32x4, 1, kBeams>(base, t.row_bytes, block * kBlock, from_s, beams);
  else if (unit == 4)
    move_rows<uint32_t, kUnits, kBeams>(base, t.row_bytes, block * kBlock * kUnits, from_s, beams);
  else if (unit == 2)
    move_rows<uint16_t, kUnits, kBeams>(base, t.row_bytes, block * kBlock * kUnits, from_s, beams);
  else
    move_rows<uint8_t, kUnits, kBeams>(base, t.row_bytes, block * kBlock * kUnits, from_s, beams);
}

}  // namespace

extern "C" {

int64_t tfd_beam_work_bytes(int groups, int beams, int vocab) {
  if (!beam_shape(groups, beams, vocab)) return 0;
  const BeamPlan p = beam_plan(groups * beams, vocab);
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
  if (!(a.penalty >= 0.f) || a.penalty > 100.f)
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
  const BeamPlan p = beam_plan(rows, a.vocab);
  ChunkSum* const sums = (ChunkSum*)a.work;
  uint64_t* const lists = (uint64_t*)(sums + (int64_t)rows * p.chunks);
  const bool vec = a.vocab % 4 == 0 && a.ldl % 4 == 0 && (uintptr_t)a.logits % (4 * size) == 0;
  const unsigned grid = (unsigned)(rows * p.chunks);
  auto s = (hipStream_t)stream;
#define TFD_SCAN(T, P)                                                                   \
  if (vec) k_beam_scan<T, P, true><<<grid, kScan, 0, s>>>(a, p.chunks, sums, lists);     \
  else k_beam_scan<T, P, false><<<grid, kScan, 0, s>>>(a, p.chunks, sums, lists);
#define TFD_SCAN_TYPE(T)                         \
  {                                              \
    if (p.per == 4) { TFD_SCAN(T, 4) }           \
    else if (p.per == 8) { TFD_SCAN(T, 8) }      \
    else if (p.per == 16) { TFD_SCAN(T, 16) }    \
    else { TFD_SCAN(T, 32) }                     \
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
  return row_bytes > 0 ? state_blocks(base, row_bytes) : 0;
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
  if (beams <= 4) k_reorder<4><<<grid, kBlock, 0, s>>>(states, n, parents, beams, err);
  else if (beams <= 8) k_reorder<8><<<grid, kBlock, 0, s>>>(states, n, parents, beams, err);
  else if (beams <= 16) k_reorder<16><<<grid, kBlock, 0, s>>>(states, n, parents, beams, err);
  else if (beams <= 32) k_reorder<32><<<grid, kBlock, 0, s>>>(states, n, parents, beams, err);
  else k_reorder<64><<<grid, kBlock, 0, s>>>(states, n, parents, beams, err);
  return launched("reorder_states");
}

}  // extern "C"
