// Drafted tokens that form a tree: masks, acceptance, and attention over a paged cache.
#include <algorithm>

#include "host_common.h"
#include "panel.h"
#include "tf_search.h"

using namespace tfd;
using namespace tfd_host;

namespace {

constexpr int kErrPosRange = 2, kErrPageRange = 4, kErrRowRange = TFD_ERR_ROW_RANGE;
constexpr int kMaxNodes = TFD_TREE_MAX_NODES, kMaxWords = kMaxNodes / 64;

__device__ __forceinline__ int row_nodes(const int* counts, int row, int nodes) {
  return counts ? max(0, min(counts[row], nodes)) : nodes;
}

// ---------------------------------------------------------------------------
// Masks and depths by pointer doubling: after round i a node's mask holds itself and 2^i - 1
// ancestors, and it points at the next one.  A block per row, a thread per node.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kMaxNodes) void k_tree_masks(const int* __restrict__ parents,
                                                          const int* __restrict__ counts,
                                                          int nodes, uint64_t* __restrict__ masks,
                                                          int* __restrict__ depths, int* err) {
  __shared__ uint64_t m_s[kMaxWords][kMaxNodes];
  __shared__ int up_s[kMaxNodes], d_s[kMaxNodes];
  const int row = blockIdx.x, t = threadIdx.x, words = (nodes + 63) / 64;
  const int n = row_nodes(counts, row, nodes);
  int up = t < n ? parents[(int64_t)row * nodes + t] : -1;
  if (up < -1 || up >= t) {
    if (t < n) raise_error(err, kErrRowRange);
    up = -1;
  }
  uint64_t m[kMaxWords];
#pragma unroll
  for (int w = 0; w < kMaxWords; ++w) m[w] = t < n && t / 64 == w ? 1ull << (t & 63) : 0;
  int depth = up >= 0 ? 1 : 0;
  for (int reach = 1; reach < n; reach *= 2) {
#pragma unroll
    for (int w = 0; w < kMaxWords; ++w) m_s[w][t] = m[w];
    up_s[t] = up;
    d_s[t] = depth;
    __syncthreads();
    if (up >= 0) {
#pragma unroll
      for (int w = 0; w < kMaxWords; ++w) m[w] |= m_s[w][up];
      depth += d_s[up];
      up = up_s[up];
    }
    __syncthreads();
  }
  if (t < nodes) {
    depths[(int64_t)row * nodes + t] = t < n ? depth : 0;
    for (int w = 0; w < kMaxWords; ++w)
      if (w < words) masks[((int64_t)row * nodes + t) * words + w] = m[w];
  }
}

// ---------------------------------------------------------------------------
// The accepted path: a wave per row, node l + 64 j in lane l; a step of the path is one
// ballot per 64 nodes.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kWave) void k_tree_accept(
    const int* __restrict__ tokens, const int* __restrict__ parents,
    const int* __restrict__ picks, const int* __restrict__ counts, int nodes,
    int* __restrict__ path, int* __restrict__ accepted, int* __restrict__ next) {
  const int row = blockIdx.x, lane = threadIdx.x;
  const int64_t at = (int64_t)row * nodes;
  const int n = row_nodes(counts, row, nodes);
  int tok[kMaxWords], up[kMaxWords], pick[kMaxWords];
#pragma unroll
  for (int j = 0; j < kMaxWords; ++j) {
    const int t = lane + kWave * j, u = min(t, nodes - 1);
    tok[j] = tokens[at + u];
    pick[j] = picks[at + u];
    up[j] = t < n ? parents[at + u] : -1;
    if (t < nodes) path[at + t] = -1;
  }
  auto pick_of = [&](int t) {
    int v = 0;
#pragma unroll
    for (int j = 0; j < kMaxWords; ++j)
      if (t / kWave == j) v = __builtin_amdgcn_readlane(pick[j], t % kWave);
    return v;
  };
  int cur = 0, len = 0, want = -1;
  if (n > 0) {
    // (every store of -1 above is by the lane that may store again below)
    while (true) {
      if (lane == len % kWave) path[at + len] = cur;
      ++len;
      want = pick_of(cur);
      int child = -1;
#pragma unroll
      for (int j = kMaxWords - 1; j >= 0; --j) {
        const uint64_t who = __ballot(up[j] == cur && tok[j] == want && lane + kWave * j > cur);
        if (who) child = kWave * j + (int)__builtin_ctzll(who);
      }
      if (child < 0) break;
      cur = __builtin_amdgcn_readfirstlane(child);
    }
  }
  if (lane == 0) {
    accepted[row] = len;
    next[row] = want;
  }
}

// ---------------------------------------------------------------------------
// Attention.  A row's kv head is a product of T * G query columns (node t of head g: column
// t G + g) with its n = L + count positions.  Everything is kept transposed, so that a lane
// owns one query's softmax: S^T = K Q^T gives lane l the scores of query l % 16 at
// positions 16 i + 4 (l / 16) + e, which is, packed, an operand of O^T += V^T P^T (a product's
// k may be taken in any order that both operands share).  V lies in LDS by rows, and the
// transposing read gives V^T's operands; its 32-byte pieces are permuted by the row so that the
// 16 rows of such a read take the fewest cycles.
//
// Softmax against a running reference, in f32.  The probabilities have to become bf16 for the
// second product: they stay a sum of two bf16 (2^-16 of each), however many columns there are.
// By many, a caller may ask for one (2^-8; they average: 1.4 times the error of an attention in
// f32 that rounds its output), which saves a third of the products and half of what VALU does for
// a probability: 211 to 161 us at 4 rows to 30,000 positions, 61 nodes of 32 heads over 8.
//
// Two kernels.  Few columns (k_tree_few): the keys are what is waited for, so each wave
// takes other tiles of 32 positions, its K straight into registers as operands and its V
// through a private piece of LDS, and no barrier until the waves' sums are joined.  Many
// columns (k_tree_many): the waves take 16 NQ columns each and share tiles in LDS, loaded
// straight to it three tiles ahead (from pages anywhere a load takes some 3 us), one barrier a
// tile.  Both may cut a row's positions into splits, which k_tree_join adds.
//
// Few columns are bound by memory (32 rows to 4,096 positions by 7 nodes: 93 us, 5.5 TB/s) or, by
// one row, by latency (700 positions: 14 us).  Many: MFMA (40% of the time at 61 nodes of 32
// heads), LDS, VALU and loads take turns, since registers leave room for two waves a SIMD (203 us
// and the join's 8, 590 TFLOP/s of the definition's products, whose second takes two); of 256 dims
// (8 rows to 5,003, 23 nodes of 16 heads over 2: 50 us) also by the partial sums of its splits,
// which the join reads again (10 us).
// ---------------------------------------------------------------------------
typedef short i16x4 __attribute__((ext_vector_type(4)));
constexpr int kTile = 32;                    // positions of a wave's tile

template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
  return D == 64 ? (row >> 1) & 3 : row & 7;
}
// byte of V[row][16 chunk]
template <int D>
__device__ __forceinline__ int v_at(int row, int chunk) {
  return row * D * 2 + ((chunk ^ v_swizzle<D>(row)) << 5);
}
// byte of K[row][8 chunk]: 16 rows of a chunk lie in as many places of 256 bytes
template <int D>
__device__ __forceinline__ int k_at(int row, int chunk) {
  return row * D * 2 + ((chunk ^ (D == 64 ? (row >> 1) & 7 : row & 15)) << 4);
}

// V^T's operand for dims 16 dt .. + 15 and the 32 positions at `v`.
template <int D>
__device__ __forceinline__ u32x4 v_operand(const uint8_t* v, int dt, int lane) {
  i16x4 f[2];
#pragma unroll
  for (int t = 0; t < 2; ++t)
    f[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) i16x4*)(v +
            v_at<D>(16 * t + 4 * (lane >> 4) + ((lane & 15) >> 2), dt) + (lane & 3) * 8));
  const u32x2 a = __builtin_bit_cast(u32x2, f[0]), b = __builtin_bit_cast(u32x2, f[1]);
  return u32x4{a.x, a.y, b.x, b.y};
}

// Two bf16 with zeros in the place of infinities and NaN.
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}
// 16 bytes of V at position j of a tile that reaches the drafted positions or a page that is not
// there: zeros in that page and past the last position, which hold anything, and in the place of
// drafted values that are not finite.
__device__ __forceinline__ u32x4 clean_v(u32x4 v, int j, int L, int n, bool held, bool& odd) {
  if (j >= n || !held) v = u32x4{0u, 0u, 0u, 0u};
  if (j >= L) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const uint32_t f = finite_halves(v[w]);
      odd |= f != v[w];
      v[w] = f;
    }
  }
  return v;
}

// What all lanes read alike and no kernel here writes, through the scalar cache.
typedef const __attribute__((address_space(4))) int c_int;
__device__ __forceinline__ c_int* uniform(const int* p) { return (c_int*)(uintptr_t)p; }

// One row's part of a call, as a block sees it.
struct TreeRow {
  const int* table;
  const bf16 *k, *v;                         // of the kv head, page 0
  const uint64_t* masks;
  int64_t page_size;
  int row, h, G, L, n, cols, first, words, last_page, num_pages, max_pages;
  bool bad_page;

  // A page, -1 for one that is none: its positions take no part, and loads take page 0 in its
  // place.  Entries past the last position's page need not be set (and they are read before that
  // page is known: no load waits for the row's length).
  __device__ __forceinline__ int page_at(int i) {
    const int p = table[min(i, max_pages - 1)];
    const bool ok = p >= 0 && p < num_pages;
    bad_page |= !ok && i <= last_page;
    return ok ? p : -1;
  }
  __device__ __forceinline__ int node_of(int c) const { return (first + min(c, cols - 1)) / G; }
  // bit i: a column that sees the nodes of m0 (and m1, the next word) from node `from` = j0 - L
  // on, or from 0, sees position j0 + i, i < 32 (the context: every one)
  __device__ __forceinline__ uint32_t seen(uint64_t m0, uint64_t m1, int j0) const {
    const int from = j0 - L, sh = max(from, 0) & 63;
    uint64_t bits = m0 >> sh;
    if (sh) bits |= m1 << (64 - sh);
    if (from <= -kTile) bits = 0xffffffffu;
    else if (from < 0) bits = (bits << -from) | ((1ull << -from) - 1);
    const int left = n - j0;
    if (left < kTile) bits = left > 0 ? bits & ((1ull << left) - 1) : 0;
    return (uint32_t)bits;
  }
  __device__ __forceinline__ uint32_t seen_by(int c, int j0) const {
    const uint64_t* const m = masks + (int64_t)node_of(c) * words;
    const int w = max(j0 - L, 0) >> 6;
    const uint64_t m0 = m[min(w, words - 1)], m1 = m[min(w + 1, words - 1)];
    return seen(w < words ? m0 : 0, w + 1 < words ? m1 : 0, j0);
  }
};

// `unit` = (row, kv head, split); false: nothing to do.
__device__ __forceinline__ bool tree_row(const TfdTreeAttnArgs& a, int unit, int splits, int first,
                                         TreeRow& t) {
  t.h = unit / splits % a.kv_heads;
  t.row = unit / splits / a.kv_heads;
  t.G = a.heads / a.kv_heads;
  t.first = first;
  const int count =
      a.counts ? max(0, min(uniform(a.counts)[t.row], a.nodes)) : a.nodes;
  t.cols = count * t.G - first;              // of this block on
  if (t.cols <= 0) return false;
  t.L = uniform(a.lengths)[t.row];
  t.n = t.L + count;
  if (t.L < 0 || (int64_t)t.L + count > (int64_t)a.max_pages * kPage) {
    if (threadIdx.x == 0) raise_error(a.err, kErrPosRange);
    t.L = t.n = 0;
  }
  t.words = (a.nodes + 63) / 64;
  t.table = a.page_table + (int64_t)t.row * a.max_pages;
  t.masks = a.masks + (int64_t)t.row * a.nodes * t.words;
  const int64_t head_size = kPage * a.head_dim;
  t.page_size = a.kv_heads * head_size;
  t.k = (const bf16*)a.k_pool + t.h * head_size;
  t.v = (const bf16*)a.v_pool + t.h * head_size;
  t.last_page = t.n > 0 ? (t.n - 1) / kPage : -1;
  t.num_pages = a.num_pages;
  t.max_pages = a.max_pages;
  t.bad_page = false;
  return true;
}

// A column's softmax goes on with the scores of kN x 16 positions (this lane's 4 kN): the
// reference that exponents count from, and with it what was summed so far, ...  It follows the
// maximum only when that has risen by 2^kMaxRise: probabilities up to 256 are as exact as up
// to 1 (both operands have eight exponent bits), and a rescale of all outputs then is rare.
constexpr float kMaxRise = 8.f;

template <int kN, int DT, int NQ>
__device__ __forceinline__ float tree_maximum(const f32x4 (&st)[kN], float c2, float& mx,
                                              float& sum, f32x4 (&o)[DT][NQ], int qt) {
  float tm = st[0][0];
#pragma unroll
  for (int i = 1; i < 4 * kN; ++i) tm = fmaxf(tm, st[i / 4][i % 4]);
  float lo, hi;
  pair16(tm, lo, hi);
  tm = fmaxf(lo, hi);
  pair32(tm, lo, hi);
  const float m1 = fmaxf(mx, fmaxf(lo, hi));
  if (__any(m1 * c2 > mx * c2 + kMaxRise || (mx == kPanelNegInf && m1 > mx))) {
    const float ref = m1 == kPanelNegInf ? 0.f : m1 * c2;
    const float alpha = __builtin_amdgcn_exp2f(mx * c2 - ref);
    mx = m1;
    sum *= alpha;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[dt][qt][e] *= alpha;
  }
  return mx == kPanelNegInf ? 0.f : mx * c2;
}
// ... and the probabilities of 32 of them as operands: bf16, and with kTwo what that leaves out.
template <bool kTwo>
__device__ __forceinline__ void tree_weights(const f32x4& s0, const f32x4& s1, float c2, float ref,
                                             float& sum, u32x4& hi4, u32x4& lo4) {
  float p[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    p[i] = __builtin_amdgcn_exp2f(fmaf(i < 4 ? s0[i % 4] : s1[i % 4], c2, -ref));
    sum += p[i];
  }
  hi4 = u32x4{pack2(p[0], p[1]), pack2(p[2], p[3]), pack2(p[4], p[5]), pack2(p[6], p[7])};
  if constexpr (!kTwo) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) p[i] -= i % 2 ? bf_hi(hi4[i / 2]) : bf_lo(hi4[i / 2]);
  lo4 = u32x4{pack2(p[0], p[1]), pack2(p[2], p[3]), pack2(p[4], p[5]), pack2(p[6], p[7])};
}

__device__ __forceinline__ float quad_sum(float v) {   // over a column's four lanes
  float lo, hi;
  pair16(v, lo, hi);
  v = lo + hi;
  pair32(v, lo, hi);
  return lo + hi;
}

// A product would take a value that is not finite into every column (0 * inf): such values of
// drafted nodes were left out of it and come in here, where they are seen.  y: dims 16 dt +
// 4 kq .. + 3 of column c; positions j0 .. j1 - 1.
__device__ __forceinline__ void add_odd(TreeRow& t, f32x4& y, int c, int d, int j0, int j1, int D) {
  const uint64_t* const m = t.masks + (int64_t)t.node_of(c) * t.words;
#pragma unroll 1
  for (int j = max(j0, t.L); j < min(j1, t.n); ++j) {
    const int page = t.page_at(j / kPage);
    if (page < 0) continue;
    const u32x2 x =
        *reinterpret_cast<const u32x2*>(t.v + page * t.page_size + (j % kPage) * D + d);
    const bool see = (m[(j - t.L) >> 6] >> ((j - t.L) & 63)) & 1;
    const uint32_t z[2] = {x.x, x.y};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float v = e % 2 ? bf_hi(z[e / 2]) : bf_lo(z[e / 2]);
      if (see && !(fabsf(v) < __builtin_huge_valf())) y[e] += v;
    }
  }
}

// So do the context's, which every column sees: a dim of the output in which the product came
// out not finite is what those values make it, since each has a weight above zero, however small.
// They are looked for then alone: 3 bits of `odd` a dim (D / 8 words in LDS, 8 dims each), +inf,
// -inf and NaN.  All threads of the block; positions j0 .. j1 - 1.
template <int D>
__device__ __forceinline__ void find_odd(TreeRow& t, uint32_t* odd, int j0, int j1) {
  constexpr int kChunks = D / 8;
  const int chunk = threadIdx.x % kChunks, step = blockDim.x / kChunks;
  const int end = min(j1, t.L);
  uint32_t found = 0;
#pragma unroll 4
  for (int j = j0 + (int)threadIdx.x / kChunks; j < end; j += step) {
    const int page = t.page_at(j / kPage);
    const u32x4 x = load16(t.v + max(page, 0) * t.page_size + (j % kPage) * D + 8 * chunk);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t h = e % 2 ? x[e / 2] >> 16 : x[e / 2] & 0xffffu;
      if (page >= 0 && (h & 0x7f80u) == 0x7f80u)
        found |= (h & 0x7fu ? 4u : h >> 15 ? 2u : 1u) << (3 * e);
    }
  }
  if (found) atomicOr(&odd[chunk], found);
}
// ... and put in their dims' places: 4 dims from d on.
__device__ __forceinline__ void put_odd(f32x4& y, const uint32_t* odd, int d) {
  const uint32_t bits = odd[d / 8] >> (3 * (d % 8));
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t b = bits >> (3 * e) & 7;
    if (b) y[e] = b == 1 ? __builtin_huge_valf() : b == 2 ? -__builtin_huge_valf()
                                                         : __builtin_nanf("");
  }
}
// Whether a column's sums may hold such values' products: not finite, of finite probabilities.
template <int DT, int NQ>
__device__ __forceinline__ bool lost(const f32x4 (&o)[DT][NQ], int qt, float sum) {
  float z[4] = {0.f, 0.f, 0.f, 0.f};         // (0 times what is not finite is NaN)
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = fmaf(o[dt][qt][e], 0.f, z[e]);
  return !((z[0] + z[1]) + (z[2] + z[3]) == 0.f) && sum == sum;
}

__device__ __forceinline__ int64_t out_at(const TfdTreeAttnArgs& a, int64_t rr, int head, int d) {
  return a.out_panel ? panel_off(rr, head * a.head_dim + d, a.heads * a.head_dim)
                     : (rr * a.heads + head) * a.head_dim + d;
}

// The block's unit and tile of columns: blocks that read the same keys lie 8 apart, on one XCD.
__device__ __forceinline__ void tree_block(int mtiles, int& unit, int& mt) {
  const int per8 = 8 * mtiles;
  unit = (int)(blockIdx.x / per8) * 8 + (int)(blockIdx.x % 8);
  mt = (int)(blockIdx.x % per8) / 8;
}

// ------------------------------------------------------------------------ few columns
// What a wave's lanes hand each other through LDS lies in order: its LDS operations run in theirs,
// and the compiler moves none past this.
__device__ __forceinline__ void wave_lds() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
}

template <int D, int NQ, int W>
constexpr int few_lds() {
  return 16 * NQ * D * 2 + W * kTile * D * 2;
}

template <int D, int NQ, int W>
__global__ __launch_bounds__(W * kWave, D * NQ <= 64 ? 4 : D * NQ <= 128 ? 3 : 2)
void k_tree_few(TfdTreeAttnArgs a, int splits, int mtiles, float* __restrict__ part_o,
                float* __restrict__ part_ml) {
  constexpr int DS = D / 32, DT = D / 16, kCols = 16 * NQ;
  constexpr int kV = D / 16;                 // V loads of a tile: 1 KiB each
  constexpr int kRowsPerLoad = 512 / D;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float m_s[W][kCols], l_s[W][kCols], inv_s[kCols];
  __shared__ uint32_t far_s[D / 8];
  __shared__ int odd_s, lost_s;
  uint8_t* const q_s = smem;                 // operand order: 1 KiB per (16 columns, 32 dims)
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15, kq = lane >> 4;
  uint8_t* const v_s = smem + kCols * D * 2 + wave * kTile * D * 2;
  int unit, mt;
  tree_block(mtiles, unit, mt);
  if (unit >= a.rows * a.kv_heads * splits) return;
  const int split = unit % splits;
  TreeRow t;
  if (!tree_row(a, unit, splits, mt * kCols, t)) return;
  const int tiles = (t.n + kTile - 1) / kTile;

  u32x4 kr[2][DS], vr[kV];
  auto load_k = [&](int p0, int p1) {
    const bf16* const k0 = t.k + max(p0, 0) * t.page_size + r * D + 8 * kq;
    const bf16* const k1 = t.k + max(p1, 0) * t.page_size + r * D + 8 * kq;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      kr[0][s] = load16(k0 + 32 * s);
      kr[1][s] = load16(k1 + 32 * s);
    }
  };
  auto load_v = [&](int p0, int p1) {
    const bf16* const v0 = t.v + max(p0, 0) * t.page_size + lane * 8;
    const bf16* const v1 = t.v + max(p1, 0) * t.page_size + lane * 8;
#pragma unroll
    for (int i = 0; i < kV / 2; ++i) {
      vr[i] = load16(v0 + i * 512);
      vr[i + kV / 2] = load16(v1 + i * 512);
    }
  };

  const float c2 = a.scale * 1.44269504088896340736f;
  float mx[NQ], sum[NQ];
  f32x4 o[DT][NQ];
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    mx[qt] = kPanelNegInf;
    sum[qt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int slots = splits * W, tile0 = split * W + wave;
  int tile = tile0;
  bool odd = false;                          // a drafted value is not finite
  // lane l holds the page of half l % 2 of this wave's next l / 2-th tile: a scalar load of two
  // would be waited for with the next LDS read
  int ids = 0;
  auto refill = [&](int from) {
    ids = t.page_at(2 * (from + (lane >> 1) * slots) + (lane & 1));
  };
  auto page = [&](int turn, int half) {
    return __builtin_amdgcn_readlane(ids, 2 * (turn % 32) + half);
  };
  refill(tile0);
  int turn = 0, p0 = page(0, 0), p1 = page(0, 1);
  if (tile < tiles) {
    load_v(p0, p1);
    load_k(p0, p1);
  }
  uint64_t see[NQ];                          // (up to 64 nodes)
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) see[qt] = t.masks[t.node_of(16 * qt + r)];
  for (int i = tid; i < kCols * D / 8; i += W * kWave) {
    const int b = i / 64, l = i % 64;        // block b: columns 16 (b / DS), dims 32 (b % DS)
    const int c = t.first + min(16 * (b / DS) + (l & 15), t.cols - 1);
    const int d = 32 * (b % DS) + 8 * (l >> 4);
    *reinterpret_cast<u32x4*>(q_s + i * 16) =
        load16((const bf16*)a.q + t.row * a.q_row + c / t.G * a.q_node +
               (t.h * t.G + c % t.G) * a.q_head + d);
  }
  if (tid == 0) odd_s = lost_s = 0;
  if (tid < D / 8) far_s[tid] = 0;
  __syncthreads();                           // the queries are in place

  for (; tile < tiles; tile += slots) {
    const int j0 = tile * kTile;
    const uint32_t held = (p0 < 0 ? 0u : 0xffffu) | (p1 < 0 ? 0u : 0xffff0000u);
    // drafted positions, or none, in this tile
    const bool edge = j0 + kTile > t.L || held != 0xffffffffu;
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int rr = i * kRowsPerLoad + lane / (D / 8), c8 = lane % (D / 8);
      u32x4 v = vr[i];
      if (edge) v = clean_v(v, j0 + rr, t.L, t.n, (i < kV / 2 ? p0 : p1) >= 0, odd);
      *reinterpret_cast<u32x4*>(v_s + v_at<D>(rr, c8 >> 1) + (c8 & 1) * 16) = v;
    }
    wave_lds();
    const bool more = tile + slots < tiles;
    if (++turn % 32 == 0) refill(tile + slots);
    p0 = page(turn, 0), p1 = page(turn, 1);
    if (more) load_v(p0, p1);
    u32x4 ph[NQ], pl[NQ];
#pragma unroll
    for (int qt = 0; qt < NQ; ++qt) {
      f32x4 st[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int s = 0; s < DS; ++s) {
        const u32x4 qf = *reinterpret_cast<const u32x4*>(q_s + (qt * DS + s) * 1024 + lane * 16);
        st[0] = mfma(kr[0][s], qf, st[0]);
        st[1] = mfma(kr[1][s], qf, st[1]);
      }
      if (edge) {
        const uint32_t bits = (t.seen(j0 - t.L < 64 ? see[qt] : 0, 0, j0) & held) >> (4 * kq);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          st[i / 4][i % 4] = (bits >> (16 * (i / 4) + i % 4)) & 1 ? st[i / 4][i % 4] : kPanelNegInf;
      }
      const float ref = tree_maximum<2, DT, NQ>(st, c2, mx[qt], sum[qt], o, qt);
      tree_weights<true>(st[0], st[1], c2, ref, sum[qt], ph[qt], pl[qt]);
    }
    if (more) load_k(p0, p1);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const u32x4 vf = v_operand<D>(v_s, dt, lane);
#pragma unroll
      for (int qt = 0; qt < NQ; ++qt) o[dt][qt] = mfma(vf, pl[qt], o[dt][qt]);
#pragma unroll
      for (int qt = 0; qt < NQ; ++qt) o[dt][qt] = mfma(vf, ph[qt], o[dt][qt]);
    }
    wave_lds();                              // (the next tile's V goes to the same place)
  }

  // join the waves: maxima and sums, then DT / NQ times 16 dims of all columns at a time
  if (odd) odd_s = 1;
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    sum[qt] = quad_sum(sum[qt]);
    if (lost(o, qt, sum[qt])) lost_s = 1;
    if (kq == 0) {
      m_s[wave][16 * qt + r] = mx[qt];
      l_s[wave][16 * qt + r] = sum[qt];
    }
  }
  __syncthreads();                           // (V's pieces are free from here on)
  const bool far = lost_s;
  if (far) {
    for (int k = split * W; k < tiles; k += slots)
      find_odd<D>(t, far_s, k * kTile, (k + W) * kTile);
    __syncthreads();
  }
  const int64_t pcol = ((int64_t)unit * mtiles + mt) * kCols;
  float scale[NQ];
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    const int c = 16 * qt + r;
    float m = m_s[0][c];
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, m_s[w][c]);
    // (a wave that saw nothing: a sum of zero; a sum of NaN is one whatever its maximum)
    scale[qt] = sum[qt] != sum[qt] ? sum[qt]
                : mx[qt] == kPanelNegInf ? 0.f
                                         : __builtin_amdgcn_exp2f((mx[qt] - m) * c2);
  }
  if (tid < kCols) {
    float m = m_s[0][tid], l = 0.f;
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, m_s[w][tid]);
#pragma unroll
    for (int w = 0; w < W; ++w)
      l += l_s[w][tid] * (m_s[w][tid] == kPanelNegInf
                              ? 1.f
                              : __builtin_amdgcn_exp2f((m_s[w][tid] - m) * c2));
    inv_s[tid] = l == 0.f ? 0.f : 1.f / l;
    if (splits > 1 && tid < t.cols) {
      part_ml[(pcol + tid) * 2] = m;
      part_ml[(pcol + tid) * 2 + 1] = l;
    }
  }
  float* const join = reinterpret_cast<float*>(smem + kCols * D * 2);
  constexpr int kDims = DT / NQ;             // 16 dims each, of a pass
  constexpr int kAll = NQ * kDims * 64;      // values of a pass, in fours
#pragma unroll
  for (int pass = 0; pass < NQ; ++pass) {
    if (pass) __syncthreads();
#pragma unroll
    for (int i = 0; i < kDims; ++i)
#pragma unroll
      for (int qt = 0; qt < NQ; ++qt) {
        f32x4 y = o[pass * kDims + i][qt] * scale[qt];
        if (scale[qt] == 0.f) y = f32x4{0.f, 0.f, 0.f, 0.f};
        *reinterpret_cast<f32x4*>(join + ((wave * NQ + qt) * kDims + i) * 256 + r * 16 + kq * 4) =
            y;
      }
    __syncthreads();
#pragma unroll 1
    for (int i = tid; i < kAll; i += W * kWave) {
      f32x4 y = *reinterpret_cast<const f32x4*>(join + i * 4);
#pragma unroll
      for (int w = 1; w < W; ++w)
        y += *reinterpret_cast<const f32x4*>(join + (w * kAll + i) * 4);
      const int c = 16 * (i / 64 / kDims) + i % 64 / 4;
      const int d = 16 * (pass * kDims + i / 64 % kDims) + i % 4 * 4;
      if (c >= t.cols) continue;
      if (far) put_odd(y, far_s, d);
      if (odd_s)
        for (int k = t.L / kTile; k < tiles; ++k)
          if (k / W % splits == split) add_odd(t, y, c, d, k * kTile, k * kTile + kTile, D);
      if (splits == 1) {
        const float f = inv_s[c];
        if (f == 0.f) y = f32x4{0.f, 0.f, 0.f, 0.f};
        const int cc = t.first + c, node = cc / t.G;
        *reinterpret_cast<u32x2*>((bf16*)a.out + out_at(a, (int64_t)t.row * a.nodes + node,
                                                        t.h * t.G + cc - node * t.G, d)) =
            u32x2{pack2(y[0] * f, y[1] * f), pack2(y[2] * f, y[3] * f)};
      } else {
        *reinterpret_cast<f32x4*>(part_o + (pcol + c) * D + d) = y;
      }
    }
  }
  if (t.bad_page) raise_error(a.err, kErrPageRange);
}

// ----------------------------------------------------------------------- many columns
template <int D, int W>
constexpr int many_tile() {                  // positions: 32 KiB of LDS a tile, 16 of small blocks
  return D <= 128 && W == 8 ? 64 : 32;
}
constexpr int kManyNq = 2;                   // 16s of columns of a wave
constexpr int kStages = 4;                   // tiles of K and V in LDS
template <int D, int W>
constexpr int many_lds() {
  return kStages * 2 * many_tile<D, W>() * D * 2;
}

// 16 bytes a lane from `base` + `at` straight to LDS, 1 KiB from byte `to` on.  Written out: the
// compiler waits for all such loads before it reads any LDS, where here three tiles' stay in
// flight.  There is no register that they write, and what they have written is read behind
// landed() and a barrier.
__device__ __forceinline__ void load_to_lds(const bf16* base, uint32_t at, uint32_t to) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, %2"
      :
      : "s"(to), "v"(at), "s"(base)
      : "memory", "m0");
}
// All but the last kN of this wave's loads have landed.
template <int kN>
__device__ __forceinline__ void landed() {
  asm volatile("s_waitcnt vmcnt(%0)" : : "n"(kN) : "memory");
}

template <int D, int W, bool kTwo>
__global__ __launch_bounds__(W * kWave, 2)
void k_tree_many(TfdTreeAttnArgs a, int splits, int mtiles, float* __restrict__ part_o,
                 float* __restrict__ part_ml) {
  constexpr int NQ = kManyNq, DS = D / 32, DT = D / 16, kPos = many_tile<D, W>();
  constexpr int kCols = 16 * NQ * W, kBytes = kPos * D * 2;
  constexpr int kLoads = kBytes / 1024 / W;  // of K, of V, by a wave: 1 KiB each
  constexpr int kChunks = D / 8;             // 16 bytes each, of a position
  constexpr int kRows = kWave / kChunks;     // positions of a load
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t far_s[D / 8];
  __shared__ int odd_s, lost_s;
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15, kq = lane >> 4;
  int unit, mt;
  tree_block(mtiles, unit, mt);
  if (unit >= a.rows * a.kv_heads * splits) return;
  const int split = unit % splits;
  TreeRow t;
  if (!tree_row(a, unit, splits, mt * kCols, t)) return;
  const int c0 = wave * 16 * NQ;             // this wave's columns, within the block's

  // this split's tiles
  const int tiles = (t.n + kPos - 1) / kPos;
  const int begin = (int)((int64_t)tiles * split / splits);
  const int end = (int)((int64_t)tiles * (split + 1) / splits);

  // Load i of this wave takes positions kRows (i W + wave) .. of a tile; a lane's place in LDS
  // follows from its number, so it loads the 16 bytes that belong there.
  uint32_t k_from[kLoads], v_from[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int row = (i * W + wave) * kRows + lane / kChunks, slot = lane % kChunks;
    const int kc = slot ^ (k_at<D>(row, 0) - row * D * 2) / 16;
    const int vc = slot ^ (v_at<D>(row, 0) - row * D * 2) / 16;
    k_from[i] = (uint32_t)(row % kPage * D + kc * 8) * 2;
    v_from[i] = (uint32_t)(row % kPage * D + vc * 8) * 2;
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)smem;
  // Pages of the next kPages / kPagesOf tiles, in LDS: a scalar load of some would be waited for
  // with the next LDS read, a vector load behind all tiles' loads.
  constexpr int kPagesOf = kPos / kPage, kPages = 1024;
  __shared__ int page_s[kPages];
  auto fill_pages = [&](int tile) {
    for (int i = tid; i < kPages; i += W * kWave) page_s[i] = t.page_at(tile * kPagesOf + i);
  };
  auto load_tile = [&](int tile) {
    const int n = tile - begin;
    const uint32_t buf = lds0 + (uint32_t)(n % kStages) * 2 * kBytes;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int page = max(0, __builtin_amdgcn_readfirstlane(
          page_s[n * kPagesOf % kPages + (i * W + wave) * kRows / kPage]));
      const uint32_t to = buf + (uint32_t)(i * W + wave) * 1024;
      load_to_lds(t.k + page * t.page_size, k_from[i], to);
      load_to_lds(t.v + page * t.page_size, v_from[i], to + kBytes);
    }
  };

  u32x4 qf[NQ][DS];
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    const int c = t.first + min(c0 + 16 * qt + r, t.cols - 1);
    const bf16* const q = (const bf16*)a.q + t.row * a.q_row + c / t.G * a.q_node +
                          (t.h * t.G + c % t.G) * a.q_head + 8 * kq;
#pragma unroll
    for (int s = 0; s < DS; ++s) qf[qt][s] = load16(q + 32 * s);
  }
  const float c2 = a.scale * 1.44269504088896340736f;
  float mx[NQ], sum[NQ];
  f32x4 o[DT][NQ];
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    mx[qt] = kPanelNegInf;
    sum[qt] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt][qt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (tid == 0) odd_s = lost_s = 0;
  if (tid < D / 8) far_s[tid] = 0;
  fill_pages(begin);
  // (the queries are waited for here: else a tile's products would do it, and so wait for the
  // loads of the tiles behind)
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt)
#pragma unroll
    for (int s = 0; s < DS; ++s) asm volatile("" : "+v"(qf[qt][s]));
  // whether any of the pages is not there: then every tile looks for itself which are
  bool gaps = __syncthreads_or(t.bad_page);
#pragma unroll
  for (int i = 0; i + 1 < kStages; ++i)
    if (begin + i < end) load_tile(begin + i);
  constexpr int kTileLoads = 2 * kLoads;     // of a wave
  // tile's loads have landed, those of the tiles behind it may be in flight
  auto wait_for = [&](int tile) {
    if (tile + 2 < end) landed<2 * kTileLoads>();
    else if (tile + 1 < end) landed<kTileLoads>();
    else landed<0>();
  };
  static_assert(kStages == 4, "wait_for counts two tiles behind the one that is read next");
  if (begin < end) wait_for(begin);
  __syncthreads();
  for (int tile = begin; tile < end; ++tile) {
    uint8_t* const buf = smem + (tile - begin) % kStages * 2 * kBytes;
    // (into the buffer of the tile before, which all have read)
    const int ahead = tile + kStages - 1;
    if (ahead < end) {
      if ((ahead - begin) * kPagesOf % kPages == 0) {
        fill_pages(ahead);
        gaps = __syncthreads_or(t.bad_page);
      }
      load_tile(ahead);
    }
    const bool edge = (tile + 1) * kPos > t.L || gaps;
    uint32_t held[kPos / kTile];
#pragma unroll
    for (int kk = 0; kk < kPos / kTile; ++kk) {
      held[kk] = 0xffffffffu;
      if (!gaps) continue;
      const int i = tile * kPagesOf + 2 * kk;
      held[kk] = (t.page_at(i) < 0 ? 0u : 0xffffu) | (t.page_at(i + 1) < 0 ? 0u : 0xffff0000u);
    }
    if (edge) {                              // drafted positions, or none: clean V
      bool odd = false;                      // a drafted value is not finite
#pragma unroll
      for (int i = 0; i < kLoads; ++i) {
        const int at = (i * W + wave) * kWave + lane, row = at / kChunks;
        u32x4* const v = reinterpret_cast<u32x4*>(buf + kBytes + at * 16);
        const uint32_t bits = kPos == kTile || row < kTile ? held[0] : held[kPos / kTile - 1];
        *v = clean_v(*v, tile * kPos + row, t.L, t.n, bits >> row % kTile & 1, odd);
      }
      if (odd) odd_s = 1;
      __syncthreads();
    }
    if (c0 < t.cols) {
      // (operands' places are worked out for every tile: 256 dims leave no registers to hold them)
      int at = lane;
      if (D == 256) asm volatile("" : "+v"(at));
      f32x4 st[NQ][kPos / 16];
#pragma unroll
      for (int qt = 0; qt < NQ; ++qt)
#pragma unroll
        for (int p = 0; p < kPos / 16; ++p) st[qt][p] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < DS; ++s)
#pragma unroll
        for (int p = 0; p < kPos / 16; ++p) {
          const u32x4 kf =
              *reinterpret_cast<const u32x4*>(buf + k_at<D>(16 * p + (at & 15), 4 * s + (at >> 4)));
#pragma unroll
          for (int qt = 0; qt < NQ; ++qt) st[qt][p] = mfma(kf, qf[qt][s], st[qt][p]);
        }
      float ref[NQ];
#pragma unroll
      for (int qt = 0; qt < NQ; ++qt) {
        if (edge) {
#pragma unroll
          for (int kk = 0; kk < kPos / kTile; ++kk) {
            const uint32_t bits =
                (t.seen_by(c0 + 16 * qt + r, tile * kPos + kk * kTile) & held[kk]) >> (4 * kq);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              f32x4& x = st[qt][2 * kk + i / 4];
              x[i % 4] = (bits >> (16 * (i / 4) + i % 4)) & 1 ? x[i % 4] : kPanelNegInf;
            }
          }
        }
        ref[qt] = tree_maximum<kPos / 16, DT, NQ>(st[qt], c2, mx[qt], sum[qt], o, qt);
      }
#pragma unroll
      for (int kk = 0; kk < kPos / kTile; ++kk) {
        u32x4 ph[NQ], pl[NQ];
#pragma unroll
        for (int qt = 0; qt < NQ; ++qt)
          tree_weights<kTwo>(st[qt][2 * kk], st[qt][2 * kk + 1], c2, ref[qt], sum[qt], ph[qt],
                             pl[qt]);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const u32x4 vf = v_operand<D>(buf + kBytes + kk * kTile * D * 2, dt, at);
          if constexpr (kTwo) {
#pragma unroll
            for (int qt = 0; qt < NQ; ++qt) o[dt][qt] = mfma(vf, pl[qt], o[dt][qt]);
          }
#pragma unroll
          for (int qt = 0; qt < NQ; ++qt) o[dt][qt] = mfma(vf, ph[qt], o[dt][qt]);
        }
      }
    }
    if (tile + 1 < end) {
      wait_for(tile + 1);
      __syncthreads();
    }
  }
  const bool odd = odd_s;                    // (set before the last tile's barrier)
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    sum[qt] = quad_sum(sum[qt]);
    if (lost(o, qt, sum[qt])) lost_s = 1;
  }

  const int64_t pcol = ((int64_t)unit * mtiles + mt) * kCols;
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    const int c = c0 + 16 * qt + r;
    const float l = sum[qt], inv = l == 0.f ? 0.f : 1.f / l;
    if (c >= t.cols) continue;
    if (splits > 1 && kq == 0) {
      part_ml[(pcol + c) * 2] = mx[qt];
      part_ml[(pcol + c) * 2 + 1] = l;
    }
    const int cc = t.first + c, node = cc / t.G, head = t.h * t.G + cc - node * t.G;
    const int64_t rr = (int64_t)t.row * a.nodes + node;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int d = 16 * dt + 4 * kq;
      f32x4 y = o[dt][qt];
      if (splits == 1) {
        if (inv == 0.f) y = f32x4{0.f, 0.f, 0.f, 0.f};
        *reinterpret_cast<u32x2*>((bf16*)a.out + out_at(a, rr, head, d)) =
            u32x2{pack2(y[0] * inv, y[1] * inv), pack2(y[2] * inv, y[3] * inv)};
      } else {
        *reinterpret_cast<f32x4*>(part_o + (pcol + c) * D + d) = y;
      }
    }
  }
  __syncthreads();
  const bool far = lost_s;
  if (far) {
    find_odd<D>(t, far_s, begin * kPos, end * kPos);
    __syncthreads();
  }
  if (far || odd) {                          // what a lane has written it reads again
#pragma unroll 1
    for (int c = c0 + r; c < min(c0 + 16 * NQ, t.cols); c += 16) {
      const int cc = t.first + c, node = cc / t.G, head = t.h * t.G + cc - node * t.G;
      const int64_t rr = (int64_t)t.row * a.nodes + node;
#pragma unroll 1
      for (int d = 4 * kq; d < D; d += 16) {
        u32x2* const to = reinterpret_cast<u32x2*>((bf16*)a.out + out_at(a, rr, head, d));
        f32x4* const part = reinterpret_cast<f32x4*>(part_o + (pcol + c) * D + d);
        f32x4 y;
        if (splits == 1) y = f32x4{bf_lo(to->x), bf_hi(to->x), bf_lo(to->y), bf_hi(to->y)};
        else y = *part;
        if (far) put_odd(y, far_s, d);
        if (odd) add_odd(t, y, c, d, begin * kPos, end * kPos, D);
        if (splits == 1) *to = u32x2{pack2(y[0], y[1]), pack2(y[2], y[3])};
        else *part = y;
      }
    }
  }
  if (t.bad_page) raise_error(a.err, kErrPageRange);
}

// ---------------------------------------------------------------------------
// The splits' sums joined: a wave per (row, node, head); lane s holds split s's maximum and
// sum, so that all weights take one round of loads.
// ---------------------------------------------------------------------------
constexpr int kMaxSplits = kWave;

template <int D>
__global__ __launch_bounds__(kBlock) void k_tree_join(TfdTreeAttnArgs a, int splits, int pad_cols,
                                                      const float* __restrict__ part_o,
                                                      const float* __restrict__ part_ml) {
  constexpr int kPer = D / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t i = (int64_t)blockIdx.x * kWavesPerBlock +
                    __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int64_t rr = i / a.heads;
  const int head = (int)(i % a.heads), row = (int)(rr / a.nodes), node = (int)(rr % a.nodes);
  if (row >= a.rows || node >= row_nodes(a.counts, row, a.nodes)) return;
  const int G = a.heads / a.kv_heads, h = head / G, c = node * G + head % G;
  const float c2 = a.scale * 1.44269504088896340736f;
  const int64_t at0 = ((int64_t)row * a.kv_heads + h) * splits * pad_cols + c;
  const int64_t mine = at0 + (int64_t)min(lane, splits - 1) * pad_cols;
  const float ms = part_ml[mine * 2], ls = lane < splits ? part_ml[mine * 2 + 1] : 0.f;
  // (a split that saw nothing: a sum of zero)
  const float m = wave_max(ls == 0.f ? kPanelNegInf : ms);
  const float w = ls == 0.f ? 0.f : ms == kPanelNegInf ? 1.f
                                                       : __builtin_amdgcn_exp2f((ms - m) * c2);
  const float l = wave_sum(ls * w);
  float y[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) y[e] = 0.f;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
    const float* const p = part_o + (at0 + (int64_t)s * pad_cols) * D + lane * kPer;
    float x[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) x[e] = p[e];
#pragma unroll
    for (int e = 0; e < kPer; ++e)
      y[e] += fabsf(x[e]) < __builtin_huge_valf() ? f * x[e] : x[e];
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e)
    ((bf16*)a.out)[out_at(a, rr, head, lane * kPer + e)] = f2bf(l == 0.f ? 0.f : y[e] / l);
}

// How a call runs (all times: one call in a captured graph, 16 heads over 8, 128 dims).
//
// Short: where every wave needs one tile of 32 positions, with 16 columns a block and no more
// blocks than compute units, blocks of as many waves as their registers leave room for.  Two
// tiles a wave instead of two splits save the join's launch: 1 row of 560 positions by 16 nodes
// 11.4 us and 13.2 with the join, of 700, where nearly all waves take a second tile, 13.9 and 14.2;
// 64 dims, 900 by 40 nodes, 10.4 and 11.9; 32 heads over 8, 600 by 8, 11.2 and 13.0; 256 dims,
// whose tiles take longest, 300 by 13, 16.7 and 16.2.  1 row of 6,000 by 16 nodes: 18.0 us, by
// blocks of four waves of 32 columns 24.1; by 8 nodes 16.7 and 19.7.  16 columns whose tiles blocks
// of four waves hold at once too are faster by those (700 positions, 8 nodes: 11.4 us, 13.2),
// down to what a single block holds (200: 10.1, 9.0).
//
// Few: up to 64 columns, 16 of 256 dims, in blocks of four waves of up to 32 (2 rows of 32,000 by
// 32 nodes: 71 us, by the kernel for many 78; 32 rows of 4,096 by 30: 117 and 134; by 48 nodes
// 185 and 137).
// One block a compute unit: what the splits leave is read again, and four waves' loads are
// enough in flight (32 rows of 4,096 by 7 nodes: 97.6 us, with three a unit 104.1; 1 of 6,000 by 8:
// 19.7 and 25.0).
//
// Many: eight waves of 32 columns, whose longer tiles cost less a position (32 rows of 4,096 by 60
// nodes: 145 us, by two blocks of four waves 153); up to 128 columns four waves of 64 dims
// (8 rows of 8,000: 58.2 us, by eight 59.6), or where there are more row heads than compute units
// (33 rows of 400 by 33: 33.0 us, 43.1).  Splits fill the compute units once (twice as many: 4 rows
// of 30,000 by 61 nodes of 32 heads 233 us for 211, 8 of 5,003 by 256 dims 85 for 55).
struct TreePlan {
  int nq, waves, mtiles, cols, splits;       // nq 0: many columns; cols: of a block
};

constexpr int short_waves(int head_dim) { return head_dim == 64 ? 16 : head_dim == 128 ? 12 : 8; }
constexpr int kFewWaves = 4, kFewNodes = 64;

TreePlan tree_plan(int rows, int nodes, int heads, int kv_heads, int head_dim, int max_pages) {
  TreePlan p;
  const int cols = nodes * (heads / kv_heads);
  const int64_t tiles = ((int64_t)max_pages + 1) / 2, units = (int64_t)rows * kv_heads;
  const int64_t cus = compute_units(), mtiles = (cols + 15) / 16, wide = short_waves(head_dim);
  // blocks a row head and 16 columns have to have for one tile a wave
  const int64_t turns = std::min<int64_t>((tiles + wide - 1) / wide, kMaxSplits);
  const int64_t by_four =
      std::min<int64_t>(cus / std::max<int64_t>(units, 1), kMaxSplits) * kFewWaves;
  int64_t per_cu = 1, most;                  // blocks of a compute unit, splits that have work
  if (cols <= 128 && nodes <= kFewNodes && units * mtiles * turns <= cus &&
      (cols > 16 || turns == 1 || tiles > by_four)) {
    p.nq = 1;
    p.waves = (int)wide;
    p.cols = 16;
    most = turns == 2 && cols > 16 ? 1 : turns;
  } else if (cols <= 16 || (cols <= 64 && head_dim <= 128)) {
    p.nq = cols <= 16 ? 1 : 2;
    p.waves = kFewWaves;
    p.cols = 16 * p.nq;
    most = (tiles + p.waves - 1) / p.waves;
  } else {
    const bool four = cols <= 4 * 16 * kManyNq &&
                      (head_dim == 64 || (head_dim == 128 && units > cus));
    p.nq = 0;
    p.waves = four ? 4 : 8;
    p.cols = p.waves * 16 * kManyNq;
    per_cu = 8 / p.waves;
    most = (tiles + 7) / 8;
  }
  p.mtiles = (cols + p.cols - 1) / p.cols;
  const int64_t want = per_cu * cus / std::max<int64_t>(units * p.mtiles, 1);
  p.splits = (int)std::max<int64_t>(std::min({want, most, (int64_t)kMaxSplits}), 1);
  return p;
}

bool tree_shape(int rows, int nodes, int heads, int kv_heads, int head_dim, int max_pages) {
  return rows >= 0 && rows <= 65535 && nodes >= 1 && nodes <= kMaxNodes && kv_heads >= 1 &&
         heads >= kv_heads && heads <= 65535 && heads % kv_heads == 0 && max_pages >= 1 &&
         max_pages <= (1 << 22) && (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

}  // namespace

extern "C" {

int tfd_tree_masks(const int32_t* parents, const int32_t* counts, int rows, int nodes,
                   uint64_t* masks, int32_t* depths, int32_t* err, void* stream) {
  if (rows < 0 || nodes < 1 || nodes > kMaxNodes)
    return fail(kBadShape, "tree_masks: rows=%d nodes=%d (1..%d)", rows, nodes, kMaxNodes);
  if (rows == 0) return 0;
  if (!parents || !masks || !depths) return fail(kBadArg, "tree_masks: null pointer");
  k_tree_masks<<<rows, kMaxNodes, 0, (hipStream_t)stream>>>(parents, counts, nodes, masks, depths,
                                                            err);
  return launched("tree_masks");
}

int tfd_tree_accept(const int32_t* tokens, const int32_t* parents, const int32_t* picks,
                    const int32_t* counts, int rows, int nodes, int32_t* path,
                    int32_t* accepted, int32_t* next, void* stream) {
  if (rows < 0 || nodes < 1 || nodes > kMaxNodes)
    return fail(kBadShape, "tree_accept: rows=%d nodes=%d (1..%d)", rows, nodes, kMaxNodes);
  if (rows == 0) return 0;
  if (!tokens || !parents || !picks || !path || !accepted || !next)
    return fail(kBadArg, "tree_accept: null pointer");
  k_tree_accept<<<rows, kWave, 0, (hipStream_t)stream>>>(tokens, parents, picks, counts, nodes,
                                                         path, accepted, next);
  return launched("tree_accept");
}

int64_t tfd_tree_attn_work_bytes(int rows, int nodes, int heads, int kv_heads, int head_dim,
                                 int max_pages) {
  if (!tree_shape(rows, nodes, heads, kv_heads, head_dim, max_pages) || rows == 0) return 0;
  const TreePlan p = tree_plan(rows, nodes, heads, kv_heads, head_dim, max_pages);
  if (p.splits == 1) return 0;
  return (int64_t)rows * kv_heads * p.splits * p.mtiles * p.cols * (head_dim + 2) * 4;
}

int tfd_tree_attn_form(int rows, int nodes, int heads, int kv_heads, int head_dim, int max_pages,
                       int32_t form[4]) {
  if (!form) return fail(kBadArg, "tree_attn_form: null pointer");
  if (!tree_shape(rows, nodes, heads, kv_heads, head_dim, max_pages) || rows == 0)
    return fail(kBadShape, "tree_attn_form: rows=%d nodes=%d heads=%d kv_heads=%d", rows, nodes,
                heads, kv_heads);
  const TreePlan p = tree_plan(rows, nodes, heads, kv_heads, head_dim, max_pages);
  form[0] = p.nq;
  form[1] = p.waves;
  form[2] = p.mtiles;
  form[3] = p.splits;
  return 0;
}

int tfd_tree_attn(const TfdTreeAttnArgs* args, void* stream) {
  if (!args) return fail(kBadArg, "tree_attn: null args");
  const TfdTreeAttnArgs& a = *args;
  if (!tree_shape(a.rows, a.nodes, a.heads, a.kv_heads, a.head_dim, a.max_pages) ||
      a.num_pages < 1)
    return fail(kBadShape,
                "tree_attn: rows=%d nodes=%d heads=%d kv_heads=%d head_dim=%d max_pages=%d "
                "num_pages=%d",
                a.rows, a.nodes, a.heads, a.kv_heads, a.head_dim, a.max_pages, a.num_pages);
  if (!(a.scale > 0.f) || a.scale > 3.402823466e38f)
    return fail(kBadArg, "tree_attn: scale must be positive and finite");
  if (a.rows == 0) return 0;
  if (!a.q || !a.k_pool || !a.v_pool || !a.page_table || !a.lengths || !a.masks || !a.out)
    return fail(kBadArg, "tree_attn: null pointer");
  if ((uintptr_t)a.q % 16 || a.q_row % 8 || a.q_node % 8 || a.q_head % 8 ||
      (uintptr_t)a.k_pool % 16 || (uintptr_t)a.v_pool % 16 || (uintptr_t)a.out % 16)
    return fail(kBadArg, "tree_attn: q, the pools and out must be 16-byte aligned");
  const TreePlan p = tree_plan(a.rows, a.nodes, a.heads, a.kv_heads, a.head_dim, a.max_pages);
  const int64_t cols = (int64_t)a.rows * a.kv_heads * p.splits * p.mtiles * p.cols;
  if (p.splits > 1 && (!a.work || (uintptr_t)a.work % 16 ||
                       a.work_bytes < cols * (a.head_dim + 2) * 4))
    return fail(kBadArg, "tree_attn: work of %lld bytes", (long long)a.work_bytes);
  const int64_t units = ((int64_t)a.rows * a.kv_heads * p.splits + 7) / 8 * 8;
  if (units * p.mtiles > (1 << 23) || (int64_t)a.rows * a.nodes * a.heads > (1 << 25))
    return fail(kUnsupported, "tree_attn: more than one launch holds");
  float* const po = (float*)a.work;
  float* const pml = po + cols * a.head_dim;
  const unsigned blocks = (unsigned)(units * p.mtiles);
  const int pad = p.mtiles * p.cols;
  const unsigned joins =
      (unsigned)(((int64_t)a.rows * a.nodes * a.heads + kWavesPerBlock - 1) / kWavesPerBlock);
  auto s = (hipStream_t)stream;
  // (past 64 KiB of LDS a kernel has to be allowed)
#define TFD_TREE_RUN(KERNEL, LDS, GRID, THREADS, ...)                                         \
  {                                                                                           \
    constexpr int lds = LDS;                                                                  \
    if (lds > 60000) {                                                                        \
      const hipError_t e = hipFuncSetAttribute((const void*)KERNEL,                           \
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds); \
      if (e != hipSuccess) return fail((int)e, "tree_attn: %s", hipGetErrorString(e));        \
    }                                                                                         \
    KERNEL<<<GRID, THREADS, lds, s>>>(__VA_ARGS__);                                           \
  }
#define TFD_TREE_FEW(D, NQ, W) \
  TFD_TREE_RUN((k_tree_few<D, NQ, W>), (few_lds<D, NQ, W>()), blocks, W * kWave, a, p.splits, \
               p.mtiles, po, pml)
#define TFD_TREE_MANY(D, W)                                                                 \
  if (a.rounded)                                                                            \
    TFD_TREE_RUN((k_tree_many<D, W, false>), (many_lds<D, W>()), blocks, W * kWave, a,      \
                 p.splits, p.mtiles, po, pml)                                               \
  else                                                                                      \
    TFD_TREE_RUN((k_tree_many<D, W, true>), (many_lds<D, W>()), blocks, W * kWave, a,       \
                 p.splits, p.mtiles, po, pml)
#define TFD_TREE_DIM(D)                                                                       \
  {                                                                                           \
    if (p.nq == 1 && p.waves == kFewWaves) TFD_TREE_FEW(D, 1, kFewWaves)                      \
    else if (p.nq == 1) TFD_TREE_FEW(D, 1, short_waves(D))                                    \
    else if (p.nq == 2) {                                                                     \
      if constexpr (D <= 128) TFD_TREE_FEW(D, 2, kFewWaves)                                   \
    } else if (p.waves == 4) {                                                                \
      if constexpr (D <= 128) { TFD_TREE_MANY(D, 4) }                                         \
    } else {                                                                                  \
      TFD_TREE_MANY(D, 8)                                                                     \
    }                                                                                         \
    if (p.splits > 1) k_tree_join<D><<<joins, kBlock, 0, s>>>(a, p.splits, pad, po, pml);     \
  }
  if (a.head_dim == 64) TFD_TREE_DIM(64)
  else if (a.head_dim == 128) TFD_TREE_DIM(128)
  else TFD_TREE_DIM(256)
#undef TFD_TREE_DIM
#undef TFD_TREE_MANY
#undef TFD_TREE_FEW
#undef TFD_TREE_RUN
  return launched("tree_attn");
}

}  // extern "C"
