// Drafted tokens that form a tree: masks, acceptance, and attention over a paged cache.
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
// k may be taken in any order that both operands share).
//
// A wave takes every (4 splits)-th tile of 32 positions (two pages) for 16 NQ columns:
// its K goes from memory into registers as operands, its V through a private piece of LDS, from
// which the transposing read gives V^T's operands.  No barrier until the waves' sums are
// joined; the next tile's loads are in flight behind the current one's products.  V lies in
// LDS by rows, its 32-byte pieces permuted by the row so that the 16 rows of a transposing read
// take the fewest cycles.
//
// Softmax with a running maximum, in f32; a rescale only where a maximum moved.  A
// probability is the sum of two bf16, so that it is not the less exact operand.
// ---------------------------------------------------------------------------
typedef short i16x4 __attribute__((ext_vector_type(4)));
constexpr int kTile = 32;                    // positions

template <int D>
__device__ __forceinline__ int v_swizzle(int row) {
  return D == 64 ? (row >> 1) & 3 : row & 7;
}
// byte of V[row][16 chunk]
template <int D>
__device__ __forceinline__ int v_at(int row, int chunk) {
  return row * D * 2 + ((chunk ^ v_swizzle<D>(row)) << 5);
}

struct TreePlan {
  int nq, mtiles, splits;
};

template <int D, int NQ>
constexpr int tree_lds() {
  const int v = 4 * kTile * D * 2, join = 4 * NQ * 1024;
  return 16 * NQ * D * 2 + (v > join ? v : join);
}

// Blocks of a compute unit that the registers of a variant allow.
template <int D, int NQ>
constexpr int tree_blocks() {
  return D * NQ <= 64 ? 4 : D * NQ <= 128 ? 3 : D * NQ <= 256 ? 2 : 1;
}

// Two bf16 with zeros in the place of infinities and NaN.
__device__ __forceinline__ uint32_t finite_halves(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
  return w;
}

template <int D, int NQ>
__global__ __launch_bounds__(kBlock, (tree_blocks<D, NQ>())) void k_tree_attn(
    TfdTreeAttnArgs a, int splits, int mtiles,
                                                      float* __restrict__ part_o,
                                                      float* __restrict__ part_ml) {
  constexpr int DS = D / 32, DT = D / 16, kCols = 16 * NQ;
  constexpr int kV = D / 16;                 // V loads of a tile: 1 KiB each
  constexpr int kRowsPerLoad = 512 / D;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float ml_s[2][kWavesPerBlock][kCols];
  uint8_t* const q_s = smem;                 // operand order: 1 KiB per (16 columns, 32 dims)
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int r = lane & 15, kq = lane >> 4;
  uint8_t* const v_s = smem + kCols * D * 2 + wave * kTile * D * 2;

  // blocks that read the same keys lie 8 apart: one XCD's L2
  const int per8 = 8 * mtiles;
  const int unit = (int)(blockIdx.x / per8) * 8 + (int)(blockIdx.x % 8);
  const int mt = (int)(blockIdx.x % per8) / 8;
  if (unit >= a.rows * a.kv_heads * splits) return;
  const int split = unit % splits, h = unit / splits % a.kv_heads, row = unit / splits / a.kv_heads;
  const int G = a.heads / a.kv_heads;
  const int count = row_nodes(a.counts, row, a.nodes);
  const int cols = count * G - mt * kCols;   // of this block
  if (cols <= 0) return;
  int L = a.lengths[row];
  const bool bad_length = L < 0 || (int64_t)L + count > (int64_t)a.max_pages * kPage;
  if (bad_length) {
    if (tid == 0) raise_error(a.err, kErrPosRange);
    L = 0;
  }
  const int n = bad_length ? 0 : L + count;
  const int tiles = (n + kTile - 1) / kTile, words = (a.nodes + 63) / 64;
  const int* __restrict__ table = a.page_table + (int64_t)row * a.max_pages;
  const int64_t head_size = kPage * D, page_size = (int64_t)a.kv_heads * head_size;
  const bf16* const kp = (const bf16*)a.k_pool + h * head_size;
  const bf16* const vp = (const bf16*)a.v_pool + h * head_size;
  const int last_page = max(0, (n - 1) / kPage);

  bool page_bad = false;
  auto page_at = [&](int i) {
    const int p = table[min(i, last_page)];
    const bool ok = p >= 0 && p < a.num_pages;
    page_bad |= !ok;
    return ok ? p : 0;
  };

  // the block's queries
  for (int i = tid; i < kCols * D / 8; i += kBlock) {
    const int b = i / 64, l = i % 64;        // block b: columns 16 (b / DS), dims 32 (b % DS)
    const int c = 16 * (b / DS) + (l & 15), d = 32 * (b % DS) + 8 * (l >> 4);
    const int cc = mt * kCols + min(c, cols - 1);
    const int node = cc / G, head = h * G + cc % G;
    *reinterpret_cast<u32x4*>(q_s + i * 16) = load16(
        (const bf16*)a.q + row * a.q_row + node * a.q_node + head * a.q_head + d);
  }

  u32x4 kr[2][DS], vr[kV];
  auto load_k = [&](int p0, int p1) {
    const bf16* const k0 = kp + p0 * page_size + r * D + 8 * kq;
    const bf16* const k1 = kp + p1 * page_size + r * D + 8 * kq;
#pragma unroll
    for (int s = 0; s < DS; ++s) {
      kr[0][s] = load16(k0 + 32 * s);
      kr[1][s] = load16(k1 + 32 * s);
    }
  };
  auto load_v = [&](int p0, int p1) {
    const bf16* const v0 = vp + p0 * page_size + lane * 8;
    const bf16* const v1 = vp + p1 * page_size + lane * 8;
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

  const int slots = splits * kWavesPerBlock;
  const int tile0 = split * kWavesPerBlock + wave;
  int tile = tile0, p0 = 0, p1 = 0;
  bool odd = false;                          // a drafted value is not finite
  if (tile < tiles) {
    p0 = page_at(2 * tile), p1 = page_at(2 * tile + 1);
    load_v(p0, p1);
    load_k(p0, p1);
    p0 = page_at(2 * (tile + slots)), p1 = page_at(2 * (tile + slots) + 1);
  }
  __syncthreads();                           // the queries are in place

  for (; tile < tiles; tile += slots) {
    const int j0 = tile * kTile;
    const bool edge = j0 + kTile > L;        // drafted positions, or none, in this tile
    // V into LDS; positions past the last hold anything and read as zeros, drafted values that
    // are not finite too (below)
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int rr = i * kRowsPerLoad + lane / (D / 8), c8 = lane % (D / 8);
      u32x4 v = vr[i];
      if (edge) {
        if (j0 + rr >= n) v = u32x4{0u, 0u, 0u, 0u};
        if (j0 + rr >= L) {
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const uint32_t f = finite_halves(v[w]);
            odd |= f != v[w];
            v[w] = f;
          }
        }
      }
      *reinterpret_cast<u32x4*>(v_s + v_at<D>(rr, c8 >> 1) + (c8 & 1) * 16) = v;
    }
    const bool more = tile + slots < tiles;
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
        // bit i: this column sees position j0 + i (the context: every one)
        const int node = (mt * kCols + min(16 * qt + r, cols - 1)) / G, from = j0 - L;
        const uint64_t* const mrow = a.masks + ((int64_t)row * a.nodes + node) * words;
        const int w = max(from, 0) >> 6, sh = max(from, 0) & 63;
        const uint64_t m0 = mrow[w], m1 = mrow[min(w + 1, words - 1)];
        uint64_t bits = m0 >> sh;
        if (sh && w + 1 < words) bits |= m1 << (64 - sh);
        if (from < 0) bits = (bits << -from) | ((1ull << -from) - 1);
        if (n - j0 < kTile) bits &= (1ull << (n - j0)) - 1;
        const uint32_t see = (uint32_t)bits >> (4 * kq);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            st[t][e] = (see >> (16 * t + e)) & 1 ? st[t][e] : kPanelNegInf;
      }
      float tm = fmaxf(fmaxf(fmaxf(st[0][0], st[0][1]), fmaxf(st[0][2], st[0][3])),
                       fmaxf(fmaxf(st[1][0], st[1][1]), fmaxf(st[1][2], st[1][3])));
      float lo, hi;
      pair16(tm, lo, hi);
      tm = fmaxf(lo, hi);
      pair32(tm, lo, hi);
      const float m1 = fmaxf(mx[qt], fmaxf(lo, hi));
      const float ref = m1 == kPanelNegInf ? 0.f : m1 * c2;
      if (__any(m1 != mx[qt])) {
        const float alpha = __builtin_amdgcn_exp2f(mx[qt] * c2 - ref);
        mx[qt] = m1;
        sum[qt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[dt][qt][e] *= alpha;
      }
      float p[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        p[i] = __builtin_amdgcn_exp2f(fmaf(st[i / 4][i % 4], c2, -ref));
        sum[qt] += p[i];
      }
      ph[qt] = u32x4{pack2(p[0], p[1]), pack2(p[2], p[3]), pack2(p[4], p[5]), pack2(p[6], p[7])};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        p[i] -= i % 2 ? bf_hi(ph[qt][i / 2]) : bf_lo(ph[qt][i / 2]);
      pl[qt] = u32x4{pack2(p[0], p[1]), pack2(p[2], p[3]), pack2(p[4], p[5]), pack2(p[6], p[7])};
      if (NQ > 2) __builtin_amdgcn_sched_barrier(0);   // (else registers are spilled)
    }
    if (more) {
      load_k(p0, p1);
      p0 = page_at(2 * (tile + 2 * slots)), p1 = page_at(2 * (tile + 2 * slots) + 1);
    }

#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      i16x4 f[2];
#pragma unroll
      for (int t = 0; t < 2; ++t)
        f[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) i16x4*)(v_s +
                v_at<D>(16 * t + 4 * kq + (r >> 2), dt) + (r & 3) * 8));
      const u32x2 f0 = __builtin_bit_cast(u32x2, f[0]), f1 = __builtin_bit_cast(u32x2, f[1]);
      const u32x4 vf = u32x4{f0.x, f0.y, f1.x, f1.y};
#pragma unroll
      for (int qt = 0; qt < NQ; ++qt) {
        o[dt][qt] = mfma(vf, pl[qt], o[dt][qt]);
        o[dt][qt] = mfma(vf, ph[qt], o[dt][qt]);
      }
      if (NQ > 2 && dt % 2) __builtin_amdgcn_sched_barrier(0);
    }
  }
  odd = __any(odd);

  // join the waves: maxima and sums, then 16 dims of all columns at a time
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    float lo, hi, l = sum[qt];
    pair16(l, lo, hi);
    l = lo + hi;
    pair32(l, lo, hi);
    l = lo + hi;
    if (kq == 0) {
      ml_s[0][wave][16 * qt + r] = mx[qt];
      ml_s[1][wave][16 * qt + r] = l;
    }
  }
  __syncthreads();                           // (V's pieces are free from here on)
  float scale[NQ];
#pragma unroll
  for (int qt = 0; qt < NQ; ++qt) {
    const int c = 16 * qt + r;
    float m = ml_s[0][0][c];
#pragma unroll
    for (int w = 1; w < kWavesPerBlock; ++w) m = fmaxf(m, ml_s[0][w][c]);
    // a sum of NaN is one whatever its maximum
    const float l = ml_s[1][wave][c];
    scale[qt] = l != l ? l : mx[qt] == kPanelNegInf ? 0.f
                                                    : __builtin_amdgcn_exp2f((mx[qt] - m) * c2);
  }
  // A product would take a value that is not finite into every column (0 * inf): such values
  // of drafted nodes were left out of it and come in here, where they are seen.
  auto add_odd = [&](f32x4& y, int dt, int qt) {
    const int node = (mt * kCols + min(16 * qt + r, cols - 1)) / G;
    const uint64_t* const mrow = a.masks + ((int64_t)row * a.nodes + node) * words;
#pragma unroll 1
    for (int t = tile0; t < tiles; t += slots)
#pragma unroll 1
      for (int j = max(t * kTile, L); j < min(t * kTile + kTile, n); ++j) {
        const u32x2 x = *reinterpret_cast<const u32x2*>(
            vp + page_at(j / kPage) * page_size + (j % kPage) * D + 16 * dt + 4 * kq);
        const bool see = (mrow[(j - L) >> 6] >> ((j - L) & 63)) & 1;
        const uint32_t z[2] = {x.x, x.y};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v = e % 2 ? bf_hi(z[e / 2]) : bf_lo(z[e / 2]);
          if (see && !(fabsf(v) < __builtin_huge_valf())) y[e] += v;
        }
      }
  };
  float* const join = reinterpret_cast<float*>(smem + kCols * D * 2);
  const int64_t pcol = (int64_t)unit * mtiles * kCols + mt * kCols;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    if (dt) __syncthreads();
#pragma unroll
    for (int qt = 0; qt < NQ; ++qt) {
      f32x4 y = o[dt][qt] * scale[qt];
      if (scale[qt] == 0.f) y = f32x4{0.f, 0.f, 0.f, 0.f};
      if (odd) add_odd(y, dt, qt);
      *reinterpret_cast<f32x4*>(join + (wave * NQ + qt) * 256 + r * 16 + kq * 4) = y;
    }
    __syncthreads();
#pragma unroll
    for (int qt = 0; qt < NQ; ++qt) {
      const int c = 16 * qt + tid / 16, d = 16 * dt + tid % 16;
      float m = ml_s[0][0][c], l = 0.f, y = 0.f;
#pragma unroll
      for (int w = 1; w < kWavesPerBlock; ++w) m = fmaxf(m, ml_s[0][w][c]);
#pragma unroll
      for (int w = 0; w < kWavesPerBlock; ++w) {
        y += join[(w * NQ + qt) * 256 + tid];
        // (nothing seen: a sum of zero)
        const float f = ml_s[0][w][c] == kPanelNegInf
                            ? 1.f
                            : __builtin_amdgcn_exp2f((ml_s[0][w][c] - m) * c2);
        l += ml_s[1][w][c] * f;
      }
      if (c >= cols) continue;
      if (splits == 1) {
        const int cc = mt * kCols + c, node = cc / G, head = h * G + cc % G;
        const float v = l == 0.f ? 0.f : y / l;
        const int64_t rr = (int64_t)row * a.nodes + node;
        const int64_t at = a.out_panel ? panel_off(rr, head * D + d, a.heads * D)
                                       : (rr * a.heads + head) * D + d;
        ((bf16*)a.out)[at] = f2bf(v);
      } else {
        part_o[(pcol + c) * D + d] = y;
        if (dt == 0 && tid % 16 == 0) {
          part_ml[(pcol + c) * 2] = m;
          part_ml[(pcol + c) * 2 + 1] = l;
        }
      }
    }
  }
  if (page_bad && lane == 0) raise_error(a.err, kErrPageRange);
}

// The splits' sums joined: a wave per (row, node, head).
template <int D>
__global__ __launch_bounds__(kBlock) void k_tree_join(TfdTreeAttnArgs a, int splits, int pad_cols,
                                                      const float* __restrict__ part_o,
                                                      const float* __restrict__ part_ml) {
  constexpr int kPer = D / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const int64_t i = (int64_t)blockIdx.x * kWavesPerBlock + threadIdx.x / kWave;
  const int64_t rr = i / a.heads;
  const int head = (int)(i % a.heads), row = (int)(rr / a.nodes), node = (int)(rr % a.nodes);
  if (row >= a.rows || node >= row_nodes(a.counts, row, a.nodes)) return;
  const int G = a.heads / a.kv_heads, h = head / G, c = node * G + head % G;
  const float c2 = a.scale * 1.44269504088896340736f;
  const int64_t first = ((int64_t)row * a.kv_heads + h) * splits;
  float m = kPanelNegInf, l = 0.f, y[kPer];
#pragma unroll
  for (int e = 0; e < kPer; ++e) y[e] = 0.f;
  for (int s = 0; s < splits; ++s) m = fmaxf(m, part_ml[((first + s) * pad_cols + c) * 2]);
  for (int s = 0; s < splits; ++s) {
    const int64_t at = (first + s) * pad_cols + c;
    const float ms = part_ml[at * 2];
    const float ls = part_ml[at * 2 + 1];
    if (ls == 0.f) continue;                 // it saw nothing
    const float w = ms == kPanelNegInf ? 1.f : __builtin_amdgcn_exp2f((ms - m) * c2);
    l += w * ls;
#pragma unroll
    for (int e = 0; e < kPer; ++e) y[e] += w * part_o[at * D + lane * kPer + e];
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const int d = lane * kPer + e;
    const int64_t at = a.out_panel ? panel_off(rr, head * D + d, a.heads * D)
                                   : (rr * a.heads + head) * D + d;
    ((bf16*)a.out)[at] = f2bf(l == 0.f ? 0.f : y[e] / l);
  }
}

TreePlan tree_plan(int rows, int nodes, int heads, int kv_heads, int head_dim, int max_pages) {
  TreePlan p;
  const int cols = nodes * (heads / kv_heads);
  p.nq = cols <= 16 ? 1 : cols <= 32 || head_dim == 256 ? 2 : 4;
  p.mtiles = (cols + 16 * p.nq - 1) / (16 * p.nq);
  const int64_t base = (int64_t)rows * kv_heads * p.mtiles;
  const int64_t tiles = ((int64_t)max_pages + 1) / 2;
  const int64_t want = (3 * (int64_t)compute_units() + base - 1) / base;
  const int64_t most = (tiles + kWavesPerBlock - 1) / kWavesPerBlock;
  p.splits = (int)(want < most ? want : most);
  if (p.splits > 64) p.splits = 64;
  if (p.splits < 1) p.splits = 1;
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
  return (int64_t)rows * kv_heads * p.splits * p.mtiles * 16 * p.nq * (head_dim + 2) * 4;
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
      (uintptr_t)a.k_pool % 16 || (uintptr_t)a.v_pool % 16)
    return fail(kBadArg, "tree_attn: q and the pools must be 16-byte aligned");
  const TreePlan p = tree_plan(a.rows, a.nodes, a.heads, a.kv_heads, a.head_dim, a.max_pages);
  const int64_t cols = (int64_t)a.rows * a.kv_heads * p.splits * p.mtiles * 16 * p.nq;
  if (p.splits > 1 && (!a.work || (uintptr_t)a.work % 16 ||
                       a.work_bytes < cols * (a.head_dim + 2) * 4))
    return fail(kBadArg, "tree_attn: work of %lld bytes", (long long)a.work_bytes);
  const int64_t units = ((int64_t)a.rows * a.kv_heads * p.splits + 7) / 8 * 8;
  if (units * p.mtiles > (1 << 23) || (int64_t)a.rows * a.nodes * a.heads > (1 << 25))
    return fail(kUnsupported, "tree_attn: more than one launch holds");
  float* const po = (float*)a.work;
  float* const pml = po + cols * a.head_dim;
  const dim3 grid((unsigned)(units * p.mtiles));
  auto s = (hipStream_t)stream;
#define TFD_TREE(D, NQ)                                                                       \
  {                                                                                           \
    constexpr int lds = tree_lds<D, NQ>();                                                    \
    if (lds > 65536) {                                                                        \
      const hipError_t e = hipFuncSetAttribute((const void*)k_tree_attn<D, NQ>,               \
                                               hipFuncAttributeMaxDynamicSharedMemorySize, lds); \
      if (e != hipSuccess) return fail((int)e, "tree_attn: %s", hipGetErrorString(e));        \
    }                                                                                         \
    k_tree_attn<D, NQ><<<grid, kBlock, lds, s>>>(a, p.splits, p.mtiles, po, pml);             \
  }
#define TFD_TREE_DIM(D)                                                                       \
  {                                                                                           \
    if (p.nq == 1) TFD_TREE(D, 1)                                                             \
    else if (p.nq == 2) TFD_TREE(D, 2)                                                        \
    else if constexpr (D <= 128) TFD_TREE(D, 4)                                               \
    if (p.splits > 1)                                                                         \
      k_tree_join<D><<<(unsigned)(((int64_t)a.rows * a.nodes * a.heads + kWavesPerBlock - 1) / \
                                  kWavesPerBlock),                                            \
                       kBlock, 0, s>>>(a, p.splits, p.mtiles * 16 * p.nq, po, pml);           \
  }
  if (a.head_dim == 64) TFD_TREE_DIM(64)
  else if (a.head_dim == 128) TFD_TREE_DIM(128)
  else TFD_TREE_DIM(256)
#undef TFD_TREE_DIM
#undef TFD_TREE
  return launched("tree_attn");
}

}  // extern "C"
