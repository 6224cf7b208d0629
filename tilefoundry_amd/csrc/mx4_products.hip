// Products by microscaled 4-bit weights: a projection's, and the routed experts'.
//
// Weights are read as tfd_mx4_pack lays them out (mx4.h).  bf16 rows meet weights
// converted to bf16 in registers, exactly, on the bf16 matrix instruction; rows that
// are microscaled too go with the weights' codes into the scaled one.  Sums are f32
// throughout, each output rounded once.  The weight is the A operand, so a lane ends
// up with four consecutive outputs of one row.
#include <type_traits>

#include "host_common.h"
#include "mx4.h"
#include "tf_decode.h"
#include "tf_mx4.h"

using namespace tfd;
using namespace tfd_host;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

enum XKind { kXBf16 = 0, kXMx4 = 1 };
enum Mode { kDense = 0, kHere = 1, kListed = 2 };   // rows: all; grouped in the block; before
enum Epi { kBf16 = 0, kF32 = 1, kSwiglu = 2, kSwigluTwo = 3 };

constexpr uint32_t kRange = 0x7fffffffu;   // of a row tile's descriptor: offsets up to 2 GiB
constexpr int kHereMax = 128;    // entries that a block groups itself
constexpr int kHereRows = 16;    // rows of a fused step: its mix has a thread for each column

struct Job {
  const uint8_t* x;              // rows, bf16 or codes
  int64_t ldx;                   // bytes
  const uint8_t* xs;             // microscaled rows' scales
  int64_t ldxs;
  const uint8_t* w;              // packed weights
  int64_t w_tiles;               // 16-row tiles of all of them
  int K, kb, N;                  // N: outputs (of one expert)
  int M;                         // dense: rows; experts: entries
  void* out;
  int64_t ldo;
  int vec;                       // four outputs of a row may go in one store
  int whole;                     // dense: items before those that run in quarters
  int slices;                    // dense: parts of K, each with its own f32 rows in out
  int64_t slice;                 // floats from one's rows to the next one's
  int64_t second;                // kSwigluTwo: bytes from a hidden row to its second part
  // experts: entry i is place i % k of row i / k; its row of x is i / div
  const int32_t* ids;
  int ldi, k, div, E;
  const int* groups;             // kListed: tiles, then the entries in their order
  int32_t* err;
};

// The scaled product; a lane's scales are byte kA of sa and byte kB of sb.
template <int kA, int kB>
__device__ __forceinline__ f32x4 mfma_mx4(u32x4 a, uint32_t sa, u32x4 b, uint32_t sb, f32x4 c) {
  const i32x8 x = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8 y = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, kA, (int)sa, kB, (int)sb);
}
// A compile-time loop: f(integral_constant<int, 0>) ... f(integral_constant<int, N - 1>).
template <int N, typename F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (N > 0) {
    unrolled<N - 1>(f);
    f(std::integral_constant<int, N - 1>{});
  }
}

__device__ __forceinline__ u32x4 ld16(const uint8_t* p) {
  return *(const __attribute__((address_space(1))) u32x4*)p;
}
__device__ __forceinline__ u32x4 ld16_stream(const uint8_t* p) {
  return __builtin_nontemporal_load((const __attribute__((address_space(1))) u32x4*)p);
}
__device__ __forceinline__ uint32_t ld1(const uint8_t* p) {
  return *(const __attribute__((address_space(1))) uint8_t*)p;
}

// ---------------------------------------------------------------------------
// Entries (row, place) grouped by expert in tiles of kWidth, by the block that uses
// them: up to kHereMax entries, each compared with those before it, which costs less
// than a launch of its own.  Ids outside the experts make no entry; any but -1 raises
// the error bit.
// ---------------------------------------------------------------------------
struct Tiles {
  int n, first_wave;
  int id[kHereMax], rank[kHereMax];
  int expert[kHereMax], count[kHereMax];
  uint8_t tile[kHereMax];
  uint8_t entry[kHereMax][16];
};

template <int kWidth>              // entries of a tile at most
__device__ void group_here(const Job& a, Tiles& s) {
  const int i = threadIdx.x, lane = i & (kWave - 1);
  int id = -1;
  if (i < kHereMax) {
    if (i < a.M) {
      id = a.ids[(int64_t)(i / a.k) * a.ldi + i % a.k];
      if (id < 0 || id >= a.E) {
        if (id != -1 && blockIdx.x == 0 && a.err) raise_error(a.err, kErrTokenRange);
        id = -1;
      }
    }
    s.id[i] = id;
    s.count[i] = 0;
  }
  __syncthreads();
  int rank = 0, first = i;
  if (id >= 0)
    for (int j = i - 1; j >= 0; --j)
      if (s.id[j] == id) {
        ++rank;
        first = j;
      }
  const bool leads = id >= 0 && rank % kWidth == 0;
  const uint64_t before = __ballot(leads);
  if (i < kHereMax) s.rank[i] = rank;
  if (i == 0) s.first_wave = __popcll(before);
  __syncthreads();
  int t = 0;
  if (i < kHereMax) {
    const int base = i < kWave ? 0 : s.first_wave;
    t = base + __popcll(before & ((1ull << lane) - 1));
    if (leads) {
      s.tile[i] = (uint8_t)t;
      s.expert[t] = id;
    }
    if (i == kHereMax - 1) s.n = base + __popcll(before);
  }
  __syncthreads();
  if (id >= 0) {
    int lead = first;
    if (rank >= kWidth)
      for (lead = first; s.id[lead] != id || s.rank[lead] != rank - rank % kWidth;) ++lead;
    t = s.tile[lead];
    s.entry[t][rank % kWidth] = (uint8_t)i;
    atomicMax(&s.count[t], rank % kWidth + 1);
  }
  __syncthreads();
}

// The tile of expert rows that item `rt` works on (the same for a whole wave, and held so).
template <int kMode>
struct RowTile {
  int expert, count;
  int first;                     // kDense: row; kListed: place in the order
  __device__ __forceinline__ RowTile(const Job& a, const Tiles* s, int rt, int rows) {
    if (kMode == kDense) {
      expert = 0;
      first = rt * rows;
      count = min(rows, a.M - first);
    } else if (kMode == kHere) {
      expert = __builtin_amdgcn_readfirstlane(s->expert[rt]);
      first = rt;
      count = __builtin_amdgcn_readfirstlane(s->count[rt]);
    } else {
      const int* t = a.groups + 4 + rt * 4;
      expert = __builtin_amdgcn_readfirstlane(t[0]);
      first = __builtin_amdgcn_readfirstlane(t[1]);
      count = __builtin_amdgcn_readfirstlane(t[2]);
    }
  }
  // the i-th row's place: a row of the dense product, or an entry (past the end: the last)
  __device__ __forceinline__ int at(const Job& a, const Tiles* s, int i, int tiles) const {
    i = min(i, count - 1);
    if (kMode == kDense) return first + i;
    if (kMode == kHere) return s->entry[first][i];
    return a.groups[4 + tiles * 4 + first + i];
  }
};

// The row tiles that fit a list's head, as k_mx4_group wrote it there.
__device__ __forceinline__ int listed_room(const Job& a) { return a.groups[1]; }

template <int kEpi>
__device__ __forceinline__ void put(const Job& a, int row, int n, f32x4 v, int slice = 0) {
  if (kEpi == kSwiglu || kEpi == kSwigluTwo) {
    // (gate, up) pairs.  The hidden value is the next product's operand, hence bf16, or in a
    // step of few rows the sum of two bf16 (2^-17): its matrix tiles have rows to spare, so
    // the only rounding to bf16 that counts is the output's.  An infinity has no second part.
    const float h0 = silu_f(v.x) * v.y, h1 = silu_f(v.z) * v.w;
    bf16* o = (bf16*)a.out + (int64_t)row * a.ldo + n / 2;
    const uint32_t first = pack2(h0, h1);
    *reinterpret_cast<uint32_t*>(o) = first;
    if (kEpi == kSwigluTwo) {
      const float f0 = bf_lo(first), f1 = bf_hi(first);
      const float r0 = fabsf(f0) < __builtin_huge_valf() ? h0 - f0 : 0.f;
      const float r1 = fabsf(f1) < __builtin_huge_valf() ? h1 - f1 : 0.f;
      *reinterpret_cast<uint32_t*>((uint8_t*)o + a.second) = pack2(r0, r1);
    }
    return;
  }
  if (kEpi == kF32) {
    float* o = (float*)a.out + slice * a.slice + (int64_t)row * a.ldo + n;
    if (a.vec && n + 4 <= a.N) {
      *reinterpret_cast<f32x4*>(o) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < a.N) o[i] = v[i];
    }
    return;
  }
  bf16* o = (bf16*)a.out + (int64_t)row * a.ldo + n;
  if (a.vec && n + 4 <= a.N) {
    *reinterpret_cast<u32x2*>(o) = u32x2{pack2(v.x, v.y), pack2(v.z, v.w)};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < a.N) o[i] = f2bf(v[i]);
  }
}

// ---------------------------------------------------------------------------
// Few rows: the weights' stream bounds it.  An item is a tile of MT x 16 rows by TN
// column tiles over all of K.  With kSplit items are dealt to the blocks in turn, and a
// block's waves split K and meet in LDS (few items, or a long K); without, each wave takes
// items of its own.  A wave has the next D steps' (128 k) weights, scales and rows in
// flight across items, so the stream does not stop where an item ends.  Rows come straight
// from memory (L2), once for TN column tiles.
// Measured: one row x 2048 x 12288 5.5 us (2.4 TB/s: the launch and one round of loads), the
// gate/up of eight Granite rows 26.7 us (170 MB, 6.3 TB/s from the last-level cache).
// ---------------------------------------------------------------------------
template <int kX, int MT, int TN, int D, int kMode, int kEpi, int kWaves = 4, bool kSplit = true>
__global__ __launch_bounds__(kWaves * kWave) void k_mx4_few(Job a) {
  constexpr int kR = 16 * MT;
  __shared__ f32x4 red[kSplit ? 2 : 1][kSplit ? kWaves : 1][kSplit ? MT * TN : 1]
                      [kSplit ? kWave : 1];
  __shared__ typename std::conditional<kMode == kHere, Tiles, int>::type group_s;
  const Tiles* tiles = nullptr;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int nl = lane & 15, kq = lane >> 4;
  int nT, room = 0;
  if constexpr (kMode == kHere) {
    group_here<16>(a, group_s);
    tiles = &group_s;
    nT = group_s.n;
  } else if (kMode == kListed) {
    nT = a.groups[0];
    room = listed_room(a);
  } else {
    nT = (a.M + kR - 1) / kR;
  }
  const int ntiles = (a.N + 15) / 16;
  const int nC = (ntiles + TN - 1) / TN;
  const int items = nT * nC;
  const int G = (int)gridDim.x * (kSplit ? 1 : kWaves);
  const int me = kSplit ? (int)blockIdx.x : (int)blockIdx.x * kWaves + wave;
  if (me >= items) return;
  const int mine = (items - 1 - me) / G + 1;
  // steps of a wave's part of K
  const int ns = kSplit ? (a.kb + kWaves - 1) / kWaves : a.kb;
  const int k0 = kSplit ? wave * ns : 0;
  const int sg = mx4_scale_groups(a.kb);
  const uint8_t* scales = a.w + a.w_tiles * a.kb * 1024;

  struct Item {
    int64_t tile[TN];
    const uint8_t *x[MT], *xs[MT];
  };
  auto decode = [&](int j) {
    const int it = me + j * G, rt = it % nT, c = it / nT;
    const RowTile<kMode> r(a, tiles, rt, kR);
    Item d;
#pragma unroll
    for (int t = 0; t < TN; ++t)
      d.tile[t] = (int64_t)r.expert * ntiles + min(c * TN + t, ntiles - 1);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int at = r.at(a, tiles, m * 16 + nl, room);
      const int64_t row = kMode == kDense ? at : at / a.div;
      d.x[m] = a.x + row * a.ldx;
      d.xs[m] = kX == kXMx4 ? a.xs + row * a.ldxs : nullptr;
    }
    return d;
  };
  u32x4 w[D][TN];
  uint32_t ws[D][TN];
  constexpr int kXr = kX == kXMx4 ? 1 : 4;      // 16-byte registers of a row's step
  u32x4 x[D][MT][kXr];
  uint32_t xs[D][MT];
  Item nx = decode(0);
  int jn = 0, sn = 0;
  auto issue = [&](int u) {
    const int b = min(k0 + sn, a.kb - 1);
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      w[u][t] = ld16_stream(a.w + (nx.tile[t] * a.kb + b) * 1024 + lane * 16);
      ws[u][t] = ld1(scales + (nx.tile[t] * sg + (b >> 2)) * 256 + lane * 4 + (b & 3));
    }
    // a lane's 32 k; those past K read the row's first and are cleared before use.  (Loads of
    // 64 bytes of a row by four lanes, transposed by lane swaps, measured no faster: 19 rows
    // 10.6 us for 10.4, eight rows' experts 52 for 48.)
    const int k = b * kMx4K + 32 * kq, kk = k < a.K ? k : 0;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (kX == kXMx4) {
        x[u][m][0] = ld16(nx.x[m] + (kk >> 1));
        xs[u][m] = ld1(nx.xs[m] + (kk >> 5));
      } else {
#pragma unroll
        for (int s = 0; s < kXr; ++s) x[u][m][s] = ld16(nx.x[m] + 2 * kk + 16 * s);
      }
    }
    if (++sn == ns && jn + 1 < mine) {
      sn = 0;
      nx = decode(++jn);
    }
  };
  f32x4 c[TN][MT];
#pragma unroll
  for (int t = 0; t < TN; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) c[t][m] = f32x4{0.f, 0.f, 0.f, 0.f};
  int jc = 0, sc = 0;
  auto compute = [&](int u) {
    const int b = k0 + sc;
    if (b < a.kb) {
      if (b == a.kb - 1 && b * kMx4K + 32 * kq >= a.K) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
#pragma unroll
          for (int s = 0; s < kXr; ++s) x[u][m][s] = u32x4{0u, 0u, 0u, 0u};
          xs[u][m] = 127;
        }
      }
      if (kX == kXMx4) {
#pragma unroll
        for (int t = 0; t < TN; ++t)
#pragma unroll
          for (int m = 0; m < MT; ++m)
            c[t][m] = mfma_mx4<0, 0>(w[u][t], ws[u][t], x[u][m][0], xs[u][m], c[t][m]);
      } else {
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          const float scale = mx4_scale(ws[u][t]);
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const u32x4 v = fp4x8_to_bf16(w[u][t][s], scale);
#pragma unroll
            for (int m = 0; m < MT; ++m) c[t][m] = mfma(v, x[u][m][kX == kXMx4 ? 0 : s], c[t][m]);
          }
        }
      }
    }
    if (++sc < ns) return;
    // the item is done: the parts of K meet in LDS (two buffers, so one barrier an
    // item is enough) and the waves take turns to write
    const int j = jc++;
    sc = 0;
    if (kSplit) {
#pragma unroll
      for (int t = 0; t < TN; ++t)
#pragma unroll
        for (int m = 0; m < MT; ++m) red[j & 1][wave][t * MT + m][lane] = c[t][m];
      __syncthreads();
    }
    const int it = me + j * G, rt = it % nT, cc = it / nT;
    const RowTile<kMode> r(a, tiles, rt, kR);
#pragma unroll
    for (int q = 0; q < TN * MT; ++q) {
      const int t = q / MT, m = q % MT;
      f32x4 v = c[t][m];
      c[t][m] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (kSplit) {
        if ((q + j) % kWaves != wave) continue;
        v = red[j & 1][0][q][lane];
#pragma unroll
        for (int p = 1; p < kWaves; ++p) v += red[j & 1][p][q][lane];
      }
      const int n = (cc * TN + t) * 16 + 4 * kq;
      if (m * 16 + nl < r.count && cc * TN + t < ntiles && n < a.N)
        put<kEpi>(a, r.at(a, tiles, m * 16 + nl, room), n, v);
    }
  };
  const int total = mine * ns;
#pragma unroll
  for (int u = 0; u < D; ++u) issue(u);
  int q0 = 0;
  for (; q0 + D < total; q0 += D) {
#pragma unroll
    for (int u = 0; u < D; ++u) {
      compute(u);
      issue(u);
    }
  }
#pragma unroll
  for (int u = 0; u < D; ++u)
    if (q0 + u < total) compute(u);
}

// ---------------------------------------------------------------------------
// Many rows.  A block of four waves takes up to TM x 16 rows by 4 x TN x 16 columns.
// Its rows pass through LDS, a stage (128 k of bf16, 256 k of codes) at a time in two
// buffers, in the order the matrix instruction takes them (a wave's read is 1 KiB in a row,
// and a write's eight lanes are 128 bytes in a row: no bank conflicts; those of microscaled
// rows' scales, a byte a lane, are 18% of that product's LDS cycles); each wave's own weights go straight to its registers, two blocks of 128 k
// ahead, and are converted there.  bf16 rows come in two halves, each loaded and written
// beside the products of half a stage: with all in flight at once the kernel needs more
// than the 256 registers at which two blocks share a compute unit.  (DMA into LDS needs
// none, but every LDS read behind it waits for it.)
// Measured: 4,001 x 2048 x 12288 of bf16 146 to 157 us (1,280 to 1,380 TFLOP/s; 4,096 x 8192 x
// 8192 1,550; a large library product of bf16 reaches 1,413 here): the matrix cores, busy 57%
// of a profiled launch, and the ends of a pipeline of 16 blocks of k.  4,001 x 4096 x
// 8512 of codes 92 us (3,000 TFLOP/s): nothing is full there.  Matrix instructions take 31%
// of the time, the VALU 26%, LDS 17%; L2 is asked every 2.4 cycles a channel (about 15 bytes
// a cycle and compute unit, 86% hits).  Of the waves' time 46% waits to issue, 23% for loads,
// LDS or barriers: the order of two waves a SIMD, not a rate, keeps it there.
// ---------------------------------------------------------------------------
template <int kX, int TM>
struct ManyLds {
  static constexpr int kBlocks = kX == kXMx4 ? 2 : 1;               // of 128 k in a stage
  static constexpr int kBytes = TM * (kX == kXMx4 ? 1024 : 4096);   // of a block
  // a lane's scales of all row tiles and blocks side by side: one read gives them all
  static constexpr int kScPad = kBlocks * TM;
  static constexpr int kScales = kX == kXMx4 ? kScPad * kWave : 0;
  static constexpr int kTotal = 2 * (kBlocks * kBytes + kScales);   // rows, then scales
};

// One item: a row tile `r` of at most TM x 16 rows, column block `cb` and, of a dense product
// of few blocks, part `slice` of K (whole fours of 128 k).
template <int kX, int TM, int TN, int kMode, int kEpi>
__device__ __forceinline__ void many_item(const Job& a, const RowTile<kMode>& r, int room, int cb,
                                          int slice, uint8_t* lds) {
  constexpr bool kMx = kX == kXMx4;
  using Lds = ManyLds<kX, TM>;
  constexpr int KC = Lds::kBlocks, kScPad = Lds::kScPad;
  static_assert(!kMx || kScPad % 8 == 0, "whole pieces, and a lane's scales of a stage one read");
  const int quads = mx4_scale_groups(a.kb), slices = kMode == kDense ? a.slices : 1;
  const int q_first = quads * slice / slices, q_last = quads * (slice + 1) / slices;
  const int b_last = min(4 * q_last, a.kb);
  constexpr int kPieces = kMx ? (KC * TM + 3) / 4 : (TM + 1) / 2;   // loads in flight a thread
  const int tid = threadIdx.x, lane = tid & (kWave - 1);
  auto xs_s = [&](int buf) { return lds + buf * (KC * Lds::kBytes); };
  auto xsc_s = [&](int buf) { return lds + 2 * KC * Lds::kBytes + buf * Lds::kScales; };
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int nl = lane & 15, kq = lane >> 4;
  const int ntiles = (a.N + 15) / 16;
  const int sg = mx4_scale_groups(a.kb);
  const uint8_t* scales = a.w + a.w_tiles * a.kb * 1024;

  // Eight lanes of a load take 128 bytes of one row, a whole cache line: rows a power of two
  // apart share a set of the L1, which keeps no line until another wave wants its other half
  // (64 bytes of 16 rows: 203 us for 4,001 x 2048 x 12288, 171 on padded rows).  bf16: of row
  // tile m, rows 2 (lane / 8) + wave % 2, k 64 (wave / 2) + 8 (lane % 8); codes: piece q
  // is rows 2 (lane / 8) + i % 2 of row tile i / 2, i = 4 q + wave, both blocks of a stage.
  // 32-bit offsets from a base that all lanes share (the entries check that they fit).
  const uint8_t* xb = a.x + (kMode == kDense ? r.first * a.ldx : 0);
  const uint8_t* xsb = kMx ? a.xs + (kMode == kDense ? r.first * a.ldxs : 0) : nullptr;
  auto offset = [&](int i, int64_t ld) {
    const int at = r.at(a, nullptr, i, room);
    return (uint32_t)(kMode == kDense ? at - r.first : at / a.div) * (uint32_t)ld;
  };
  const int lr = lane >> 3, lp = lane & 7;
  // scale bytes: of row tile (4 q + wave) % TM, row nl, 32 k group kq of block (4 q + wave) / TM
  constexpr int kScTiles = kMx ? TM / 4 : 1;
  uint32_t xo[kMx ? kPieces : TM], xso[kScTiles];
#pragma unroll
  for (int q = 0; q < (kMx ? kPieces : TM); ++q) {
    const int i = kMx ? q * 4 + wave : 2 * q + (wave & 1);
    xo[q] = offset((i >> 1) * 16 + 2 * lr + (i & 1), a.ldx) + 16 * lp +
            (kMx ? 0 : 128 * (wave >> 1));
    if (kMx && q < kScTiles) xso[q] = offset(i * 16 + nl, a.ldxs);
  }
  u32x4 xr[kPieces];
  uint32_t xsr[kMx ? kPieces : 1];
  // pieces past K, and past the last block, are out of the descriptors' range: zeros (a zero
  // scale byte is 2^-127) without a branch between a load and its use
  const auto xrs = rsrc_bounded(xb, kRange);
  const auto xsrs = rsrc_bounded(xsb, kRange);
  auto load_x = [&](int half, int b0) {
    if (kMx) {
      const bool in = b0 * kMx4K + 32 * lp < a.K;
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        const int k = (b0 + (q * 4 + wave) / TM) * kMx4K + 32 * kq;
        xr[q] = __builtin_amdgcn_raw_buffer_load_b128(xrs, in ? xo[q] : kOutOfRange, b0 * 64, 0);
        xsr[q] = __builtin_amdgcn_raw_buffer_load_b8(
            xsrs, k < a.K ? xso[q % kScTiles] + (k >> 5) : kOutOfRange, 0, 0);
      }
    } else {
      const bool in = b0 * kMx4K + 64 * (wave >> 1) + 8 * lp < a.K;
#pragma unroll
      for (int q = 0; q < kPieces; ++q) {
        const int m = half * kPieces + q;
        if (m < TM)
          xr[q] = __builtin_amdgcn_raw_buffer_load_b128(xrs, in ? xo[m] : kOutOfRange,
                                                        2 * b0 * kMx4K, 0);
      }
    }
  };
  // Where 16 bytes lie in LDS: 1 KiB for the 64 lanes of an operand, lane (row, 32 k group)
  // at row ^ f + 16 group.  A 16-byte access is served for lanes 0-3, 12-15, 20-23 and 24-27
  // of 32 together, then the others, without conflict where their places differ mod 16.  A
  // row's eight pieces go to four operands (or groups) times two groups (or blocks) of f 0..3
  // and 12 apart: with even or odd rows in a load those lanes' places differ, and a read,
  // whose lanes' f differ by 0..3 or 12 only, takes them as rows in a row would lie.
  auto operand = [&](int buf, int i, int row, int group, int f) {
    return &xs_s(buf)[i * 1024 + ((row ^ f) + 16 * group) * 16];
  };
  auto stage = [&](int half, int buf) {
#pragma unroll
    for (int q = 0; q < kPieces; ++q) {
      if (kMx) {
        const int i = q * 4 + wave;
        *reinterpret_cast<u32x4*>(operand(buf, (lp >> 2) * TM + (i >> 1), 2 * lr + (i & 1),
                                          lp & 3, (lp & 3) + 12 * (lp >> 2))) = xr[q];
        xsc_s(buf)[lane * kScPad + i] = (uint8_t)xsr[q];
      } else {
        const int m = half * kPieces + q, group = 2 * (wave >> 1) + (lp >> 2);
        if (m < TM)
          *reinterpret_cast<u32x4*>(operand(buf, m * 4 + (lp & 3), 2 * lr + (wave & 1), group,
                                            (lp & 3) + 12 * (group & 1))) = xr[q];
      }
    }
  };
  int64_t wt[TN];
#pragma unroll
  for (int t = 0; t < TN; ++t)
    wt[t] = (int64_t)r.expert * ntiles + min((cb * 4 + wave) * TN + t, ntiles - 1);
  // two blocks' codes ahead; the scales of four blocks are one dword
  u32x4 w[2][TN];
  uint32_t ws[TN], ws_next[TN];
  auto load_w = [&](int u, int b) {
    const int64_t at = min(b, b_last - 1);
#pragma unroll
    for (int t = 0; t < TN; ++t)
      w[u][t] = ld16(a.w + (wt[t] * a.kb + at) * 1024 + lane * 16);
  };
  auto load_ws = [&](int q) {
    const int64_t at = min(q, q_last - 1);
#pragma unroll
    for (int t = 0; t < TN; ++t)
      ws_next[t] = *(const __attribute__((address_space(1))) uint32_t*)(
          scales + (wt[t] * sg + at) * 256 + lane * 4);
  };
  f32x4 c[TM][TN];
#pragma unroll
  for (int m = 0; m < TM; ++m)
#pragma unroll
    for (int t = 0; t < TN; ++t) c[m][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  load_x(0, 4 * q_first);
  load_ws(q_first);
  load_w(0, 4 * q_first);
  load_w(1, 4 * q_first + 1);
  stage(0, 0);
  if (!kMx) {
    load_x(1, 4 * q_first);
    stage(1, 0);
  }
  __syncthreads();
  int buf = 0;
  uint32_t vs[kScPad > 8 ? kScPad / 4 : 2];
  // the 128 k of block b, the j-th of its four: weights in slot j % 2, rows in the current
  // buffer; the slot is refilled behind its use
  auto products = [&](auto jth, int b) {
    constexpr int j = decltype(jth)::value, u = j % 2;
    if constexpr (kMx) {
      u32x4 v[TM];
#pragma unroll
      for (int m = 0; m < TM; ++m)
        v[m] = *reinterpret_cast<const u32x4*>(operand(buf, u * TM + m, nl, kq, kq + 12 * u));
      unrolled<TN>([&](auto t) {
        unrolled<TM>([&](auto m) {
          constexpr int i = u * TM + m.value;
          c[m.value][t.value] = mfma_mx4<j, i % 4>(w[u][t.value], ws[t.value], v[m.value],
                                                   vs[i / 4], c[m.value][t.value]);
        });
      });
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        if (s % 2 == 0) load_x(s / 2, b + 1);
        u32x4 v[TM];
#pragma unroll
        for (int m = 0; m < TM; ++m)
          v[m] = *reinterpret_cast<const u32x4*>(
              operand(buf, m * 4 + s, nl, kq, s + 12 * (kq & 1)));
#pragma unroll
        for (int t = 0; t < TN; ++t) {
          const u32x4 q = fp4x8_to_bf16(w[u][t][s], mx4_scale((ws[t] >> (8 * j)) & 0xffu));
#pragma unroll
          for (int m = 0; m < TM; ++m) c[m][t] = mfma(q, v[m], c[m][t]);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (s % 2 == 1) stage(s / 2, 1 - buf);
        // keeps the next step's LDS reads from being gathered here: registers
        asm volatile("" ::: "memory");
      }
    }
    load_w(u, b + 2);
    __builtin_amdgcn_sched_barrier(0);
  };
  auto turn = [&] {
    __syncthreads();
    buf = 1 - buf;
  };
  // blocks b and b + 1, the j-th two of four
  auto two = [&](auto jth, int b) {
    constexpr int j = decltype(jth)::value;
    if constexpr (kMx) {
      load_x(0, b + 2);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kScPad == 16) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(&xsc_s(buf)[lane * kScPad]);
        vs[0] = v.x, vs[1] = v.y, vs[2] = v.z, vs[3] = v.w;
      } else {
        const u32x2 v = *reinterpret_cast<const u32x2*>(&xsc_s(buf)[lane * kScPad]);
        vs[0] = v.x, vs[1] = v.y;
      }
    }
    products(std::integral_constant<int, 2 * j>{}, b);
    if (b + 1 < b_last) {
      if (!kMx) turn();
      products(std::integral_constant<int, 2 * j + 1>{}, b + 1);
    }
    if (kMx) stage(0, 1 - buf);
    turn();
  };
  for (int q = q_first; q < q_last; ++q) {
#pragma unroll
    for (int t = 0; t < TN; ++t) ws[t] = ws_next[t];
    load_ws(q + 1);
    two(std::integral_constant<int, 0>{}, 4 * q);
    if (4 * q + 2 < b_last) two(std::integral_constant<int, 1>{}, 4 * q + 2);
  }
#pragma unroll
  for (int m = 0; m < TM; ++m) {
    const int i = m * 16 + nl;
    if (i >= r.count) continue;
    const int at = r.at(a, nullptr, i, room);
#pragma unroll
    for (int t = 0; t < TN; ++t) {
      const int tile = (cb * 4 + wave) * TN + t, n = tile * 16 + 4 * kq;
      if (tile < ntiles && n < a.N) put<kEpi>(a, at, n, c[m][t], slice);
    }
  }
}

template <int kX, int TM, int TN, int kMode, int kEpi>
__global__ __launch_bounds__(kBlock, TM * TN > 16 ? 2 : 3) void k_mx4_many(Job a, int nT_host) {
  __shared__ __align__(16) uint8_t lds[ManyLds<kX, TM>::kTotal];
  const int nT = kMode == kListed ? a.groups[0] : nT_host;
  const int room = kMode == kListed ? listed_room(a) : 0;
  const int ntiles = (a.N + 15) / 16;
  const int nC = (ntiles + 4 * TN - 1) / (4 * TN);
  // Blocks go to the XCDs in turn, and what an XCD's blocks share stays in its L2.  Dense:
  // an XCD has a run of items, eight row tiles by a few column blocks at a time, then its
  // part of the items that run in quarters (64 rows by half the columns).  Lists: an
  // XCD has every eighth row tile with all its columns, so that all get their part of the
  // large ones.
  const int xcd = blockIdx.x & 7, local = blockIdx.x >> 3;
  int rt, cb, slice = 0, quarter = -1;
  if (kMode == kListed) {
    rt = local / nC * 8 + xcd;
    cb = local % nC;
    if (rt >= nT) return;
  } else {
    const int total = nT * nC * a.slices, per = (a.whole + 7) / 8;
    int g = xcd * per + local;
    if (local >= per) {
      const int parts = 4 * (total - a.whole), part = xcd * ((parts + 7) / 8) + local - per;
      if (local - per >= (parts + 7) / 8 || part >= parts) return;
      g = a.whole + part / 4;
      quarter = part % 4;
    } else if (g >= a.whole) {
      return;
    }
    slice = g / (nT * nC);
    g %= nT * nC;
    const int grp = g / (8 * nC), within = g % (8 * nC);
    const int gm = min(8, nT - grp * 8);
    rt = grp * 8 + within % gm;
    cb = within / gm;
  }
  if constexpr (kMode == kDense && TM == 8 && TN == 4) {
    if (quarter >= 0) {
      rt = 2 * rt + (quarter & 1);
      cb = 2 * cb + (quarter >> 1);
      const RowTile<kMode> r(a, nullptr, rt, 64);
      if (r.count > 0 && cb * 8 < ntiles)
        many_item<kX, 4, 2, kMode, kEpi>(a, r, room, cb, slice, lds);
      return;
    }
  }
  const RowTile<kMode> r(a, nullptr, rt, 16 * TM);
  // a list's tile may hold fewer rows: it runs as the smallest tile that holds them
  const int used = (r.count + 15) >> 4;
  if constexpr (kMode == kListed && TM == 4) {
    if (used <= 2) return many_item<kX, 2, TN, kMode, kEpi>(a, r, room, cb, slice, lds);
    if (used == 3) return many_item<kX, 3, TN, kMode, kEpi>(a, r, room, cb, slice, lds);
  }
  if constexpr (kMode == kListed && TM == 8) {
    if (used <= 2) return many_item<kX, 2, TN, kMode, kEpi>(a, r, room, cb, slice, lds);
    if (used <= 4) return many_item<kX, 4, TN, kMode, kEpi>(a, r, room, cb, slice, lds);
    if (used == 5) return many_item<kX, 5, TN, kMode, kEpi>(a, r, room, cb, slice, lds);
    if (used == 6) return many_item<kX, 6, TN, kMode, kEpi>(a, r, room, cb, slice, lds);
    if (used == 7) return many_item<kX, 7, TN, kMode, kEpi>(a, r, room, cb, slice, lds);
  }
  many_item<kX, TM, TN, kMode, kEpi>(a, r, room, cb, slice, lds);
}

// ---------------------------------------------------------------------------
// Down projection and mix of a step of few rows, in one launch: a block per column
// tile holds every entry's 16 outputs, so the weighted sum needs no second pass over
// memory.  Tiles hold eight entries, whose second halves of the hidden values are the
// matrix tile's other eight rows: both products for the price of one.  A wave takes (row
// tile, part of K) units in turn, its next D steps in flight across them; each unit's sums
// have a place of their own in LDS, and a row's places are added in their order: the result
// does not depend on which wave ran when.
// Bound: the weights' stream; eight Granite rows 51 us for both launches (about 250 MB, 4.9
// TB/s), D 3 to 8 within 2%.
// ---------------------------------------------------------------------------
constexpr int kMixWaves = 8;
constexpr int kDppRotate8 = 0x128;   // lane i <- lane (i + 8) % 16 of its sixteen
constexpr int kMixParts = 256;   // (entry, part of K) places, 16 columns each

template <int D>
__global__ __launch_bounds__(kMixWaves * kWave) void k_mx4_down_mix(
    Job a, const float* __restrict__ weights, int rows, float mult, int out_f32, int accumulate) {
  __shared__ Tiles s;
  __shared__ float part[kMixParts][16];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int nl = lane & 15, kq = lane >> 4;
  const int ct = blockIdx.x, ntiles = a.N / 16;
  group_here<8>(a, s);
  const int nT = s.n;
  // with fewer tiles than waves a tile's K goes to several waves, as far as every entry's
  // parts (empty places count) have room
  const int parts = nT >= kMixWaves || nT == 0
                        ? 1
                        : min(min(a.kb, (kMixWaves + nT - 1) / nT), kMixParts / a.M);
  const int ns = (a.kb + parts - 1) / parts;
  const int units = nT * parts;
  const int mine = wave < units ? (units - 1 - wave) / kMixWaves + 1 : 0;
  const int sg = mx4_scale_groups(a.kb);
  const uint8_t* scales = a.w + a.w_tiles * a.kb * 1024;
  u32x4 w[D], x[D][4];
  uint32_t ws[D];
  int64_t tile = 0;
  const uint8_t* xp = a.x;
  int k0 = 0, jn = 0, sn = 0;
  auto decode = [&](int j) {
    const int u = wave + j * kMixWaves, rt = u / parts;
    k0 = u % parts * ns;
    tile = (int64_t)s.expert[rt] * ntiles + ct;
    xp = a.x + (int64_t)s.entry[rt][min(nl & 7, s.count[rt] - 1)] * a.ldx + (nl & 8 ? a.second : 0);
  };
  auto issue = [&](int u) {
    const int b = min(k0 + sn, a.kb - 1);
    w[u] = ld16_stream(a.w + (tile * a.kb + b) * 1024 + lane * 16);
    ws[u] = ld1(scales + (tile * sg + (b >> 2)) * 256 + lane * 4 + (b & 3));
    const int k = b * kMx4K + 32 * kq, kk = k < a.K ? k : 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) x[u][q] = ld16(xp + 2 * kk + 16 * q);
    if (++sn == ns && jn + 1 < mine) {
      sn = 0;
      decode(++jn);
    }
  };
  f32x4 c = {0.f, 0.f, 0.f, 0.f};
  int jc = 0, sc = 0;
  auto compute = [&](int u) {
    const int unit = wave + jc * kMixWaves, rt = unit / parts, p = unit % parts;
    const int b = p * ns + sc;
    if (b < a.kb) {
      if (b == a.kb - 1 && b * kMx4K + 32 * kq >= a.K) {
#pragma unroll
        for (int q = 0; q < 4; ++q) x[u][q] = u32x4{0u, 0u, 0u, 0u};
      }
      const float scale = mx4_scale(ws[u]);
#pragma unroll
      for (int q = 0; q < 4; ++q) c = mfma(fp4x8_to_bf16(w[u][q], scale), x[u][q], c);
    }
    if (++sc < ns) return;
    sc = 0;
    ++jc;
    // an entry's two halves of the hidden values are columns nl and nl + 8
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] += dpp_f<kDppRotate8>(c[i]);
    if (nl < s.count[rt])
      *reinterpret_cast<f32x4*>(&part[s.entry[rt][nl] * parts + p][4 * kq]) = c;
    c = f32x4{0.f, 0.f, 0.f, 0.f};
  };
  if (mine > 0) {
    decode(0);
    const int total = mine * ns;
#pragma unroll
    for (int u = 0; u < D; ++u) issue(u);
    int q0 = 0;
    for (; q0 + D < total; q0 += D) {
#pragma unroll
      for (int u = 0; u < D; ++u) {
        compute(u);
        issue(u);
      }
    }
#pragma unroll
    for (int u = 0; u < D; ++u)
      if (q0 + u < total) compute(u);
  }
  __syncthreads();
  const int r = threadIdx.x / 16, n = threadIdx.x % 16;
  if (r >= rows) return;
  float y = 0.f;
  for (int j = 0; j < a.k; ++j) {
    const int e = r * a.k + j;
    if (s.id[e] < 0) continue;
    float d = part[e * parts][n];
    for (int p = 1; p < parts; ++p) d += part[e * parts + p][n];
    y += weights[(int64_t)r * a.ldi + j] * d;
  }
  y *= mult;
  const int64_t at = (int64_t)r * a.ldo + ct * 16 + n;
  if (out_f32) {
    float* o = (float*)a.out + at;
    *o = accumulate ? *o + y : y;
  } else {
    bf16* o = (bf16*)a.out + at;
    *o = f2bf(accumulate ? bf2f(*o) + y : y);
  }
}

// ---------------------------------------------------------------------------
// Entries of many rows by expert: counts, places and the list of row tiles, by one
// block.  The order of an expert's entries is free (each is computed by itself).
// ---------------------------------------------------------------------------
constexpr int kGroupThreads = 1024;

__global__ __launch_bounds__(kGroupThreads) void k_mx4_group(Job a, int tile_rows, int room,
                                                             int* __restrict__ groups) {
  constexpr int kE = TFD_ROUTE_MAX_EXPERTS, kKeep = 16;
  constexpr int kSizes = 8;              // of a tile, in sixteens
  __shared__ int count[kE], more[kE], wave_rows[kE / kWave], size_s[kSizes];
  __shared__ uint16_t order_s[kKeep * kGroupThreads];
  const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
  if (tid < kE) count[tid] = more[tid] = 0;
  if (tid < kSizes) size_s[tid] = 0;
  auto at = [&](int i) {
    return a.ids[a.ldi == a.k ? i : (int64_t)(i / a.k) * a.ldi + i % a.k];
  };
  auto valid = [&](int id) {
    if ((unsigned)id < (unsigned)a.E) return id;
    if (id != -1 && a.err) raise_error(a.err, kErrTokenRange);
    return -1;
  };
  // a thread's first ids, and their places among their expert's, stay in registers for the
  // second pass (all loads before a use); the others are counted apart, behind them
  int kept[kKeep], rank[kKeep];
#pragma unroll
  for (int j = 0; j < kKeep; ++j) kept[j] = at(min(tid + j * kGroupThreads, a.M - 1));
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    kept[j] = tid + j * kGroupThreads < a.M ? valid(kept[j]) : -1;
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    if (kept[j] >= 0) rank[j] = atomicAdd(&count[kept[j]], 1);
  for (int i = tid + kKeep * kGroupThreads; i < a.M; i += kGroupThreads) {
    const int id = valid(at(i));
    if (id >= 0) atomicAdd(&more[id], 1);
  }
  __syncthreads();
  // an expert's rows spread evenly over its tiles, in sixteens: a tile costs by those.  The
  // list has the largest tiles first: the last to start are then the shortest.
  const int mine = tid < a.E ? count[tid] + more[tid] : 0;
  const int tiles = (mine + tile_rows - 1) / tile_rows;
  const int even = tiles ? ((mine + tiles - 1) / tiles + 15) / 16 : 0;
  if (tiles) atomicAdd(&size_s[kSizes - even], tiles);
  int rows_to = mine;
#pragma unroll
  for (int d = 1; d < kWave; d *= 2) {
    const int r = __shfl_up(rows_to, d, kWave);
    rows_to += lane >= d ? r : 0;
  }
  if (tid < kE && lane == kWave - 1) wave_rows[wave] = rows_to;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kE / kWave; ++v)
    if (v < wave) rows_to += wave_rows[v];
  if (tid == 0) {
    int all = 0;
#pragma unroll
    for (int v = 0; v < kSizes; ++v) {
      const int n = size_s[v];
      size_s[v] = all;
      all += n;
    }
    groups[0] = all;
    groups[1] = room;
  }
  __syncthreads();
  if (tiles) {
    const int f = rows_to - mine, t0 = atomicAdd(&size_s[kSizes - even], tiles);
    for (int t = 0; t < tiles; ++t) {
      int* o = groups + 4 + (t0 + t) * 4;
      o[0] = tid;
      o[1] = f + t * even * 16;
      o[2] = min(even * 16, mine - t * even * 16);
    }
    more[tid] = f + count[tid];
    count[tid] = f;
  }
  if (tid == kE - 1) wave_rows[0] = rows_to;
  __syncthreads();
  int* order = groups + 4 + room * 4;
  // by way of LDS where all are kept: a store to 64 lines takes as many cycles
  if (a.M <= kKeep * kGroupThreads) {
    const int entries = wave_rows[0];
#pragma unroll
    for (int j = 0; j < kKeep; ++j)
      if (kept[j] >= 0) order_s[count[kept[j]] + rank[j]] = (uint16_t)(tid + j * kGroupThreads);
    __syncthreads();
    for (int i = tid; i < entries; i += kGroupThreads) order[i] = order_s[i];
    return;
  }
#pragma unroll
  for (int j = 0; j < kKeep; ++j)
    if (kept[j] >= 0) order[count[kept[j]] + rank[j]] = tid + j * kGroupThreads;
  for (int i = tid + kKeep * kGroupThreads; i < a.M; i += kGroupThreads) {
    const int id = at(i);
    if ((unsigned)id < (unsigned)a.E) order[atomicAdd(&more[id], 1)] = i;
  }
}

// The weighted sum of a row's places, in their order; four columns a thread.
__global__ __launch_bounds__(kBlock) void k_mx4_mix(const float* __restrict__ d,
                                                    const int32_t* __restrict__ ids,
                                                    const float* __restrict__ weights, int ldi,
                                                    int k, int E, int H, float mult, int out_f32,
                                                    int accumulate, void* __restrict__ out,
                                                    int64_t ldo) {
  const int r = blockIdx.y, n = (blockIdx.x * kBlock + threadIdx.x) * 4;
  if (n >= H) return;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < k; ++j) {
    const int id = ids[(int64_t)r * ldi + j];
    if ((unsigned)id >= (unsigned)E) continue;
    y += weights[(int64_t)r * ldi + j] *
         *reinterpret_cast<const f32x4*>(d + ((int64_t)r * k + j) * H + n);
  }
  y *= mult;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t at = (int64_t)r * ldo + n + i;
    if (out_f32) {
      float* o = (float*)out + at;
      *o = accumulate ? *o + y[i] : y[i];
    } else {
      bf16* o = (bf16*)out + at;
      *o = f2bf(accumulate ? bf2f(*o) + y[i] : y[i]);
    }
  }
}

// How a call runs, and what of `work` it uses.
struct Plan {
  bool fused;                    // grouped in the blocks, the mix in the down launch, hidden
                                 // values as two bf16
  int tile_rows, room;
  int64_t second, d, groups, bytes;
};
Plan experts_plan(int rows, int k, int E, int H, int I) {
  const int64_t n = (int64_t)rows * k;
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  Plan p = {};
  p.fused = rows <= kHereRows && n <= kHereMax;
  // By the rows an expert has if all are picked alike (us, weights from memory): items of 16
  // rows by the stream's kernel for few, the longer gate/up's K the more (fitted to I < H;
  // down's K, which is I, does not enter) (64 Granite rows, 9 an expert:
  // 95; tiles of 64 103; 128 rows 134 and 110; 64 Qwen3.5 rows, 2 an expert, 69 and 72; 250
  // rows, 8, 109 and 105); tiles of up to 64 (512 Granite rows 167; tiles of 128 184); of up
  // to 128 past as many (1,024 Granite rows 272; 64 286).
  const int64_t mean = n / E;
  p.tile_rows = mean * 400 <= H ? 16 : mean <= 128 ? 64 : 128;
  p.room = (int)(E + n / p.tile_rows);
  p.second = up(n * I * 2);
  p.d = p.second * (p.fused ? 2 : 1);
  p.groups = p.d + (p.fused ? 0 : up(n * H * 4));
  p.bytes = p.groups + (p.fused ? 0 : up((4 + 4 * (int64_t)p.room + n) * 4));
  return p;
}
// Bytes for `rows` and for every smaller call, which may run in another way and need more:
// the most rows that run fused hold two hidden parts, and tiles of 16 the longest list.
int64_t experts_work(int rows, int k, int E, int H, int I) {
  const int64_t fused = experts_plan(min(min(rows, kHereRows), kHereMax / k), k, E, H, I).bytes;
  const Plan p = experts_plan(rows, k, E, H, I);
  if (p.fused) return fused;
  const int64_t n = (int64_t)rows * k, list = (4 + 4 * (E + n / 16) + n) * 4;
  const int64_t listed = p.groups + (list + 255) / 256 * 256;
  return fused > listed ? fused : listed;          // (the host's max takes ints)
}

template <int TM, int TN>
void launch_listed(const Job& gu, const Job& down, int tiles, hipStream_t s) {
  auto grid = [&](const Job& j) {
    const int64_t nC = ((j.N + 15) / 16 + 4 * TN - 1) / (4 * TN);
    return (int)((tiles + 7) / 8 * 8 * nC);
  };
  k_mx4_many<kXBf16, TM, TN, kListed, kSwiglu><<<grid(gu), kBlock, 0, s>>>(gu, tiles);
  k_mx4_many<kXBf16, TM, TN, kListed, kF32><<<grid(down), kBlock, 0, s>>>(down, tiles);
}

int job_checks(const char* what, int K, int64_t N) {
  if (K <= 0 || K % 32 || K > (1 << 22) || N <= 0 || N > (1 << 24))
    return fail(kBadShape, "%s: K=%d N=%lld (K a multiple of 32)", what, K, (long long)N);
  return 0;
}

// The parts of K of a product, added in their order; four columns a thread.
__global__ __launch_bounds__(kBlock) void k_mx4_sum(const float* __restrict__ part, int slices,
                                                    int64_t slice, int N, int ldp, void* out,
                                                    int64_t ldo, int out_f32, int vec) {
  const int n = (blockIdx.x * kBlock + threadIdx.x) * 4;
  if (n >= N) return;
  const float* p = part + (int64_t)blockIdx.y * ldp + n;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < slices; ++s) y += *reinterpret_cast<const f32x4*>(p + s * slice);
  Job a = {};
  a.out = out;
  a.ldo = ldo;
  a.N = N;
  a.vec = vec;
  if (out_f32) put<kF32>(a, blockIdx.y, n, y);
  else put<kBf16>(a, blockIdx.y, n, y);
}

// How a dense product runs.
//   rows <= 16     items of a column tile; where a compute unit has one at most, by eight waves
//                  (1 x 6144 x 2048 6.4 us by four, 5.6; 16 rows 9.4, 9.0; from a K of 2,048 on:
//                  1 x 1024 x 2048 3.0, 3.1)
//   17 .. 64       items of 32 rows by four column tiles, which share the rows' loads, where
//                  they occupy half the compute units (17 x 4096 x 8512: 11 us; one tile an
//                  item 18); else 16 rows by a column tile, as above, where a compute unit has
//                  one at most (32 x 6144 x 2048: 9.3 us; 32 rows an item 13.8, four column
//                  tiles in 12 parts of K and a second launch 11.6); else 32 rows by a column
//                  tile (40 x 6144 x 2048: 14.3 us; 16 rows 15.8)
//   more           blocks of 128 x 256, or of 64 x 128 where the large ones leave compute
//                  units idle, and parts of K where that is estimated to pay: a block of 64 x
//                  128 takes about 0.8 us for 128 k of bf16 and 0.36 of 4 bits; adding parts
//                  takes 3.5 us and their f32 rows' way to memory and back at 5 TB/s (65 x
//                  6144 x 2048: 31 us whole, 15 in 12 parts; 1,000 rows 50 and 35; 65 x 2048 x
//                  12288 13 and 16, not taken).  Of blocks of 128 x 256 a few that would run
//                  behind all others run as quarters, on four times the compute units: up to
//                  2 / 5 of those behind whole pairs, 1 / 5 behind single blocks, whose second
//                  place was free (4,001 x 4096 x 8512, 64 behind 1,024: 218 us, 197 in
//                  quarters, codes 100 and 92; 1,024 rows, 16 behind 256: 86 and 60; 84 behind
//                  256: 91 in quarters, not taken).  Else blocks of 128 x 192, which read 15%
//                  more for a product, where 256 columns leave compute units with one block
//                  behind the last pair, or a second one (1,280 x 4096 x 8512: 76 us)
struct DensePlan {
  int rows, cols, slices;        // of an item; parts of K
  int64_t items;
  int rest;                      // the last items, which run in quarters
};
DensePlan dense_plan(bool mx, int M, int K, int N) {
  const int cus = compute_units(), kb = mx4_blocks(K), quads = mx4_scale_groups(kb);
  DensePlan p = {16, 16, 1, (N + 15) / 16, 0};
  auto shape = [&](int rows, int cols) {
    p.rows = rows;
    p.cols = cols;
    p.items = (int64_t)((M + rows - 1) / rows) * ((N + cols - 1) / cols);
  };
  if (M <= 16) return p;
  if (M <= TFD_MX4_WHOLE_ROWS) {
    shape(32, 64);
    if (p.items < cus / 2) shape(32, 16);
    if (p.cols == 16 && K >= 2048 && (M + 15) / 16 * ((N + 15) / 16) <= cus) shape(16, 16);
    return p;
  }
  shape(128, 192);
  const int64_t narrow = p.items;
  shape(128, 256);
  if (p.items >= cus) {
    // the fullest compute unit's blocks, two at a time; one alone takes 0.6 of a pair's time
    auto rounds = [&](int64_t items) {
      const int64_t n = (items + cus - 1) / cus;
      return n / 2 + (n % 2) * 0.6;
    };
    const int rest = p.items % cus;
    const bool pairs = p.items / cus % 2 == 0;
    if (rest * 5 <= cus * (pairs ? 2 : 1)) p.rest = rest;
    else if (rounds(narrow) * 3 * 1.15 < 0.9 * rounds(p.items) * 4) shape(128, 192);
    return p;
  }
  shape(64, 128);
  const double whole = (mx ? 0.36 : 0.8) * kb;
  double best = 0.8 * whole;     // the estimate has to save a fifth
  // at most two blocks a compute unit, and four of 128 k a part
  for (int s = 2; s <= quads && s * p.items <= 2 * cus; ++s) {
    const double us = whole / s + 3.5 + s * (double)M * N * 8 / 5e6;
    if (us < best) {
      best = us;
      p.slices = s;
    }
  }
  return p;
}

template <int kX, int kEpi>
int launch_dense(Job a, const DensePlan& p, hipStream_t s) {
  const int cus = compute_units();
  const int64_t items = p.items * a.slices;
  if (items > (1 << 23)) return fail(kBadShape, "mx4_gemm: M=%d N=%d", a.M, a.N);
  const int few = (int)min(items, (int64_t)4 * cus), rest = (int)p.rest;
  a.whole = (int)items - rest;
  const int many = 8 * ((a.whole + 7) / 8 + (4 * rest + 7) / 8);
  const int nT = (a.M + p.rows - 1) / p.rows;
  if (p.rows == 16 && items <= cus && a.K >= 2048)
    k_mx4_few<kX, 1, 1, 2, kDense, kEpi, 8><<<few, 8 * kWave, 0, s>>>(a);
  else if (p.rows == 16)
    k_mx4_few<kX, 1, 1, 4, kDense, kEpi><<<few, kBlock, 0, s>>>(a);
  else if (p.rows == 32 && p.cols == 64)
    k_mx4_few<kX, 2, 4, 2, kDense, kEpi><<<few, kBlock, 0, s>>>(a);
  else if (p.rows == 32)
    k_mx4_few<kX, 2, 1, 2, kDense, kEpi><<<few, kBlock, 0, s>>>(a);
  else if (p.rows == 64)
    k_mx4_many<kX, 4, 2, kDense, kEpi><<<many, kBlock, 0, s>>>(a, nT);
  else if (p.cols == 192)
    k_mx4_many<kX, 8, 3, kDense, kEpi><<<many, kBlock, 0, s>>>(a, nT);
  else
    k_mx4_many<kX, 8, 4, kDense, kEpi><<<many, kBlock, 0, s>>>(a, nT);
  return launched("mx4_gemm");
}

}  // namespace

extern "C" int64_t tfd_mx4_gemm_work_bytes(int M, int K, int N) {
  if (M <= 0 || K <= 0 || K % 32 || N <= 0) return 0;
  const int s = max(dense_plan(false, M, K, N).slices, dense_plan(true, M, K, N).slices);
  return s > 1 ? (int64_t)s * M * ((N + 3) / 4 * 4) * 4 : 0;
}

extern "C" int tfd_mx4_gemm_form(int x_mx4, int M, int K, int N, int32_t form[4]) {
  if (!form) return fail(kBadArg, "mx4_gemm_form: null form");
  if (const int rc = job_checks("mx4_gemm_form", K, N)) return rc;
  if (M <= 0) return fail(kBadShape, "mx4_gemm_form: M=%d", M);
  const DensePlan p = dense_plan(x_mx4 != 0, M, K, N);
  form[0] = p.rows, form[1] = p.cols, form[2] = p.slices, form[3] = p.rest;
  return 0;
}

extern "C" int tfd_mx4_gemm(const TfdMx4GemmArgs* args, void* stream) {
  if (!args) return fail(kBadArg, "mx4_gemm: null args");
  const TfdMx4GemmArgs& a = *args;
  if (a.out_type != TFD_TYPE_F32 && a.out_type != TFD_TYPE_BF16)
    return fail(kBadArg, "mx4_gemm: out_type %d", a.out_type);
  if (const int rc = job_checks("mx4_gemm", a.K, a.N)) return rc;
  if (a.M < 0 || a.M > (1 << 30) || a.ldx > (1 << 23) || a.ldxs > (1 << 23))
    return fail(kBadShape, "mx4_gemm: M=%d ldx=%lld ldxs=%lld", a.M, (long long)a.ldx,
                (long long)a.ldxs);
  if (a.M == 0) return 0;
  if (!a.x || !a.w || !a.out) return fail(kBadArg, "mx4_gemm: null pointer");
  const bool mx = a.x_scales != nullptr;
  const int64_t row = mx ? a.K / 2 : 2 * (int64_t)a.K, ld = mx ? a.ldx : 2 * a.ldx;
  if ((uintptr_t)a.x % 16 || (uintptr_t)a.w % 16 || (a.M > 1 && (ld % 16 || ld < row)) ||
      (mx && a.M > 1 && a.ldxs < a.K / 32) || a.ldo < a.N ||
      (uintptr_t)a.out % (a.out_type == TFD_TYPE_F32 ? 4 : 2))
    return fail(kBadArg, "mx4_gemm: ldx=%lld ldxs=%lld ldo=%lld or an alignment",
                (long long)a.ldx, (long long)a.ldxs, (long long)a.ldo);
  Job j = {};
  j.x = (const uint8_t*)a.x;
  j.ldx = ld;
  j.xs = (const uint8_t*)a.x_scales;
  j.ldxs = a.ldxs;
  j.w = (const uint8_t*)a.w;
  j.w_tiles = (a.N + 15) / 16;
  j.K = a.K;
  j.kb = mx4_blocks(a.K);
  j.N = a.N;
  j.M = a.M;
  j.out = a.out;
  j.ldo = a.ldo;
  const int size = a.out_type == TFD_TYPE_F32 ? 4 : 2;
  j.vec = a.ldo % 4 == 0 && (uintptr_t)a.out % (4 * size) == 0;
  hipStream_t s = (hipStream_t)stream;
  const DensePlan p = dense_plan(mx, a.M, a.K, a.N);
  const int ldp = (a.N + 3) / 4 * 4;
  const bool f32 = a.out_type == TFD_TYPE_F32;
  const bool parts = p.slices > 1 && a.work && (uintptr_t)a.work % 16 == 0 &&
                     a.work_bytes >= (int64_t)p.slices * a.M * ldp * 4;
  j.slices = parts ? p.slices : 1;
  if (!parts) {
    if (mx) return f32 ? launch_dense<kXMx4, kF32>(j, p, s) : launch_dense<kXMx4, kBf16>(j, p, s);
    return f32 ? launch_dense<kXBf16, kF32>(j, p, s) : launch_dense<kXBf16, kBf16>(j, p, s);
  }
  const int vec = j.vec;
  j.out = a.work;
  j.ldo = ldp;
  j.slice = (int64_t)a.M * ldp;
  j.vec = 1;
  const int rc = mx ? launch_dense<kXMx4, kF32>(j, p, s) : launch_dense<kXBf16, kF32>(j, p, s);
  if (rc) return rc;
  k_mx4_sum<<<dim3((ldp / 4 + kBlock - 1) / kBlock, a.M), kBlock, 0, s>>>(
      (const float*)a.work, j.slices, j.slice, a.N, ldp, a.out, a.ldo, f32, vec);
  return launched("mx4_gemm");
}

extern "C" {

int64_t tfd_mx4_experts_work_bytes(int rows, int k, int experts, int H, int I) {
  if (rows <= 0 || k <= 0 || experts <= 0 || H <= 0 || I <= 0) return 0;
  return experts_work(rows, k, experts, H, I);
}

int tfd_mx4_experts_tile_rows(int rows, int k, int experts, int H, int I) {
  if (rows <= 0 || rows > 65535 || k < 1 || k > 64 || experts < 1 ||
      experts > TFD_ROUTE_MAX_EXPERTS || H <= 0 || I <= 0)
    return -1;
  const Plan p = experts_plan(rows, k, experts, H, I);
  return p.fused ? 0 : p.tile_rows;
}

int tfd_mx4_experts(const TfdMx4ExpertsArgs* args, void* stream) {
  if (!args) return fail(kBadArg, "mx4_experts: null args");
  const TfdMx4ExpertsArgs& a = *args;
  if (a.out_type != TFD_TYPE_F32 && a.out_type != TFD_TYPE_BF16)
    return fail(kBadArg, "mx4_experts: out_type %d", a.out_type);
  if (a.H <= 0 || a.I <= 0 || a.H % 32 || a.I % 32 || a.H > (1 << 20) || a.I > (1 << 20))
    return fail(kBadShape, "mx4_experts: H=%d I=%d (multiples of 32)", a.H, a.I);
  if (a.experts < 1 || a.experts > TFD_ROUTE_MAX_EXPERTS || a.k < 1 || a.k > 64 || a.rows < 0 ||
      a.rows > 65535)
    return fail(kBadShape, "mx4_experts: rows=%d k=%d experts=%d", a.rows, a.k, a.experts);
  if (a.rows == 0) return 0;
  if (!a.x || !a.ids || !a.weights || !a.w_gu || !a.w_down || !a.out || !a.work)
    return fail(kBadArg, "mx4_experts: null pointer");
  // rows are read at 31-bit offsets from their first
  if (((int64_t)a.rows * (a.rows > 1 ? a.ldx : a.H)) >> 30 ||
      ((int64_t)a.rows * a.k * a.I) >> 30)
    return fail(kBadShape, "mx4_experts: rows=%d of %lld, or %d x %d hidden values, pass 2 GiB",
                a.rows, (long long)a.ldx, a.rows * a.k, a.I);
  if ((uintptr_t)a.x % 16 || (uintptr_t)a.w_gu % 16 || (uintptr_t)a.w_down % 16 ||
      (uintptr_t)a.work % 256 || (uintptr_t)a.ids % 4 || (uintptr_t)a.weights % 4 ||
      (a.rows > 1 && (a.ldx % 8 || a.ldx < a.H)) || a.ld < a.k || a.ldo < a.H ||
      (uintptr_t)a.out % (a.out_type == TFD_TYPE_F32 ? 4 : 2))
    return fail(kBadArg, "mx4_experts: ldx=%lld ld=%d ldo=%lld or an alignment",
                (long long)a.ldx, a.ld, (long long)a.ldo);
  const Plan plan = experts_plan(a.rows, a.k, a.experts, a.H, a.I);
  if (a.work_bytes < plan.bytes)
    return fail(kBadArg, "mx4_experts: work of %lld bytes, %lld needed", (long long)a.work_bytes,
                (long long)plan.bytes);
  uint8_t* work = (uint8_t*)a.work;
  const int n = a.rows * a.k;
  Job gu = {};
  gu.x = (const uint8_t*)a.x;
  gu.ldx = 2 * a.ldx;
  gu.w = (const uint8_t*)a.w_gu;
  gu.w_tiles = (int64_t)a.experts * (a.I / 8);
  gu.K = a.H;
  gu.kb = mx4_blocks(a.H);
  gu.N = 2 * a.I;
  gu.M = n;
  gu.out = work;
  gu.ldo = a.I;
  gu.vec = 1;
  gu.second = plan.second;
  gu.ids = a.ids;
  gu.ldi = a.ld;
  gu.k = gu.div = a.k;
  gu.E = a.experts;
  gu.err = a.err;
  Job down = gu;
  down.x = work;
  down.ldx = 2 * (int64_t)a.I;
  down.w = (const uint8_t*)a.w_down;
  down.w_tiles = (int64_t)a.experts * (a.H / 16);
  down.K = a.I;
  down.kb = mx4_blocks(a.I);
  down.N = a.H;
  down.div = 1;
  down.err = nullptr;              // the first launch has raised it
  hipStream_t s = (hipStream_t)stream;
  const int cus = compute_units();
  const int out_f32 = a.out_type == TFD_TYPE_F32;
  if (plan.fused) {
    down.out = a.out;
    down.ldo = a.ldo;
    // column tiles of an item, which share its rows' loads: four where the items still go
    // round (eight Granite rows: gate/up and down 48 us; one tile an item 58), else one (a
    // Qwen3.5 row: 11.5 us; four 12.2)
    const int wide = n * ((a.I / 8 + 3) / 4);
    if (wide >= 4 * cus)
      k_mx4_few<kXBf16, 1, 4, 2, kHere, kSwigluTwo><<<4 * cus, kBlock, 0, s>>>(gu);
    else
      k_mx4_few<kXBf16, 1, 1, 4, kHere, kSwigluTwo><<<min(n * (a.I / 8), 4 * cus), kBlock, 0, s>>>(gu);
    k_mx4_down_mix<4><<<a.H / 16, kMixWaves * kWave, 0, s>>>(down, a.weights, a.rows, a.mult,
                                                            out_f32, a.accumulate);
    return launched("mx4_experts");
  }
  down.out = work + plan.d;
  down.ldo = a.H;
  int* groups = (int*)(work + plan.groups);
  gu.groups = down.groups = groups;
  const int tile_rows = plan.tile_rows, tiles = a.experts + n / tile_rows;
  k_mx4_group<<<1, kGroupThreads, 0, s>>>(gu, tile_rows, plan.room, groups);
  if (tile_rows == 16) {
    k_mx4_few<kXBf16, 1, 4, 2, kListed, kSwiglu, 4, false><<<3 * cus, kBlock, 0, s>>>(gu);
    k_mx4_few<kXBf16, 1, 4, 2, kListed, kF32, 4, false><<<3 * cus, kBlock, 0, s>>>(down);
  } else if (tile_rows == 64) {
    launch_listed<4, 4>(gu, down, tiles, s);
  } else {
    launch_listed<8, 4>(gu, down, tiles, s);
  }
  k_mx4_mix<<<dim3((a.H / 4 + kBlock - 1) / kBlock, a.rows), kBlock, 0, s>>>(
      (const float*)(work + plan.d), a.ids, a.weights, a.ld, a.k, a.experts, a.H, a.mult, out_f32,
      a.accumulate, a.out, a.ldo);
  return launched("mx4_experts");
}

}  // extern "C"
