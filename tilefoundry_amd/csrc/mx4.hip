// Microscaled 4-bit tensors: quantisation, its inverse, and the layout that the
// products read.
#include "host_common.h"
#include "mx4.h"
#include "tf_mx4.h"

using namespace tfd;
using namespace tfd_host;

namespace {

// ---------------------------------------------------------------------------
// Quantisation.  Four lanes hold a block of 32, eight values each.  The shared
// exponent comes from the largest magnitude's own exponent bits; the codes from
// gfx950's scaled conversion, which divides by a power of two, rounds to the
// nearest even code and saturates at 6 -- the definition, in one instruction for
// two values (checked against it over grids of ties).
// Bound: memory; a thread reads 32 or 16 bytes and writes four.  12,288 x 2048 f32 17 us
// (6.7 TB/s, partly from the last-level cache), back to bf16 11.4 us (5.5 TB/s).
// ---------------------------------------------------------------------------
constexpr int kPerLane = 8;

template <int kType>
__device__ __forceinline__ float widen(uint32_t bits) {
  if (kType == TFD_TYPE_BF16) return __uint_as_float(bits << 16);
  return (float)__builtin_bit_cast(_Float16, (uint16_t)bits);
}

template <int kType, bool kVec>
__global__ __launch_bounds__(kBlock) void k_quantise(const void* __restrict__ x, int64_t ldx,
                                                     int64_t pieces, int per_row,
                                                     uint8_t* __restrict__ codes, int64_t ldc,
                                                     uint8_t* __restrict__ scales, int64_t lds) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  // a block's four lanes are in or out together: pieces is a multiple of four
  if (i >= pieces) return;
  const int64_t row = i / per_row;
  const int at = (int)(i - row * per_row);
  float v[kPerLane];
  if (kType == TFD_TYPE_F32) {
    const float* p = (const float*)x + row * ldx + at * kPerLane;
    if (kVec) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[j] = a[j];
        v[4 + j] = b[j];
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) v[j] = p[j];
    }
  } else {
    const uint16_t* p = (const uint16_t*)x + row * ldx + at * kPerLane;
    if (kVec) {
      const u32x4 a = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = widen<kType>(a[j] & 0xffffu);
        v[2 * j + 1] = widen<kType>(a[j] >> 16);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) v[j] = widen<kType>(p[j]);
    }
  }
  // magnitudes' bit patterns order as the values do, infinities and NaN last
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < kPerLane; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, kDppXor1, 0xF, 0xF, false));
  top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, kDppXor2, 0xF, 0xF, false));
  const bool finite = top < 0x7f800000u;
  // the exponent byte less two; values under 2^-125 share the smallest scale
  const int s = max((int)(top >> 23) - 2, 0);
  const float scale = __uint_as_float((uint32_t)s << 23);
  uint32_t q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
  *reinterpret_cast<uint32_t*>(codes + row * ldc + at * (kPerLane / 2)) = finite ? q : 0u;
  if ((at & 3) == 0) scales[row * lds + (at >> 2)] = (uint8_t)(finite ? s : 255);
}

// Eight codes and their scale to values.
template <int kType>
__global__ __launch_bounds__(kBlock) void k_dequantise(const uint8_t* __restrict__ codes,
                                                       int64_t ldc,
                                                       const uint8_t* __restrict__ scales,
                                                       int64_t lds, int64_t pieces, int per_row,
                                                       void* __restrict__ out, int64_t ldo) {
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= pieces) return;
  const int64_t row = i / per_row;
  const int at = (int)(i - row * per_row);
  const uint32_t q = *reinterpret_cast<const uint32_t*>(codes + row * ldc + at * 4);
  const float scale = __uint_as_float((uint32_t)scales[row * lds + (at >> 2)] << 23);
  const int64_t to = row * ldo + at * kPerLane;
  if (kType == TFD_TYPE_F32) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    float* o = (float*)out + to;
    const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0);
    const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1);
    const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 2);
    const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 3);
    o[0] = a.x, o[1] = a.y, o[2] = b.x, o[3] = b.y;
    o[4] = c.x, o[5] = c.y, o[6] = d.x, o[7] = d.y;
  } else if (kType == TFD_TYPE_BF16) {
    const u32x4 v = fp4x8_to_bf16(q, scale);
    uint32_t* o = (uint32_t*)((bf16*)out + to);
    o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
  } else {
    // f16's range is narrower than a scale's: by way of f32, rounded once
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    _Float16* o = (_Float16*)out + to;
    const f32x2_t a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 0);
    const f32x2_t b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 1);
    const f32x2_t c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 2);
    const f32x2_t d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q, scale, 3);
    o[0] = (_Float16)a.x, o[1] = (_Float16)a.y, o[2] = (_Float16)b.x, o[3] = (_Float16)b.y;
    o[4] = (_Float16)c.x, o[5] = (_Float16)c.y, o[6] = (_Float16)d.x, o[7] = (_Float16)d.y;
  }
}

// A lane's 16 bytes of one block, and its scale byte.
__global__ __launch_bounds__(kBlock) void k_pack(const uint8_t* __restrict__ codes,
                                                 const uint8_t* __restrict__ scales,
                                                 const uint8_t* __restrict__ codes2,
                                                 const uint8_t* __restrict__ scales2, int64_t rows,
                                                 int K, uint8_t* __restrict__ packed) {
  const int kb = mx4_blocks(K);
  const int64_t tiles = (rows + 15) / 16;
  const int groups = mx4_scale_groups(kb);
  const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
  if (i >= tiles * groups * 4 * kWave) return;      // padded blocks too: their scales
  const int lane = (int)(i & (kWave - 1));
  const int64_t block = i / kWave;
  const int b = (int)(block % (groups * 4));
  const int64_t tile = block / (groups * 4);
  const int64_t row = tile * 16 + (lane & 15);
  const int k = b * kMx4K + 32 * (lane >> 4);
  u32x4 q = {0u, 0u, 0u, 0u};
  uint8_t s = 127;
  if (row < rows && k < K) {
    const bool second = codes2 && (row & 1);
    const int64_t r = codes2 ? row >> 1 : row;
    q = *reinterpret_cast<const u32x4*>((second ? codes2 : codes) + r * (K / 2) + k / 2);
    s = (second ? scales2 : scales)[r * (K / 32) + k / 32];
  }
  if (b < kb) *reinterpret_cast<u32x4*>(packed + (tile * kb + b) * 1024 + lane * 16) = q;
  packed[tiles * kb * 1024 + (tile * groups + (b >> 2)) * 256 + lane * 4 + (b & 3)] = s;
}

// Threads of one launch: their number, rounded up to blocks, has 32 bits.
constexpr int64_t kMaxThreads = ((int64_t)1 << 32) - kBlock;

int blocks_for(int64_t threads) { return (int)((threads + kBlock - 1) / kBlock); }

}  // namespace

extern "C" {

int tfd_mx4_quantise(const void* x, int64_t ldx, int type, int64_t rows, int K, void* codes,
                     int64_t ldc, void* scales, int64_t lds, void* stream) {
  if (type != TFD_TYPE_F32 && type != TFD_TYPE_BF16 && type != TFD_TYPE_F16)
    return fail(kBadArg, "mx4_quantise: type %d", type);
  if (rows < 0 || K <= 0 || K % 32)
    return fail(kBadShape, "mx4_quantise: rows=%lld K=%d (K a multiple of 32)", (long long)rows, K);
  if (rows == 0) return 0;
  if (!x || !codes || !scales) return fail(kBadArg, "mx4_quantise: null pointer");
  const int size = type == TFD_TYPE_F32 ? 4 : 2;
  if ((rows > 1 && (ldx < K || ldc < K / 2 || lds < K / 32)) || ldc % 4 ||
      (uintptr_t)codes % 4 || (uintptr_t)x % size)
    return fail(kBadArg, "mx4_quantise: ldx=%lld ldc=%lld lds=%lld or an alignment", (long long)ldx,
                (long long)ldc, (long long)lds);
  const int per_row = K / kPerLane;
  if (rows > kMaxThreads / per_row)
    return fail(kBadShape, "mx4_quantise: %lld rows of %d pass 2^35 values", (long long)rows, K);
  const int64_t pieces = rows * per_row;
  const bool vec = (uintptr_t)x % 16 == 0 && (rows == 1 || ldx * size % 16 == 0);
  const dim3 grid(blocks_for(pieces));
  hipStream_t s = (hipStream_t)stream;
#define TFD_QUANT(T, V) \
  k_quantise<T, V><<<grid, kBlock, 0, s>>>(x, ldx, pieces, per_row, (uint8_t*)codes, ldc, \
                                           (uint8_t*)scales, lds)
  if (type == TFD_TYPE_F32) {
    if (vec) TFD_QUANT(TFD_TYPE_F32, true); else TFD_QUANT(TFD_TYPE_F32, false);
  } else if (type == TFD_TYPE_BF16) {
    if (vec) TFD_QUANT(TFD_TYPE_BF16, true); else TFD_QUANT(TFD_TYPE_BF16, false);
  } else {
    if (vec) TFD_QUANT(TFD_TYPE_F16, true); else TFD_QUANT(TFD_TYPE_F16, false);
  }
#undef TFD_QUANT
  return launched("mx4_quantise");
}

int tfd_mx4_dequantise(const void* codes, int64_t ldc, const void* scales, int64_t lds,
                       int64_t rows, int K, void* out, int64_t ldo, int type, void* stream) {
  if (type != TFD_TYPE_F32 && type != TFD_TYPE_BF16 && type != TFD_TYPE_F16)
    return fail(kBadArg, "mx4_dequantise: type %d", type);
  if (rows < 0 || K <= 0 || K % 32)
    return fail(kBadShape, "mx4_dequantise: rows=%lld K=%d (K a multiple of 32)", (long long)rows,
                K);
  if (rows == 0) return 0;
  if (!codes || !scales || !out) return fail(kBadArg, "mx4_dequantise: null pointer");
  if ((rows > 1 && (ldo < K || ldc < K / 2 || lds < K / 32)) || ldc % 4 || ldo % 2 ||
      (uintptr_t)codes % 4 || (uintptr_t)out % 4)
    return fail(kBadArg, "mx4_dequantise: ldc=%lld lds=%lld ldo=%lld or an alignment",
                (long long)ldc, (long long)lds, (long long)ldo);
  const int per_row = K / kPerLane;
  if (rows > kMaxThreads / per_row)
    return fail(kBadShape, "mx4_dequantise: %lld rows of %d pass 2^35 values", (long long)rows,
                K);
  const int64_t pieces = rows * per_row;
  const dim3 grid(blocks_for(pieces));
  hipStream_t s = (hipStream_t)stream;
#define TFD_DEQUANT(T) \
  k_dequantise<T><<<grid, kBlock, 0, s>>>((const uint8_t*)codes, ldc, (const uint8_t*)scales, lds, \
                                          pieces, per_row, out, ldo)
  if (type == TFD_TYPE_F32) TFD_DEQUANT(TFD_TYPE_F32);
  else if (type == TFD_TYPE_BF16) TFD_DEQUANT(TFD_TYPE_BF16);
  else TFD_DEQUANT(TFD_TYPE_F16);
#undef TFD_DEQUANT
  return launched("mx4_dequantise");
}

int64_t tfd_mx4_packed_bytes(int64_t N, int K) {
  if (N <= 0 || K <= 0 || K % 32) return 0;
  const int kb = mx4_blocks(K);
  return (N + 15) / 16 * ((int64_t)kb * 1024 + mx4_scale_groups(kb) * 256);
}

int tfd_mx4_pack(const void* codes, const void* scales, const void* codes2, const void* scales2,
                 int64_t N, int K, void* packed, void* stream) {
  if (!codes || !scales || !packed || !codes2 != !scales2)
    return fail(kBadArg, "mx4_pack: null pointer");
  if (N <= 0 || K <= 0 || K % 32)
    return fail(kBadShape, "mx4_pack: N=%lld K=%d (K a multiple of 32)", (long long)N, K);
  if ((uintptr_t)codes % 16 || (uintptr_t)codes2 % 16 || (uintptr_t)packed % 16)
    return fail(kBadArg, "mx4_pack: codes or packed not 16-byte aligned");
  const int64_t per_tile = (int64_t)mx4_scale_groups(mx4_blocks(K)) * 4 * kWave;
  const int64_t rows = N > kMaxThreads ? N : codes2 ? 2 * N : N;
  if (rows / 16 + 1 > kMaxThreads / per_tile)
    return fail(kBadShape, "mx4_pack: N=%lld K=%d", (long long)N, K);
  const int64_t threads = (rows + 15) / 16 * per_tile;
  k_pack<<<blocks_for(threads), kBlock, 0, (hipStream_t)stream>>>(
      (const uint8_t*)codes, (const uint8_t*)scales, (const uint8_t*)codes2,
      (const uint8_t*)scales2, rows, K, (uint8_t*)packed);
  return launched("mx4_pack");
}

}  // extern "C"
