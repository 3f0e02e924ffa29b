// Device helpers shared by the kernels that read the 8-bit block cache (q8.hip,
// rows.hip, tiled.hip): stored bytes to bf16, and the splits of a row's keys.
#pragma once
#include "common.h"
#include "indexing.h"
#include "kernels.h"

namespace omni {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int from_lane(int v, int lane) { return __builtin_amdgcn_ds_bpermute(lane << 2, v); }

// 2^(biased - 127) for 1 <= biased <= 254.
__device__ __forceinline__ float pow2_biased(int biased) { return __int_as_float(biased << 23); }

// The four values of a word of bytes.
template <int FMT>
__device__ __forceinline__ void from_bytes(uint32_t w, float* v) {
  if constexpr (FMT == kQ8E4m3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = (float)(int8_t)(w >> (8 * i));
  }
}

// Eight stored bytes as bf16, exactly (E4M3 has 4 significant bits, the integers 7).
template <int FMT>
__device__ __forceinline__ bf16x8 bf16_of(uint32_t w0, uint32_t w1) {
  uint4 u;
  if constexpr (FMT == kQ8E4m3) {
    u.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w0, 1.f, false));
    u.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w0, 1.f, true));
    u.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w1, 1.f, false));
    u.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w1, 1.f, true));
  } else {
    float v[8];
    from_bytes<FMT>(w0, v), from_bytes<FMT>(w1, v + 4);
    u.x = pack_bf16x2(v[0], v[1]), u.y = pack_bf16x2(v[2], v[3]);
    u.z = pack_bf16x2(v[4], v[5]), u.w = pack_bf16x2(v[6], v[7]);
  }
  return __builtin_bit_cast(bf16x8, u);
}

// Lanes col < 8 of 16 keep x and take their y from lane col + 8's x; lanes
// col >= 8 keep y and take their x from lane col - 8's y.
__device__ __forceinline__ void trade_halves(uint4& x, uint4& y) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const int x0 = (int)(&x.x)[w], y0 = (int)(&y.x)[w];
    (&x.x)[w] = (uint32_t)__builtin_amdgcn_update_dpp(x0, y0, 0x128, 0xf, 0xc, false);
    (&y.x)[w] = (uint32_t)__builtin_amdgcn_update_dpp(y0, x0, 0x128, 0xf, 0x3, false);
  }
}

// The larger of v in the four lanes with the same lane % 16.
__device__ __forceinline__ float max_of_groups(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Keys per split of a row of len keys: the plan's, or more where a row is
// longer than the plan's bound (multiples of 64 keys, as the plan's).
__device__ __forceinline__ int split_len_of(int chunk, int splits, int len) {
  return max(chunk, ((len - 1) / splits + 64) / 64 * 64);
}

// rotated_split evens out the splits over the XCDs; but an XCD hands its
// workgroups to its 32 CUs in turn, and where S divides 32 its CU would get the
// same split index from every one of them (a row's last splits are the ones that
// are short or empty). So the rotation moves on by one every 256 workgroups too.
__device__ __forceinline__ int spread_split(int slot, int u, int S) {
  return (int)((rotated_split(slot, u, S) + (((int64_t)S * u) >> 8)) % S);
}

}  // namespace omni
