// The 8-bit block cache (gfx950, wave64): the rotary + quantized write before
// attention, and decode attention over it.
//
// A block is 16 tokens of a page (pages are multiples of 16 tokens). Per K or V
// head it holds 16 x 128 bytes, FP8 E4M3 or signed integers, and one exponent e:
// a byte b stands for value(b) 2^(e - 127). e is the smallest exponent that
// brings the largest finite magnitude of the block's head into the format's
// range (448 or 127), so a growing block re-scales by an exact power of two.
// K heads lie [16 tokens][128 dims]; V heads [128 dims][16 tokens].
#include "common.h"
#include "kernels.h"
#include "rotary.h"

#include <algorithm>

namespace omni {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float row16_max(float v) {
  v = fmaxf(v, dpp<kQuadSwap1>(v));
  v = fmaxf(v, dpp<kQuadSwap2>(v));
  v = fmaxf(v, dpp<kRowHalfMirror>(v));
  v = fmaxf(v, dpp<kRowMirror>(v));
  return v;
}

template <int CTRL>
__device__ __forceinline__ int dpp_or(int v) {
  return v | __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}
__device__ __forceinline__ int row16_or(int v) {
  return dpp_or<kRowMirror>(dpp_or<kRowHalfMirror>(dpp_or<kQuadSwap2>(dpp_or<kQuadSwap1>(v))));
}

// 2^(biased - 127) for 1 <= biased <= 254.
__device__ __forceinline__ float pow2_biased(int biased) { return __int_as_float(biased << 23); }

// The exponent of a block whose largest finite magnitude is amax: from amax =
// m 2^x with 1 <= m < 2, and top = 1.75 2^8 (448) or 1.984375 2^6 (127).
template <int FMT>
__device__ __forceinline__ int block_exponent(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const uint32_t top = __float_as_uint(FMT == kQ8E4m3 ? 448.f : 127.f);
  const int e = (int)(bits >> 23) - (int)(top >> 23) + 127 + ((bits & 0x7fffffu) > (top & 0x7fffffu) ? 1 : 0);
  return max(e, 1);
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Four values, already divided by the block's scale, to four bytes. E4M3 holds
// no infinity: infinities become NaN. Integers hold neither: a NaN becomes 0, an
// infinity the largest of its sign.
template <int FMT>
__device__ __forceinline__ uint32_t to_bytes(float a, float b, float c, float d) {
  if constexpr (FMT == kQ8E4m3) {
    const float nan = __uint_as_float(0x7fc00000u);
    a = finite(a) ? a : nan, b = finite(b) ? b : nan, c = finite(c) ? c : nan, d = finite(d) ? d : nan;
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    const auto one = [](float x) {
      const float r = fminf(fmaxf(rintf(x), -127.f), 127.f);
      return (uint32_t)(int)(x != x ? 0.f : r) & 0xffu;
    };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
  }
}

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

template <int FMT>
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float by) {
  float v[4];
  from_bytes<FMT>(w, v);
  return to_bytes<FMT>(v[0] * by, v[1] * by, v[2] * by, v[3] * by);
}

// cos and sin of pairs 8 (c & 7) .. + 7 at position p, for lane c of a DPP row.
// The angle p theta^(-i/64) is reduced to a fraction of a turn in 64 bits
// (theta^(-1/64) raised by squaring): in 32 it is off by 2^-8 at positions past
// 65536. Lanes c and c ^ 8 need the same eight pairs and compute four each.
__device__ __forceinline__ void turn_of(const RopeQ8Args& a, int p, int c, float* cs, float* sn) {
  const bool lo = c < 8;
  const int i0 = 8 * (c & 7) + (lo ? 0 : 4);
  double f = (double)p * 0.15915494309189535;  // turns per radian
  double r = a.inv_theta64;
  const double r1 = r;
#pragma unroll
  for (int b = 0; b < 6; ++b) {
    if (i0 >> b & 1) f *= r;
    r *= r;
  }
  float c4[4], s4[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float t = (float)(f - rint(f));
    sincospif(2.f * t, &s4[e], &c4[e]);
    f *= r1;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float co = dpp<kRowRor8>(c4[e]), so = dpp<kRowRor8>(s4[e]);
    cs[e] = lo ? c4[e] : co, cs[e + 4] = lo ? co : c4[e];
    sn[e] = lo ? s4[e] : so, sn[e + 4] = lo ? so : s4[e];
  }
}

// Workgroup (row n, y): y < hk writes K/V head y of row n's block, if none of the
// 15 rows before n is in that block: thread group t (16 lanes, 8 dims each) takes
// the block's token t, the last of rows n .. n + 15 that has its slot, an old
// token (re-scaled if the exponent grows) or, in a block whose token 0 is
// written, zeros. y >= hk turns 16 of row n's q heads.
template <int FMT>
__global__ __launch_bounds__(kThreads) void rope_q8(RopeQ8Args a) {
  const int n = blockIdx.x, c = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int slot = a.slots[n];
  if (slot < 0) return;
  if ((int)blockIdx.y >= a.hk) {
    const int head = 16 * (blockIdx.y - a.hk) + grp;
    if (head >= a.hq) return;
    float x[8], w[8], v[8], o[8], cs[8], sn[8];
    widen8(ldg16(a.qkv + (int64_t)n * a.ld + (int64_t)head * kHead + 8 * c), x);
    widen8(ldg16(a.q_norm + 8 * c), w);
    turn_of(a, a.pos[n], c, cs, sn);
    rms_norm_head(x, w, a.eps, v);
    rotate_half(v, cs, sn, c < 8, o);
    *reinterpret_cast<uint4*>(a.q + (int64_t)n * a.q_ld + (int64_t)head * kHead + 8 * c) = pack8(o);
    return;
  }
  // Lane c of every group looks at rows n + c and n - 1 - c.
  const int ahead = n + c < a.rows ? a.slots[n + c] : -1;
  const int behind = c < kQ8Block - 1 && n - 1 - c >= 0 ? a.slots[n - 1 - c] : -1;
  if (__any(behind >= 0 && behind >> 4 == slot >> 4)) return;
  const bool here = ahead >= 0 && ahead >> 4 == slot >> 4;
  const int written = row16_or(here ? 1 << (ahead & 15) : 0);
  const bool keep = !(written & 1);  // the block goes on: its other tokens stay
  const uint32_t mine = (uint32_t)(__ballot(here && (ahead & 15) == grp) >> (threadIdx.x & 48)) & 0xffffu;
  const bool is_new = mine != 0;
  const int kh = blockIdx.y, row = n + 31 - __builtin_clz(mine | 1);
  const int64_t block = slot >> 4;
  uint8_t* kb = a.kv + (block * 2 * a.hk + kh) * kQ8HeadBytes;
  uint8_t* vb = kb + (int64_t)a.hk * kQ8HeadBytes;
  uint8_t* eb = a.kv_scale + block * 2 * a.hk + kh;
  __shared__ float s_max[2][16];
  __shared__ uint32_t s_v[kHead * 4];  // V bytes [128 dims][16 tokens]

  float kx[8], vx[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) kx[e] = vx[e] = 0.f;
  if (is_new) {
    const bf16_t* src = a.qkv + (int64_t)row * a.ld + (int64_t)(a.hq + kh) * kHead + 8 * c;
    float x[8], w[8], v[8], cs[8], sn[8];
    widen8(ldg16(src), x);
    widen8(ldg16(src + (int64_t)a.hk * kHead), vx);
    widen8(ldg16(a.k_norm + 8 * c), w);
    turn_of(a, a.pos[row], c, cs, sn);
    rms_norm_head(x, w, a.eps, v);
    rotate_half(v, cs, sn, c < 8, kx);
    const uint4 kr = pack8(kx);
    widen8(kr, kx);  // the cache holds what the bf16 row holds
    if (a.k) *reinterpret_cast<uint4*>(a.k + (int64_t)row * a.k_ld + (int64_t)kh * kHead + 8 * c) = kr;
  }
  float km = 0.f, vm = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    km = fmaxf(km, finite(kx[e]) ? fabsf(kx[e]) : 0.f);
    vm = fmaxf(vm, finite(vx[e]) ? fabsf(vx[e]) : 0.f);
  }
  km = row16_max(km), vm = row16_max(vm);
  if (c == 0) s_max[0][grp] = km, s_max[1][grp] = vm;
  __syncthreads();
  km = row16_max(s_max[0][c]), vm = row16_max(s_max[1][c]);
  const int k_old = keep ? eb[0] : 1, v_old = keep ? eb[a.hk] : 1;
  const int k_e = max(k_old, block_exponent<FMT>(km)), v_e = max(v_old, block_exponent<FMT>(vm));
  const float ki = pow2_biased(254 - k_e), vi = pow2_biased(254 - v_e);
  __syncthreads();  // every thread has the old exponents
  if (threadIdx.x == 0) eb[0] = (uint8_t)k_e, eb[a.hk] = (uint8_t)v_e;

  uint2* kd = reinterpret_cast<uint2*>(kb + grp * kHead + 8 * c);
  uint2 kw = make_uint2(0, 0);
  if (is_new) {
    kw.x = to_bytes<FMT>(kx[0] * ki, kx[1] * ki, kx[2] * ki, kx[3] * ki);
    kw.y = to_bytes<FMT>(kx[4] * ki, kx[5] * ki, kx[6] * ki, kx[7] * ki);
  } else if (keep) {
    const float by = pow2_biased(max(127 + k_old - k_e, 1));
    kw = *kd;
    if (k_e > k_old) kw = make_uint2(rescaled<FMT>(kw.x, by), rescaled<FMT>(kw.y, by));
  }
  *kd = kw;
  // V: the new tokens' bytes through LDS into [dim][token] order.
  uint8_t* sv = reinterpret_cast<uint8_t*>(s_v);
  const uint32_t w0 = to_bytes<FMT>(vx[0] * vi, vx[1] * vi, vx[2] * vi, vx[3] * vi);
  const uint32_t w1 = to_bytes<FMT>(vx[4] * vi, vx[5] * vi, vx[6] * vi, vx[7] * vi);
#pragma unroll
  for (int e = 0; e < 8; ++e) sv[(8 * c + e) * kQ8Block + grp] = (uint8_t)((e < 4 ? w0 : w1) >> (8 * (e & 3)));
  __syncthreads();
  if (threadIdx.x < kHead) {
    uint4* vd = reinterpret_cast<uint4*>(vb + threadIdx.x * kQ8Block);
    const uint4 add = *reinterpret_cast<const uint4*>(sv + threadIdx.x * kQ8Block);
    uint32_t out[4] = {add.x, add.y, add.z, add.w};
    if (keep) {
      const uint4 was = *vd;
      const uint32_t old[4] = {was.x, was.y, was.z, was.w};
      const float by = pow2_biased(max(127 + v_old - v_e, 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t stay = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          if (!(written >> (4 * i + b) & 1)) stay |= 0xffu << (8 * b);
        out[i] = (out[i] & ~stay) | ((v_e > v_old ? rescaled<FMT>(old[i], by) : old[i]) & stay);
      }
    }
    *vd = make_uint4(out[0], out[1], out[2], out[3]);
  }
}

// ------------------------------------------------------------------- decode

constexpr int kMostGroup = 16;  // query heads per K/V head
constexpr int kTile = 32;       // keys per step: two blocks
constexpr int kIds = 64 / (kTile / kQ8Block);  // tiles whose blocks a wave looks up at once

// Keys per split of a row of len keys: the plan's, or more where a row is
// longer than the plan's bound (multiples of 64 keys, as the plan's).
__device__ __forceinline__ int split_len_of(const DecodeQ8Args& a, int len) {
  return max(a.chunk, ((len + a.splits - 1) / a.splits + 63) / 64 * 64);
}

// rotated_split evens out the splits over the XCDs; but an XCD hands its
// workgroups to its 32 CUs in turn, and where S divides 32 its CU would get the
// same split index from every one of them (a row's last splits are the ones that
// are short or empty). So the rotation moves on by one every 256 workgroups too.
__device__ __forceinline__ int spread_split(int slot, int u, int S) {
  return (int)((rotated_split(slot, u, S) + (((int64_t)S * u) >> 8)) % S);
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

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
    u = pack8(v);
  }
  return __builtin_bit_cast(bf16x8, u);
}

__device__ __forceinline__ int from_lane(int v, int lane) { return __builtin_amdgcn_ds_bpermute(lane << 2, v); }

// The larger of v in the four lanes with the same lane % 16.
__device__ __forceinline__ float max_of_groups(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

constexpr int kDecodeWaves = kThreads / 64;
constexpr int kBlocksPerTile = kTile / kQ8Block;

// One workgroup per (split, K/V head, row); its waves take the split's 32-key
// tiles in turn, each with a running maximum, sum and O of its own, merged
// through LDS at the end. Lane l is column n = l % 16 (query head) and group
// g = l / 16 of the v_mfma_f32_16x16x32_bf16 operands:
//   S^T (16 keys x 16 heads), two of them: row 4 x + r of product j is token
//     8 (x % 2) + 4 j + r of the tile's block x / 2, so a lane ends with tokens
//     8 (g % 2) .. + 7 of block g / 2 for its head, in order, which is P^T's
//     operand as it stands: no data crosses lanes between the two products but
//     the maximum.
//   O^T (16 dims x 16 heads) += V^T . P^T: V lies [dim][token] in the cache. A
//     lane loads the 16 tokens of one dim (groups 2 b and 2 b + 1 two dims of
//     block b) and the two groups trade halves, which gives each its tokens of
//     both dims.
// P is carried as two bf16 terms (hi + lo, 16 bits): the matrix cores are a
// tenth of the time. Both scales act per block, that is per lane: on the scores
// and, an exact power of two, on P.
template <int FMT>
__global__ __launch_bounds__(kThreads, 4) void decode_q8(DecodeQ8Args a) {
  const int kh = blockIdx.y, n = blockIdx.z, G = a.hq / a.hk, tid = threadIdx.x;
  const int split = spread_split(blockIdx.x, kh + a.hk * n, a.splits);
  const int p = a.pos[n];
  const int32_t* pg = a.pages + a.indptr[a.ragged ? max(a.seq[n], 0) : n];
  const int len = p < 0 ? 0 : p + 1;
  const int64_t h0 = (int64_t)n * a.hq + kh * G;
  if (len == 0) {
    if (split == 0)
      for (int i = tid; i < G * kHead; i += kThreads) a.out[h0 * kHead + i] = 0;
    return;
  }
  const int split_len = split_len_of(a, len);
  if ((int64_t)split * split_len >= len) return;
  const int t0 = split * split_len, t1 = min(len, t0 + split_len);
  const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int tiles = (t1 - t0 + kTile - 1) / kTile;
  const int mine = (tiles - wave + kDecodeWaves - 1) / kDecodeWaves;  // tiles wave, wave + 4, ..
  const int last_block = (t1 - 1) / kQ8Block;

  // q: product step kk holds dims 64 (kk / 2) + 16 g + 8 (kk % 2) .. + 7.
  bf16x8 q[4];
  {
    const bf16_t* qp = a.q + (int64_t)n * a.q_stride + (int64_t)(kh * G + min(col, G - 1)) * kHead;
#pragma unroll
    for (int kk = 0; kk < 4; ++kk)
      q[kk] = __builtin_bit_cast(bf16x8, ldg16(qp + 64 * (kk >> 1) + 16 * grp + 8 * (kk & 1)));
  }

  // Blocks of kIds of the wave's tiles at a time: lane 2 k + b holds block b of
  // tile k and its two exponents.
  const int64_t row_blocks = 2LL * a.hk;
  int ids = 0, exps = 0;
  auto next_blocks = [&](int k0) __attribute__((always_inline)) {
    const int tile = wave + kDecodeWaves * (k0 + (lane >> 1));
    const int b = min(t0 / kQ8Block + tile * kBlocksPerTile + (lane & 1), last_block);
    ids = (int)page_slot(a.pd, pg[page_index(a.pd, b)], b);
    const uint8_t* e = a.kv_scale + ids * row_blocks + kh;
    exps = e[0] | e[a.hk] << 16;
  };

  uint4 kr[2][2], vr[4];
  auto load_k = [&](int k) __attribute__((always_inline)) {
    const int64_t block = from_lane(ids, 2 * (k & (kIds - 1)) + (col >> 3));
    const uint8_t* kb = a.kv + (block * row_blocks + kh) * kQ8HeadBytes + (2 * (col & 4) + (col & 3)) * kHead + 16 * grp;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) kr[j][c] = ldg16(kb + 4 * j * kHead + 64 * c);
  };
  auto load_v = [&](int k) __attribute__((always_inline)) {
    const int64_t block = from_lane(ids, 2 * (k & (kIds - 1)) + (grp >> 1));
    const uint8_t* vb = a.kv + (block * row_blocks + a.hk + kh) * kQ8HeadBytes + (16 * (grp & 1) + col) * kQ8Block;
#pragma unroll
    for (int i = 0; i < 4; ++i) vr[i] = ldg16_stream(vb + i * 32 * kQ8Block);
  };

  f32x4 o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  if (mine > 0) {
    next_blocks(0);
    load_k(0);
  }
  for (int k = 0; k < mine; ++k) {
    // V of this tile, then (when its scores are taken) K of the next: one of the two is always in flight.
    load_v(k);
    const int e2 = from_lane(exps, 2 * (k & (kIds - 1)) + (grp >> 1));
    const int left = t1 - t0 - (wave + kDecodeWaves * k) * kTile;  // keys from this tile on
    float s[8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_of<FMT>(kr[j][c].x, kr[j][c].y), q[2 * c], d, 0, 0, 0);
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bf16_of<FMT>(kr[j][c].z, kr[j][c].w), q[2 * c + 1], d, 0, 0, 0);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) s[4 * j + r] = d[r];
    }
    if (k + 1 < mine) {
      if (((k + 1) & (kIds - 1)) == 0) next_blocks(k + 1);
      load_k(k + 1);
    }
    const float ks = pow2_biased(e2 & 0xff) * a.scale_log2, vs = pow2_biased(e2 >> 16);
#pragma unroll
    for (int t = 0; t < 8; ++t) s[t] *= ks;
    if (left < kTile) {  // the row's last tile: nothing past its last token counts, whatever it holds
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (8 * grp + t >= left) s[t] = -INFINITY;
      const int tokens = left - kQ8Block * (grp >> 1);  // of this lane's block
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const int n_ok = min(max(tokens - 4 * w, 0), 4);
        const uint32_t stay = n_ok == 4 ? ~0u : (1u << (8 * n_ok)) - 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) (&vr[i].x)[w] &= stay;
      }
    }
    float mx = s[0];
#pragma unroll
    for (int t = 1; t < 8; ++t) mx = fmaxf(mx, s[t]);
    mx = max_of_groups(mx);
    // The base moves only when the maximum grows by more than 8 (log2): p <= 2^8.
    const bool grow = mx > m + 8.f;
    if (__any(grow)) {
      const float alpha = grow ? fast_exp2(m - mx) : 1.f;
      m = grow ? mx : m;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] *= alpha;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      s[t] = fast_exp2(s[t] - base);
      l += s[t];
      s[t] *= vs;
    }
    const uint4 hi = pack8(s);
    float rest[8];
    widen8(hi, rest);
#pragma unroll
    for (int t = 0; t < 8; ++t) rest[t] = s[t] - rest[t];
    const bf16x8 ph = __builtin_bit_cast(bf16x8, hi), pl = __builtin_bit_cast(bf16x8, pack8(rest));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // Even groups keep tokens 0-7 of their dim and take those of the odd group's, and the other way round.
      const auto a0 = __builtin_amdgcn_permlane16_swap(vr[i].x, vr[i].z, false, false);
      const auto a1 = __builtin_amdgcn_permlane16_swap(vr[i].y, vr[i].w, false, false);
      const bf16x8 v0 = bf16_of<FMT>(a0[0], a1[0]), v1 = bf16_of<FMT>(a0[1], a1[1]);
      o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, ph, o[2 * i], 0, 0, 0);
      o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, ph, o[2 * i + 1], 0, 0, 0);
      o[2 * i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v0, pl, o[2 * i], 0, 0, 0);
      o[2 * i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v1, pl, o[2 * i + 1], 0, 0, 0);
    }
  }

  // The waves' parts, merged: O rows [head][dim], then (m, l).
  __shared__ float s_o[kDecodeWaves][kMostGroup][kHead + 4], s_m[kDecodeWaves][kMostGroup], s_l[kDecodeWaves][kMostGroup];
  l += xor_lane(l, 16);
  l += xor_lane(l, 32);
  if (col < G) {
#pragma unroll
    for (int i = 0; i < 8; ++i) *reinterpret_cast<f32x4*>(&s_o[wave][col][16 * i + 4 * grp]) = o[i];
    if (grp == 0) s_m[wave][col] = m, s_l[wave][col] = l;
  }
  __syncthreads();
  const int waves = min(tiles, kDecodeWaves);
  for (int i = tid; i < G * kHead; i += kThreads) {
    const int g = i / kHead, d = i % kHead;
    float top = s_m[0][g];
    for (int w = 1; w < waves; ++w) top = fmaxf(top, s_m[w][g]);
    const float base = top == -INFINITY ? 0.f : top;
    float num = 0.f, den = 0.f;
    for (int w = 0; w < waves; ++w) {
      const float e = fast_exp2(s_m[w][g] - base);
      num = fmaf(s_o[w][g][d], e, num);
      den = fmaf(s_l[w][g], e, den);
    }
    if (split_len >= len) {
      a.out[(h0 + g) * kHead + d] = (bf16_t)f2bf(num / den);
    } else {
      // den = 0: every score is -inf, and the split weighs nothing beside the others.
      a.ws_o[((h0 + g) * a.splits + split) * kHead + d] = den == 0.f ? 0.f : num / den;
      if (d == 0) a.ws_lse[(h0 + g) * a.splits + split] = base + __log2f(den);
    }
  }
}

// Merge the splits of a (row, head): sum of o_i 2^(lse_i - max) over the sum of
// those weights. 32 lanes of 4 dims, eight groups that take the splits in turn,
// kMergeBatch at a time: the partials are asked for before their weights are
// known, so a row of up to 32 splits costs one memory round trip behind pos.
constexpr int kMergeGroups = kThreads / 32;
constexpr int kMergeBatch = 4;

__global__ __launch_bounds__(kThreads) void merge_q8(DecodeQ8Args a) {
  const int64_t h = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, grp = tid >> 5;
  const float* lse = a.ws_lse + h * a.splits;
  const float* part = a.ws_o + h * a.splits * kHead + 4 * lane;
  const int p = a.pos[h / a.hq];
  const int len = p < 0 ? 0 : p + 1;
  const int split_len = split_len_of(a, len);
  if (split_len >= len) return;
  const int used = (len + split_len - 1) / split_len;
  f32x4 num = {0.f, 0.f, 0.f, 0.f};
  float top = -INFINITY, den = 0.f;  // of this group's splits
  for (int i0 = grp; i0 < used; i0 += kMergeGroups * kMergeBatch) {
    f32x4 o[kMergeBatch];
    float e[kMergeBatch];
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) {
      const int i = min(i0 + kMergeGroups * j, used - 1);
      e[j] = lse[i];
      o[j] = *reinterpret_cast<const f32x4*>(part + (int64_t)i * kHead);
    }
    float mx = top;
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) mx = fmaxf(mx, e[j]);  // one seen twice changes no maximum
    const float base = mx == -INFINITY ? 0.f : mx, alpha = fast_exp2(top - base);
    top = mx;
    num *= alpha, den *= alpha;
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) {
      if (i0 + kMergeGroups * j >= used) break;
      const float w = fast_exp2(e[j] - base);
      num += o[j] * w, den += w;
    }
  }
  __shared__ f32x4 s_num[kMergeGroups][32];
  __shared__ float s_top[kMergeGroups], s_den[kMergeGroups];
  s_num[grp][lane] = num;
  if (lane == 0) s_top[grp] = top, s_den[grp] = den;
  __syncthreads();
  if (grp != 0) return;
  float mx = -INFINITY;
#pragma unroll
  for (int g = 0; g < kMergeGroups; ++g) mx = fmaxf(mx, s_top[g]);
  const float base = mx == -INFINITY ? 0.f : mx;
  num = f32x4{0.f, 0.f, 0.f, 0.f}, den = 0.f;
#pragma unroll
  for (int g = 0; g < kMergeGroups; ++g) {
    const float w = fast_exp2(s_top[g] - base);
    num += s_num[g][lane] * w;
    den = fmaf(s_den[g], w, den);
  }
  *reinterpret_cast<uint2*>(a.out + h * kHead + 4 * lane) =
      make_uint2(pack_bf16x2(num[0] / den, num[1] / den), pack_bf16x2(num[2] / den, num[3] / den));
}

}  // namespace

int launch_rope_q8(const RopeQ8Args& a, hipStream_t stream) {
  const dim3 grid(a.rows, a.hk + (a.hq + 15) / 16);
  if (a.format == kQ8E4m3)
    rope_q8<kQ8E4m3><<<grid, kThreads, 0, stream>>>(a);
  else
    rope_q8<kQ8Int8><<<grid, kThreads, 0, stream>>>(a);
  return check_launch();
}

int launch_decode_q8(const DecodeQ8Args& a, int rows, hipStream_t stream) {
  const dim3 grid(a.splits, a.hk, rows);
  if (a.format == kQ8E4m3)
    decode_q8<kQ8E4m3><<<grid, kThreads, 0, stream>>>(a);
  else
    decode_q8<kQ8Int8><<<grid, kThreads, 0, stream>>>(a);
  if (check_launch() != 0) return -3;
  if (a.splits > 1) {
    merge_q8<<<dim3((unsigned)(rows * a.hq)), kThreads, 0, stream>>>(a);
    return check_launch();
  }
  return 0;
}

}  // namespace omni
