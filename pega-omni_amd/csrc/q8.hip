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
constexpr int kTile = 64;       // keys per step: four blocks

// Keys per split of a row of len keys: the plan's, or more where a row is
// longer than the plan's bound (whole tiles).
__device__ __forceinline__ int split_len_of(const DecodeQ8Args& a, int len) {
  return max(a.chunk, ((len + a.splits - 1) / a.splits + kTile - 1) / kTile * kTile);
}

// One workgroup per (split, K/V head, row): a tile of 64 keys at a time, scores
// into LDS, the softmax's running maximum and sum per query head, and thread d
// (of 128) adds up dim d.
template <int FMT>
__global__ __launch_bounds__(kThreads) void decode_q8(DecodeQ8Args a) {
  const int split = blockIdx.x, kh = blockIdx.y, n = blockIdx.z, G = a.hq / a.hk, tid = threadIdx.x;
  const int p = a.pos[n];
  const int len = p < 0 ? 0 : p + 1;
  const int64_t h0 = (int64_t)n * a.hq + kh * G;
  if (len == 0) {
    if (split == 0)
      for (int i = tid; i < G * kHead; i += kThreads) a.out[h0 * kHead + i] = 0;
    return;
  }
  const int split_len = split_len_of(a, len);
  const int t0 = split * split_len, t1 = min(len, t0 + split_len);
  if (t0 >= len) return;
  const int32_t* pg = a.pages + a.indptr[a.ragged ? a.seq[n] : n];
  __shared__ float s_q[kMostGroup][kHead], s_p[kMostGroup][kTile], s_alpha[kMostGroup], s_m[kMostGroup], s_l[kMostGroup];
  for (int i = tid; i < G * kHead; i += kThreads)
    s_q[i / kHead][i % kHead] = lo_bf16(a.q[(int64_t)n * a.q_stride + (int64_t)kh * G * kHead + i]);
  if (tid < G) s_m[tid] = -INFINITY, s_l[tid] = 0.f;
  float acc[kMostGroup];
#pragma unroll
  for (int g = 0; g < kMostGroup; ++g) acc[g] = 0.f;
  __syncthreads();
  const auto block_of = [&](int t) {
    const int b = t / kQ8Block, j = page_index(a.pd, b);
    return page_slot(a.pd, pg[j], b);
  };
  for (int t = t0; t < t1; t += kTile) {
    {  // scores: thread (key, quarter of the query heads)
      const int key = t + (tid & 63), part = tid >> 6;
      float k[kHead];
      if (key < t1) {
        const int64_t at = block_of(key) * 2 * a.hk + kh;
        const float sc = pow2_biased(a.kv_scale[at]) * a.scale_log2;
        const uint4* src = reinterpret_cast<const uint4*>(a.kv + at * kQ8HeadBytes + (key & 15) * kHead);
#pragma unroll
        for (int i = 0; i < kHead / 16; ++i) {
          const uint4 w = src[i];
          from_bytes<FMT>(w.x, k + 16 * i), from_bytes<FMT>(w.y, k + 16 * i + 4);
          from_bytes<FMT>(w.z, k + 16 * i + 8), from_bytes<FMT>(w.w, k + 16 * i + 12);
        }
        for (int g = part; g < G; g += 4) {
          float s = 0.f;
#pragma unroll
          for (int d = 0; d < kHead; ++d) s = fmaf(k[d], s_q[g][d], s);
          s_p[g][tid & 63] = s * sc;
        }
      } else {
        for (int g = part; g < G; g += 4) s_p[g][tid & 63] = -INFINITY;
      }
    }
    __syncthreads();
    for (int g = tid >> 6; g < G; g += 4) {
      const int lane = tid & 63;
      float x = s_p[g][lane], mx = x;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d));
      const float was = s_m[g], top = fmaxf(was, mx), base = top == -INFINITY ? 0.f : top;
      x = fast_exp2(x - base);
      s_p[g][lane] = x;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) x += __shfl_xor(x, d);
      const float alpha = fast_exp2(was - base);
      if (lane == 0) s_alpha[g] = alpha, s_m[g] = top, s_l[g] = s_l[g] * alpha + x;
    }
    __syncthreads();
    if (tid < kHead) {
#pragma unroll
      for (int g = 0; g < kMostGroup; ++g)
        if (g < G) acc[g] *= s_alpha[g];
      for (int b = 0; b < kTile / kQ8Block && t + kQ8Block * b < t1; ++b) {
        const int64_t at = block_of(t + kQ8Block * b) * 2 * a.hk + a.hk + kh;
        const float sc = pow2_biased(a.kv_scale[at]);
        const uint4 w = *reinterpret_cast<const uint4*>(a.kv + at * kQ8HeadBytes + tid * kQ8Block);
        float v[16];
        from_bytes<FMT>(w.x, v), from_bytes<FMT>(w.y, v + 4), from_bytes<FMT>(w.z, v + 8), from_bytes<FMT>(w.w, v + 12);
#pragma unroll
        for (int i = 0; i < kQ8Block; ++i) {
          const float x = t + kQ8Block * b + i < t1 ? v[i] * sc : 0.f;
#pragma unroll
          for (int g = 0; g < kMostGroup; ++g)
            if (g < G) acc[g] = fmaf(s_p[g][kQ8Block * b + i], x, acc[g]);
        }
      }
    }
    __syncthreads();
  }
  if (tid < kHead) {
#pragma unroll
    for (int g = 0; g < kMostGroup; ++g) {
      if (g >= G) break;
      const float o = acc[g] / s_l[g];
      if (split_len >= len) {
        a.out[(h0 + g) * kHead + tid] = (bf16_t)f2bf(o);
      } else {
        a.ws_o[((h0 + g) * a.splits + split) * kHead + tid] = o;
        if (tid == 0) a.ws_lse[(h0 + g) * a.splits + split] = s_m[g] + __log2f(s_l[g]);
      }
    }
  }
}

// Merge the splits of a (row, head): sum of o_i 2^(lse_i - max) over the sum of
// those weights.
__global__ __launch_bounds__(kHead) void merge_q8(DecodeQ8Args a) {
  const int64_t h = blockIdx.x;
  const int n = (int)(h / a.hq), d = threadIdx.x;
  const int len = a.pos[n] < 0 ? 0 : a.pos[n] + 1;
  const int split_len = split_len_of(a, len);
  if (split_len >= len) return;
  const int used = (len + split_len - 1) / split_len;
  const float* lse = a.ws_lse + h * a.splits;
  float top = -INFINITY;
  for (int i = 0; i < used; ++i) top = fmaxf(top, lse[i]);
  float num = 0.f, den = 0.f;
  for (int i = 0; i < used; ++i) {
    const float w = fast_exp2(lse[i] - top);
    num = fmaf(a.ws_o[(h * a.splits + i) * kHead + d], w, num);
    den += w;
  }
  a.out[h * kHead + d] = (bf16_t)f2bf(num / den);
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
    merge_q8<<<dim3((unsigned)(rows * a.hq)), kHead, 0, stream>>>(a);
    return check_launch();
  }
  return 0;
}

}  // namespace omni
