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
#include "q8_bytes.h"
#include "rotary.h"

#include <algorithm>

namespace omni {

namespace {

constexpr int kThreads = kQ8Threads;

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, a), __builtin_bit_cast(u16x2_t, b)));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max_u32(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false));
}
// The larger of each over the 16 lanes of a DPP row (side by side: a DPP read waits
// for the write before it).
__device__ __forceinline__ void row16_max2(uint32_t& a, uint32_t& b) {
  a = dpp_max_u32<kQuadSwap1>(a), b = dpp_max_u32<kQuadSwap1>(b);
  a = dpp_max_u32<kQuadSwap2>(a), b = dpp_max_u32<kQuadSwap2>(b);
  a = dpp_max_u32<kRowHalfMirror>(a), b = dpp_max_u32<kRowHalfMirror>(b);
  a = dpp_max_u32<kRowMirror>(a), b = dpp_max_u32<kRowMirror>(b);
}

// The exponent of a block whose largest finite magnitude has the bf16 bits `most`:
// from most = m 2^x with 1 <= m < 2, and top = 1.75 2^8 (448) or 1.984375 2^6 (127).
template <int FMT>
__device__ __forceinline__ int block_exponent(int most) {
  constexpr int top = FMT == kQ8E4m3 ? 0x43e0 : 0x42fe;
  return max((most >> 7) - (top >> 7) + 127 + ((most & 0x7f) > (top & 0x7f) ? 1 : 0), 1);
}

// Four values, already divided by the block's scale, to four bytes. E4M3 holds
// no infinity: infinities become NaN. Integers hold neither: a NaN becomes 0, an
// infinity the largest of its sign.
template <int FMT>
__device__ __forceinline__ uint32_t to_bytes(float a, float b, float c, float d) {
  if constexpr (FMT == kQ8E4m3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    const auto one = [](float x) {
      const float r = fminf(fmaxf(rintf(x), -127.f), 127.f);
      return (uint32_t)(int)(x != x ? 0.f : r) & 0xffu;
    };
    return one(a) | one(b) << 8 | one(c) << 16 | one(d) << 24;
  }
}

typedef short s16x2_t __attribute__((ext_vector_type(2)));

// Four bf16 values divided by 2^(biased - 127), to bytes. E4M3 has an instruction
// for it, which rounds the quotient once; the integers are multiplied (exactly).
template <int FMT>
__device__ __forceinline__ uint32_t to_bytes(uint32_t w0, uint32_t w1, int biased) {
  if constexpr (FMT == kQ8E4m3) {
    const float scale = pow2_biased(biased);
    s16x2_t r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, w0), scale, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(r, __builtin_bit_cast(bf16x2_t, w1), scale, true);
    return __builtin_bit_cast(uint32_t, r);
  } else {
    const float by = pow2_biased(254 - biased);
    return to_bytes<FMT>(lo_bf16(w0) * by, hi_bf16(w0) * by, lo_bf16(w1) * by, hi_bf16(w1) * by);
  }
}

template <int FMT>
__device__ __forceinline__ uint32_t rescaled(uint32_t w, float by) {
  float v[4];
  from_bytes<FMT>(w, v);
  return to_bytes<FMT>(v[0] * by, v[1] * by, v[2] * by, v[3] * by);
}

constexpr double kTurnsPerRadian = 0.15915494309189535;

// sin and cos of f turns. The nearest quarter turn goes in 64
// bits, so that the rest keeps f32's relative precision (a fraction of a whole
// turn rounded to f32 was off by 2e-7 radians, and a third of the bf16 values of
// K and q that differ from a 64-bit computation's differed for it). The rest, x
// of at most pi / 4, takes the Taylor series to x^9 and x^10, whose next terms
// are below 2e-9: a third of the instructions of the library's call.
__device__ __forceinline__ void sincos_turns(double f, float* sn, float* cs) {
  const double k = rint(4. * f);
  const float x = (float)(fma(-0.25, k, f) * 6.283185307179586), y = x * x;
  const float s = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), x);
  const float c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
  const int q = (int)(4. * __builtin_amdgcn_fract(0.25 * k));  // k modulo 4
  const float s1 = q & 1 ? c : s, c1 = q & 1 ? s : c;
  *sn = __int_as_float(__float_as_int(s1) ^ (q & 2) << 30);
  *cs = __int_as_float(__float_as_int(c1) ^ (q + 1 & 2) << 30);
}

// cos and signed sin of pairs 8 (c & 7) .. + 7 at position p, for lane c of a DPP
// row: minus sin in the lanes of the pairs' first elements (c < 8).
// The angle p theta^(-i/64) is reduced to a fraction of a turn in 64 bits
// (theta^(-1/64) raised by squaring): in 32 it is off by 2^-8 at positions past
// 65536. Lanes c and c ^ 8 need the same eight pairs and compute four each.
__device__ __forceinline__ void turn_of(const RopeQ8Args& a, int p, int c, float* cs, float* sn) {
  const bool lo = c < 8;
  const int i0 = 8 * (c & 7) + (lo ? 0 : 4);
  double f = (double)p * kTurnsPerRadian;
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
    sincos_turns(f, &s4[e], &c4[e]);
    f *= r1;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float co = dpp<kRowRor8>(c4[e]), so = dpp<kRowRor8>(s4[e]);
    cs[e] = lo ? c4[e] : co, cs[e + 4] = lo ? co : c4[e];
    sn[e] = lo ? -s4[e] : so, sn[e + 4] = lo ? -so : s4[e];
  }
}

// turn_of's values, bit for bit, through LDS: each pair's once for all heads of a row.
struct TurnLds {
  float cs[kHead / 2], sn[kHead / 2];
};

__device__ __forceinline__ void put_turn(const RopeQ8Args& a, int p, int i, TurnLds* s) {
  double f = (double)p * kTurnsPerRadian;
  double r = a.inv_theta64;
#pragma unroll
  for (int b = 0; b < 6; ++b) {
    if (b >= 2 && (i >> b & 1)) f *= r;
    r *= r;
  }
#pragma unroll
  for (int e = 0; e < 3; ++e)
    if (e < (i & 3)) f *= a.inv_theta64;
  sincos_turns(f, &s->sn[i], &s->cs[i]);
}

__device__ __forceinline__ void get_turn(const TurnLds& s, int c, float* cs, float* sn) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float t = s.sn[8 * (c & 7) + e];
    cs[e] = s.cs[8 * (c & 7) + e], sn[e] = c < 8 ? -t : t;
  }
}

// The rows of one block, as row n of a call sees them, if n is the first of
// them: thread group t (16 lanes, 8 dims of a head each) takes the block's token
// t, which is the last of rows n .. n + 15 that has its slot, an old token or, in
// a block whose token 0 is written, nothing yet.
struct BlockRows {
  int64_t block;
  int written;  // bit t: token t is written by this call
  int row;      // this group's row, -1 if its token is not written
  int twice;    // bit i: row n + i has a slot that a later row has too
};

// Lane l's slot of row n0 - 16 + l (-1 where there is none).
__device__ __forceinline__ int slots_around(const RopeQ8Args& a, int n0) {
  const int64_t row = (int64_t)n0 - 16 + (threadIdx.x & 63);
  return row >= 0 && row < a.rows ? a.slots[row] : -1;
}

// Whether row n0 + at - 16 (not skipped) is the only row of its block.
__device__ __forceinline__ bool is_alone(int around, int at) {
  const int slot = __builtin_amdgcn_readlane(around, at);
  const uint64_t same = __ballot(around >= 0 && around >> 4 == slot >> 4);
  return slot >= 0 && (same >> (at - 15) & 0x7fffffff) == 1 << 15;
}

// around: slots_around(n0); row n = n0 + at - 16, 16 <= at <= 48. Every lane of the workgroup gets the same answer.
__device__ __forceinline__ bool block_rows(int around, int at, int n, int grp, BlockRows* r) {
  asm("" : "+v"(around));  // the 16 comparisons below are made here: kept over a loop of rows they spill
  const int slot = __builtin_amdgcn_readlane(around, at);
  if (slot < 0) return false;
  const uint64_t same = __ballot(around >= 0 && around >> 4 == slot >> 4);
  if (same >> (at - 15) & 0x7fff) return false;  // one of the 15 rows before leads
  if ((same >> at & 0xffff) == 1) return false;   // alone
  r->block = slot >> 4;
  r->written = 0;
  r->row = -1;
  int last = 0;  // rows that are their token's last
#pragma unroll
  for (int t = 0; t < kQ8Block; ++t) {
    const uint32_t rows = (uint32_t)((same & __ballot((around & 15) == t)) >> at) & 0xffffu;
    if (rows == 0) continue;
    const int top = 31 - __builtin_clz(rows);
    r->written |= 1 << t;
    last |= 1 << top;
    r->row = grp == t ? n + top : r->row;
  }
  r->twice = (int)((same >> at) & 0xffffu) & ~last;
  return true;
}

// Four bytes of each lane, a token's dims 0-3 (w0) and 4-7 (w1), tokens 0..3 of
// the wave's four 16-lane rows, to four tokens of one dim: row r gets dims 2 r
// (w0) and 2 r + 1 (w1).
__device__ __forceinline__ void tokens_of_dims(uint32_t& w0, uint32_t& w1) {
  // Rows 0, 1: dims 0-3 of tokens r and r + 2; rows 2, 3: dims 4-7 of tokens r - 2 and r.
  const auto h = __builtin_amdgcn_permlane32_swap(w0, w1, false, false);
  const uint32_t x = __builtin_amdgcn_perm(h[1], h[0], 0x05010400);  // [a0 b0 a1 b1]
  const uint32_t y = __builtin_amdgcn_perm(h[1], h[0], 0x07030602);  // [a2 b2 a3 b3]
  // Even rows: dims 0, 1 (of their four) of tokens 0, 2 and 1, 3; odd rows: dims 2, 3.
  const auto q = __builtin_amdgcn_permlane16_swap(x, y, false, false);
  w0 = __builtin_amdgcn_perm(q[1], q[0], 0x05010400);
  w1 = __builtin_amdgcn_perm(q[1], q[0], 0x07030602);
}

// The largest magnitude of eight bf16 values of a lane, as bf16 bits. Bits compare
// as magnitudes do; FINITE leaves infinities and NaN out.
template <bool FINITE>
__device__ __forceinline__ uint32_t most_of(const uint4& x) {
  const auto of = [](uint32_t w) {
    w &= 0x7fff7fffu;
    if (FINITE) {
      if ((w & 0xffffu) >= 0x7f80u) w &= 0xffff0000u;
      if (w >= 0x7f800000u) w &= 0xffffu;
    }
    return w;
  };
  const uint32_t m = max_u16x2(max_u16x2(of(x.x), of(x.y)), max_u16x2(of(x.z), of(x.w)));
  return max(m & 0xffffu, m >> 16);
}

constexpr int kVTile = kHead * 4 + kHead / 8 * 4;  // dwords: a gap of 16 bytes every 8 dims spreads the banks
__device__ __forceinline__ int v_at(int dim) { return dim * 4 + (dim >> 3) * 4; }

struct KvLds {
  uint2 most[16];
  uint32_t v[kVTile];
};

// K and V of H heads at once (kh, kh + step, ..; those below hk), given this
// group's bf16 row of each (k: turned), quantized into the block. Zeros where the
// group has no row. Two barriers for all of them, which is what a head waits for:
// of 12 prompts of 25,850 rows the cache's part takes 58 us with one head at a
// time, 51 with two, 63 with four (registers).
template <int FMT, int H>
__device__ __forceinline__ void write_block(const RopeQ8Args& a, const BlockRows& r, int kh, int step, const uint4* k,
                                            const uint4* v, int c, int grp, KvLds* s) {
  const bool keep = !(r.written & 1);  // the block goes on: its other tokens stay
  uint8_t* kb = a.kv + (r.block * 2 * a.hk + kh) * kQ8HeadBytes;
  uint8_t* eb = a.kv_scale + r.block * 2 * a.hk + kh;
  const int64_t to_v = (int64_t)a.hk * kQ8HeadBytes, next = (int64_t)step * kQ8HeadBytes;
  const int k_at = grp * kHead + 8 * c, v_at_byte = (threadIdx.x & (kHead - 1)) * kQ8Block;
  // What the block holds, asked for before the exponents are known.
  int k_old[H], v_old[H];
  uint2 kw[H];
  uint4 was[H];
  uint32_t km[H], vm[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    k_old[h] = v_old[h] = 1;
    kw[h] = make_uint2(0, 0), was[h] = make_uint4(0, 0, 0, 0);
    if (keep && kh + h * step < a.hk) {
      k_old[h] = eb[h * step], v_old[h] = eb[h * step + a.hk];
      if (r.row < 0) kw[h] = *reinterpret_cast<const uint2*>(kb + h * next + k_at);
      if (threadIdx.x < kHead) was[h] = *reinterpret_cast<const uint4*>(kb + h * next + to_v + v_at_byte);
    }
    km[h] = most_of<false>(k[h]), vm[h] = most_of<false>(v[h]);
  }
  const auto of_block = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < H; ++h) {
      row16_max2(km[h], vm[h]);
      if (c == 0) s[h].most[grp] = make_uint2(km[h], vm[h]);
    }
    __syncthreads();
    uint32_t top = 0;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      km[h] = s[h].most[c].x, vm[h] = s[h].most[c].y;
      row16_max2(km[h], vm[h]);
      top = max(top, max(km[h], vm[h]));
    }
    return top;
  };
  if (of_block() >= 0x7f80u) {  // not finite, somewhere in the blocks: it does not count
    __syncthreads();
#pragma unroll
    for (int h = 0; h < H; ++h) km[h] = most_of<true>(k[h]), vm[h] = most_of<true>(v[h]);
    of_block();
  }
  int k_e[H], v_e[H];
#pragma unroll
  for (int h = 0; h < H; ++h) {
    k_e[h] = max(k_old[h], block_exponent<FMT>(km[h])), v_e[h] = max(v_old[h], block_exponent<FMT>(vm[h]));
    // V: the new tokens' bytes through LDS into [dim][token] order.
    uint32_t w0 = to_bytes<FMT>(v[h].x, v[h].y, v_e[h]), w1 = to_bytes<FMT>(v[h].z, v[h].w, v_e[h]);
    tokens_of_dims(w0, w1);
    const int at = v_at(8 * c + 2 * (grp & 3)) + (grp >> 2);
    s[h].v[at] = w0, s[h].v[at + 4] = w1;
    if (r.row >= 0) {
      kw[h] = make_uint2(to_bytes<FMT>(k[h].x, k[h].y, k_e[h]), to_bytes<FMT>(k[h].z, k[h].w, k_e[h]));
    } else if (k_e[h] > k_old[h]) {
      const float by = pow2_biased(max(127 + k_old[h] - k_e[h], 1));
      kw[h] = make_uint2(rescaled<FMT>(kw[h].x, by), rescaled<FMT>(kw[h].y, by));
    }
    if (kh + h * step < a.hk && (r.row >= 0 || !keep || k_e[h] > k_old[h]))
      *reinterpret_cast<uint2*>(kb + h * next + k_at) = kw[h];
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < H; ++h) {
    if (kh + h * step >= a.hk) break;
    if (threadIdx.x == 0) eb[h * step] = (uint8_t)k_e[h], eb[h * step + a.hk] = (uint8_t)v_e[h];  // every thread has the old ones
    if (threadIdx.x < kHead) {
      const uint4 add = *reinterpret_cast<const uint4*>(s[h].v + v_at(threadIdx.x));
      uint32_t out[4] = {add.x, add.y, add.z, add.w};
      if (keep) {
        const uint32_t old[4] = {was[h].x, was[h].y, was[h].z, was[h].w};
        const float by = pow2_biased(max(127 + v_old[h] - v_e[h], 1));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t stay = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b)
            if (!(r.written >> (4 * i + b) & 1)) stay |= 0xffu << (8 * b);
          out[i] = (out[i] & ~stay) | ((v_e[h] > v_old[h] ? rescaled<FMT>(old[i], by) : old[i]) & stay);
        }
      }
      *reinterpret_cast<uint4*>(kb + h * next + to_v + v_at_byte) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
}

// 1 / sqrt(v) to half a step: the instruction's value and a Newton step (which
// would make NaN of 1 / sqrt(infinity)).
__device__ __forceinline__ float inv_sqrt(float v) {
  const float r = rsqrtf(v);
  return v < INFINITY ? fmaf(0.5f * r, fmaf(-v * r, r, 1.f), r) : r;
}

__device__ __forceinline__ float dot2(uint32_t a, float sum) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, a), __builtin_bit_cast(bf16x2_t, a), sum, false);
}

// A head's 8 dims of this lane, normalised and turned, as bf16: x / rms rounded to
// bf16, as the model does, times the weight (exact in f32); then x cos + partner
// sin, the partner 64 dims away being lane c ^ 8's in the same register.
__device__ __forceinline__ uint4 turn_head(const RopeQ8Args& a, const uint4& raw, const float* w, const float* cs,
                                           const float* sn) {
  const float ss = dot2(raw.x, dot2(raw.y, dot2(raw.z, dot2(raw.w, 0.f))));
  const float r = inv_sqrt(fmaf(row16_sum(ss), 1.f / kHead, a.eps));
  float x[8];
  widen8(raw, x);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= r;
  widen8(pack8(x), x);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] *= w[e];
  float o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = fmaf(x[e], cs[e], dpp<kRowRor8>(x[e]) * sn[e]);
  return pack8(o);
}

// k_out of the rows whose slot a later row has too (their K goes nowhere else).
__device__ __forceinline__ void k_rows_twice(const RopeQ8Args& a, const BlockRows& r, int n, int y, int Y, int c, int grp) {
  if (!a.k || !(r.twice >> grp & 1)) return;
  const int row = n + grp;
  float cs[8], sn[8], w[8];
  turn_of(a, a.pos[row], c, cs, sn);
  widen8(ldg16(a.k_norm + 8 * c), w);
  for (int kh = y; kh < a.hk; kh += Y) {
    const uint4 raw = ldg16(a.qkv + (int64_t)row * a.ld + (int64_t)(a.hq + kh) * kHead + 8 * c);
    *reinterpret_cast<uint4*>(a.k + (int64_t)row * a.k_ld + (int64_t)kh * kHead + 8 * c) = turn_head(a, raw, w, cs, sn);
  }
}

// K and V of the only row of its block, by one wave: heads kh0 and kh0 + 1 (the
// second if there is one), each K in one 16-lane group and V in the next, 8 dims a
// lane; then all 64 lanes each head's bytes: V whole, as the token is a byte of
// every dim's 16 (lane l dims l and l + 64), K's other tokens if there is
// something to change in them. No barrier, and what a workgroup did for a head of
// one row it does for two heads of four: 64 rows of 16q/8kv 5.0 -> 4.3 us, 512 13.2 ->
// 7.9 (1.2 -> 2.1 TB/s), 512 of 32q/32kv 46 -> 26, 2200 of 32q/8kv 96 -> 35.
template <int FMT>
__device__ __forceinline__ void write_alone(const RopeQ8Args& a, int row, int slot, int kh0, const TurnLds& turn) {
  const int lane = threadIdx.x & 63, c = lane & 15, head = lane >> 5, token = slot & (kQ8Block - 1);
  const bool is_v = lane & 16, two = kh0 + 1 < a.hk, mine = head == 0 || two, keep = token != 0;
  const int64_t head0 = (int64_t)(slot >> 4) * 2 * a.hk + kh0;
  uint8_t* kb = a.kv + head0 * kQ8HeadBytes;
  uint8_t* vb = kb + (int64_t)a.hk * kQ8HeadBytes;
  uint8_t* eb = a.kv_scale + head0 + head + (is_v ? a.hk : 0);
  uint4 x = make_uint4(0, 0, 0, 0), was[2][2];
  int old = 1;
  if (mine) {
    x = ldg16_stream(a.qkv + (int64_t)row * a.ld + (int64_t)(a.hq + kh0 + head + (is_v ? a.hk : 0)) * kHead + 8 * c);
    if (keep) old = *eb;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      was[h][i] = make_uint4(0, 0, 0, 0);
      if (keep && (h == 0 || two)) was[h][i] = ldg16(vb + h * kQ8HeadBytes + (64 * i + lane) * kQ8Block);
    }
  float cs[8], sn[8], w[8];
  get_turn(turn, c, cs, sn);
  widen8(ldg16(a.k_norm + 8 * c), w);
  const uint4 k = turn_head(a, x, w, cs, sn);
  if (!is_v) x = k;
  if (mine && !is_v && a.k) *reinterpret_cast<uint4*>(a.k + (int64_t)row * a.k_ld + (int64_t)(kh0 + head) * kHead + 8 * c) = x;
  uint32_t most = most_of<false>(x), none = 0;
  if (__any(most >= 0x7f80u)) most = most_of<true>(x);  // not finite: it does not count
  row16_max2(most, none);
  const int e = max(old, block_exponent<FMT>(most));
  const uint32_t w0 = to_bytes<FMT>(x.x, x.y, e), w1 = to_bytes<FMT>(x.z, x.w, e);
  if (mine && !is_v) *reinterpret_cast<uint2*>(kb + head * kQ8HeadBytes + token * kHead + 8 * c) = make_uint2(w0, w1);
  if (mine && c == 0) *eb = (uint8_t)e;
  const int shift = 8 * (token & 3);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h == 1 && !two) break;
    const int v_old = __builtin_amdgcn_readlane(old, 32 * h + 16), v_e = __builtin_amdgcn_readlane(e, 32 * h + 16);
    const float by = pow2_biased(max(127 + v_old - v_e, 1));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t out[4] = {was[h][i].x, was[h][i].y, was[h][i].z, was[h][i].w};
      if (keep && v_e > v_old)
#pragma unroll
        for (int d = 0; d < 4; ++d) out[d] = rescaled<FMT>(out[d], by);
      const int from = 32 * h + 16 + 8 * i + (lane >> 3);
      const uint32_t byte = __builtin_amdgcn_perm(from_lane(w1, from), from_lane(w0, from), 0x0c0c0c00u | (lane & 7));
#pragma unroll
      for (int d = 0; d < 4; ++d)
        if (d == token >> 2) out[d] = (out[d] & ~(0xffu << shift)) | byte << shift;
      *reinterpret_cast<uint4*>(vb + h * kQ8HeadBytes + (64 * i + lane) * kQ8Block) = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
#pragma unroll 1
  for (int h = 0; h < (two ? 2 : 1); ++h) {
    const int k_old = __builtin_amdgcn_readlane(old, 32 * h), k_e = __builtin_amdgcn_readlane(e, 32 * h);
    if (keep && k_e == k_old) continue;
    const float by = pow2_biased(max(127 + k_old - k_e, 1));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (8 * i + (lane >> 3) == token) continue;
      uint4* at = reinterpret_cast<uint4*>(kb + h * kQ8HeadBytes + (64 * i + lane) * 16);
      uint4 o = make_uint4(0, 0, 0, 0);
      if (keep) {
        o = *at;
        o.x = rescaled<FMT>(o.x, by), o.y = rescaled<FMT>(o.y, by), o.z = rescaled<FMT>(o.z, by), o.w = rescaled<FMT>(o.w, by);
      }
      *at = o;
    }
  }
}

// Rows n0 .. n0 + 3 of a workgroup, those alone in their blocks: a wave each,
// heads 2 y and 2 y + 1, then 2 Y further on.
template <int FMT>
__device__ __forceinline__ void rows_alone(const RopeQ8Args& a, int around, int n0, int y, int Y, TurnLds* turns) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (2 * y >= a.hk || !is_alone(around, 16 + wave)) return;
  const int slot = __builtin_amdgcn_readlane(around, 16 + wave);
  put_turn(a, a.pos[n0 + wave], threadIdx.x & 63, &turns[wave]);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int kh = 2 * y; kh < a.hk; kh += 2 * Y) write_alone<FMT>(a, n0 + wave, slot, kh, turns[wave]);
}

// Row (or rows from) that workgroup x of 16 T looks at, LEADS of every 16: the T
// workgroups with the same rows of every 16 follow one another. In a prompt one
// row of 16 leads a block, and in row order all of those would be on one XCD.
template <int LEADS>
__device__ __forceinline__ int leads_from(const RopeQ8Args& a, int x) {
  const int T = (a.rows + 15) >> 4, s = x / T;
  return 16 * (x - s * T) + LEADS * s;
}

// Few rows, one launch. Workgroup (x, y) looks at four rows of 16. y below
// `alone`: those alone in their blocks, two K/V heads of them; the next hk: a K/V
// head of the other blocks that its rows lead; the rest: four of its rows' q heads.
// Six waves a SIMD (3 dwords spilled) against five: 1556 rows of 8 prompts 18.4 / 18.9 us,
// 64 rows each of its own sequence 4.3 / 4.3; with seven 19.9 / 4.8.
constexpr int kLeads = kThreads / 64;

template <int FMT>
__global__ __launch_bounds__(kThreads, 6) void rope_q8_rows(RopeQ8Args a, int alone) {
  const int n0 = leads_from<kLeads>(a, blockIdx.x), c = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int y = (int)blockIdx.y - alone;
  __shared__ __align__(16) TurnLds turns[kLeads];
  if (y < 0) {
    rows_alone<FMT>(a, slots_around(a, n0), n0, blockIdx.y, a.hk, turns);
    return;
  }
  float cs[8], sn[8], w[8];
  if (y >= a.hk) {
    const int n = n0 + (grp >> 2), head = 4 * (y - a.hk) + (grp & 3);
    const bool mine = n < a.rows && head < a.hq && a.slots[n] >= 0;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (mine) raw = ldg16(a.qkv + (int64_t)n * a.ld + (int64_t)head * kHead + 8 * c);
    put_turn(a, a.pos[min(n0 + (int)(threadIdx.x >> 6), a.rows - 1)], threadIdx.x & 63, &turns[threadIdx.x >> 6]);
    __syncthreads();
    if (!mine) return;
    get_turn(turns[grp >> 2], c, cs, sn);
    widen8(ldg16(a.q_norm + 8 * c), w);
    *reinterpret_cast<uint4*>(a.q + (int64_t)n * a.q_ld + (int64_t)head * kHead + 8 * c) = turn_head(a, raw, w, cs, sn);
    return;
  }
  const int kh = y, around = slots_around(a, n0);
  __shared__ KvLds lds;
  for (int lead = 0; lead < kLeads; ++lead) {
    BlockRows r;
    if (!block_rows(around, 16 + lead, n0 + lead, grp, &r)) continue;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (r.row >= 0) {
      const bf16_t* src = a.qkv + (int64_t)r.row * a.ld + (int64_t)(a.hq + kh) * kHead + 8 * c;
      const uint4 kraw = ldg16(src);
      v = ldg16(src + (int64_t)a.hk * kHead);
      turn_of(a, a.pos[r.row], c, cs, sn);
      widen8(ldg16(a.k_norm + 8 * c), w);
      k = turn_head(a, kraw, w, cs, sn);
      if (a.k) *reinterpret_cast<uint4*>(a.k + (int64_t)r.row * a.k_ld + (int64_t)kh * kHead + 8 * c) = k;
    }
    if (r.twice) k_rows_twice(a, r, n0 + lead, kh, a.hk, c, grp);
    write_block<FMT, 1>(a, r, kh, a.hk, &k, &v, c, grp, &lds);
  }
}

// Many rows, the cache: workgroup (x, y) looks at kLeads rows of 16, and for each
// that leads a block writes K/V heads y, y + Y, .. of it, a token per thread
// group, its angles computed once, kAtOnce heads at a time. In a prompt one row of
// 16 leads, and rows alone in their blocks are taken by a wave each afterwards.
// (With one row per workgroup, of 25,850 rows of 12 prompts the workgroups that
// end at once took some 50 us.) 25,850 rows of 32q/8kv (636 MB) take 122-128 us with
// turn_q_rows, 5.0-5.2 TB/s of reads and writes, where a large copy reaches 4.8-5.0;
// as integers 134.
constexpr int kAtOnce = 2;

template <int FMT>
__global__ __launch_bounds__(kThreads, 4) void rope_q8_blocks(RopeQ8Args a) {
  const int n0 = leads_from<kLeads>(a, blockIdx.x), c = threadIdx.x & 15, grp = threadIdx.x >> 4;
  const int y = blockIdx.y, Y = gridDim.y;
  const int around = slots_around(a, n0);
  __shared__ KvLds lds[kAtOnce];
  __shared__ __align__(16) TurnLds turns[kLeads];
  for (int lead = 0; lead < kLeads; ++lead) {
    const int n = n0 + lead;
    BlockRows r;
    if (!block_rows(around, 16 + lead, n, grp, &r)) continue;
    const bool mine = r.row >= 0;
    const bf16_t* src = a.qkv + (int64_t)(mine ? r.row : n) * a.ld + (int64_t)a.hq * kHead + 8 * c;
    uint4 kraw[kAtOnce], vraw[kAtOnce];
    const auto load = [&](int i, int kh) __attribute__((always_inline)) {
      kraw[i] = vraw[i] = make_uint4(0, 0, 0, 0);
      if (mine && kh < a.hk) {
        kraw[i] = ldg16_stream(src + (int64_t)kh * kHead);
        vraw[i] = ldg16_stream(src + (int64_t)(a.hk + kh) * kHead);
      }
    };
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) load(i, y + i * Y);
    float cs[8], sn[8], w[8];
    if (mine) {
      turn_of(a, a.pos[r.row], c, cs, sn);
      widen8(ldg16(a.k_norm + 8 * c), w);
    }
    for (int kh = y; kh < a.hk; kh += kAtOnce * Y) {
      uint4 k[kAtOnce], v[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        k[i] = make_uint4(0, 0, 0, 0), v[i] = vraw[i];
        if (mine) k[i] = turn_head(a, kraw[i], w, cs, sn);
        load(i, kh + (kAtOnce + i) * Y);
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i)
        if (mine && a.k && kh + i * Y < a.hk)
          *reinterpret_cast<uint4*>(a.k + (int64_t)r.row * a.k_ld + (int64_t)(kh + i * Y) * kHead + 8 * c) = k[i];
      write_block<FMT, kAtOnce>(a, r, kh, Y, k, v, c, grp, lds);
    }
    if (r.twice) k_rows_twice(a, r, n, y, Y, c, grp);
  }
  rows_alone<FMT>(a, around, n0, y, Y, turns);
}

// Many rows, q: one workgroup per row (2, 4, 8 or 16 rows of at most 8, 4, 2 or 1
// heads), a head per thread group. Up to kAhead heads of a group are asked for
// before the rows' angles are computed, 64 of them a row, once, into LDS:
// turn_of's values, bit for bit.
__global__ __launch_bounds__(kThreads) void turn_q_rows(RopeQ8Args a, int rows_shift) {
  constexpr int kAhead = 4;
  const int c = threadIdx.x & 15, grp = threadIdx.x >> 4, per = 16 >> rows_shift;  // heads at a time
  const int n0 = blockIdx.x << rows_shift, row = n0 + grp / per, h0 = grp & (per - 1);
  const bf16_t* src = a.qkv + (int64_t)row * a.ld + 8 * c;
  bf16_t* dst = a.q + (int64_t)row * a.q_ld + 8 * c;
  uint4 raw[kAhead];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (row < a.rows && h0 + i * per < a.hq) raw[i] = ldg16_stream(src + (int64_t)(h0 + i * per) * kHead);
  __shared__ __align__(16) TurnLds s_turn[16];
  for (int t = threadIdx.x; t < (kHead / 2) << rows_shift; t += kThreads) {
    const int k = t / (kHead / 2);
    put_turn(a, a.pos[min(n0 + k, a.rows - 1)], t & (kHead / 2 - 1), &s_turn[k]);
  }
  __syncthreads();
  if (row >= a.rows || a.slots[row] < 0) return;
  float cs[8], sn[8], w[8];
  get_turn(s_turn[grp / per], c, cs, sn);
  widen8(ldg16(a.q_norm + 8 * c), w);
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (h0 + i * per < a.hq) *reinterpret_cast<uint4*>(dst + (int64_t)(h0 + i * per) * kHead) = turn_head(a, raw[i], w, cs, sn);
  for (int h = h0 + kAhead * per; h < a.hq; h += per)
    *reinterpret_cast<uint4*>(dst + (int64_t)h * kHead) = turn_head(a, ldg16_stream(src + (int64_t)h * kHead), w, cs, sn);
}

// ------------------------------------------------------------------- decode

constexpr int kMostGroup = 16;  // query heads per K/V head
constexpr int kTile = 32;       // keys per step: two blocks
constexpr int kCus = 256;       // workgroups go to the CUs in turn
constexpr int kIds = 64 / (kTile / kQ8Block);  // tiles whose blocks a wave looks up at once

constexpr int kDecodeWaves = kThreads / 64;
constexpr int kBlocksPerTile = kTile / kQ8Block;

// The row of workgroup index n, and its position. Where the workgroups are more than
// the GPU takes at once, long rows come first and every other round of rows (what
// fills the GPU once) runs backwards, so that a CU's rows add up to much the same:
// index n takes the t-th longest of its 256 rows, by lengths of 6 bits, ties in their
// order. Every wave finds it from the positions it would wait for anyway, by bits
// of the length that have more than t rows at or above them. us in the rows' order /
// so ordered: 64 rows of 200-2400 keys of 16q/8kv 37.1 / 32.4, of 500-5000 of 32q/8kv
// 76 / 66, 256 of 100-3000 145 / 130, 128 of 100-3000 of 32q/32kv 271 / 256; rows of one
// length pay for it, 128 of 1600 of 32q/32kv 265.1 / 266.1.
__device__ __forceinline__ int row_of(const DecodeQ8Args& a, int n, int rows, int* p) {
  if (a.per_round == 0) {
    *p = a.pos[n];
    return n;
  }
  const int first = n & ~255, R = min(256, rows - first), lane = threadIdx.x & 63;
  const int from = (n - first) / a.per_round * a.per_round, at = n - first - from;
  int t = from / a.per_round & 1 ? min(R, from + a.per_round) - 1 - at : n - first;
  int pos[4], key[4];  // of rows first + 64 c + lane
#pragma unroll
  for (int c = 0; c < 4; ++c) pos[c] = 64 * c + lane < R ? a.pos[first + 64 * c + lane] : -1;
#pragma unroll
  for (int c = 0; c < 4; ++c) key[c] = 64 * c + lane < R ? min(max(pos[c], 0) >> a.len_shift, 63) : -1;
  int k = 0, above = 0;
#pragma unroll
  for (int b = 5; b >= 0; --b) {
    const int tried = k | 1 << b;
    int count = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) count += __popcll(__ballot(key[c] >= tried));
    if (count > t)
      k = tried;
    else
      above = count;
  }
  t -= above;
  int row = n;
  *p = -1;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint64_t same = __ballot(key[c] == k);
    const int count = __popcll(same);
    if (t >= 0 && t < count) {
      const int before = __builtin_amdgcn_mbcnt_hi((uint32_t)(same >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)same, 0));
      const int l = __builtin_ctzll(__ballot(key[c] == k && before == t));
      row = first + 64 * c + l;
      *p = __builtin_amdgcn_readlane(pos[c], l);
    }
    t -= count;
  }
  return row;
}

// One workgroup per (split, K/V head, row); its waves take the split's 32-key
// tiles in turn, each with a running maximum, sum and O of its own, merged
// through LDS at the end. Lane l is column n = l % 16 (query head) and group
// g = l / 16 of the v_mfma_f32_16x16x32_bf16 operands:
//   S^T (16 keys x 16 heads), two of them: row 4 x + r of product j is token
//     8 (x % 2) + 4 j + r of the tile's block x / 2, so a lane ends with tokens
//     8 (g % 2) .. + 7 of block g / 2 for its head, in order, which is P^T's
//     operand as it stands: no data crosses lanes between the two products but
//     the maximum. K is loaded in whole lines of 128 bytes, eight lanes a key,
//     and columns n and n + 8 trade halves.
//   O^T (16 dims x 16 heads) += V^T . P^T: V lies [dim][token] in the cache. A
//     lane loads the 16 tokens of one dim (groups 2 b and 2 b + 1 two dims of
//     block b) and the two groups trade halves, which gives each its tokens of
//     both dims.
// P is carried as two bf16 terms (hi + lo, 16 bits): the matrix cores are a
// tenth of the time. Both scales act per block, that is per lane: on the scores
// and, an exact power of two, on P.
// The cache's bytes bound it, each read once and kept in no cache (whole lines of K
// past the caches / as 64-byte halves / cached: 128 rows of 1600 keys of 32 heads 264 /
// 269 / 266 us, 4 of 100,000-130,000 of 32q/8kv 162 / 170 / 168). 128 rows of 100-3000
// keys of 32 heads (1.63 GB) take 247 us, 6.6 TB/s (255 on another card); the 4 long
// rows in 4096-key splits (0.94 GB) 153 with the merge, 6.1; 64 of 200-2400 of 16q/8kv
// (0.17 GB) 30.5, 5.6, where the longest rows' walks show. Loads alone, nothing
// computed, took 265 of 272 us on the 128 rows of 1600; 64-key tiles, two or three
// tiles asked for ahead, and two or three workgroups a CU in place of four were no
// faster. A lone row is bound by latency: 1 row of 8000 keys in 256-key splits takes
// 10.8 with the merge. Under a plan far longer than its rows the splits are the
// plan's: the 64 rows take 52 under one for 40,960 keys.
template <int FMT>
__global__ __launch_bounds__(kThreads, 4) void decode_q8(DecodeQ8Args a) {
  const int kh = blockIdx.y, G = a.hq / a.hk, tid = threadIdx.x;
  const int split = spread_split(blockIdx.x, kh + a.hk * blockIdx.z, a.splits);
  int p;
  const int n = row_of(a, blockIdx.z, gridDim.z, &p);
  const int32_t* pg = a.pages + a.indptr[!a.ragged ? n : p < 0 ? 0 : max(a.seq[n], 0)];  // no keys: any sequence may stand there
  const int len = p < 0 ? 0 : p + 1;
  const int64_t h0 = (int64_t)n * a.hq + kh * G;
  if (len == 0) {
    if (split == 0)
      for (int i = tid; i < G * kHead; i += kThreads) a.out[h0 * kHead + i] = 0;
    return;
  }
  const int split_len = split_len_of(a.chunk, a.splits, len);
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
    const uint8_t* kb = a.kv + kh * kQ8HeadBytes + (2 * (col & 4) + (col & 3)) * kHead + 16 * grp + 8 * (col & 8);
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const int64_t block = __builtin_amdgcn_readlane(ids, 2 * (k & (kIds - 1)) + b);
#pragma unroll
      for (int j = 0; j < 2; ++j) kr[j][b] = ldg16_stream(kb + block * row_blocks * kQ8HeadBytes + 4 * j * kHead);
    }
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
      trade_halves(kr[j][0], kr[j][1]);
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
    // The base is set 8 (log2) above the maximum and moves when one passes it: it
    // seldom moves, and p <= 1, so p V is no larger than V.
    const bool grow = mx > m;
    if (__any(grow)) {
      const float to = mx + 8.f, alpha = grow ? fast_exp2(m - to) : 1.f;
      m = grow ? to : m;
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
  const int split_len = split_len_of(a.chunk, a.splits, len);
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

// One launch below this many heads over all rows, two from there (us in one / in two):
// prompts of 2700 rows of 32q/8kv (130,000 heads) 28.5 / 30.3, of 3300 34.0 / 30.9; 4000 of
// 16q/8kv (128,000) 29.3 / 30.4; 1000 of 32q/32kv (96,000) 25.7 / 25.3, 1300 31.7 / 28.1;
// 20,000 of 8q/1kv (200,000) 39.1 / 39.4; rows of as many sequences, 1900 of 32q/8kv
// (91,000) 30.8 / 32.6, 3000 47.6 / 44.2.
constexpr int64_t kManyHeads = 1 << 17;

int launch_rope_q8(const RopeQ8Args& a, hipStream_t stream) {
  const unsigned T = (unsigned)(((int64_t)a.rows + 15) / 16);
  if ((int64_t)a.rows * (a.hq + 2 * (int64_t)a.hk) < kManyHeads) {
    const int alone = (a.hk + 1) / 2;
    const dim3 grid(16 / kLeads * T, alone + a.hk + (a.hq + 3) / 4);
    if (!grid_holds(grid.x, kThreads, grid.y)) return -2;
    if (a.format == kQ8E4m3)
      rope_q8_rows<kQ8E4m3><<<grid, kThreads, 0, stream>>>(a, alone);
    else
      rope_q8_rows<kQ8Int8><<<grid, kThreads, 0, stream>>>(a, alone);
    return check_launch();
  }
  // The K/V heads of a block over as many workgroups as give a prompt 1024 that lead.
  const dim3 grid(16 / kLeads * T, std::min<unsigned>(a.hk, (1024 + T - 1) / T));
  int shift = 0;
  while (shift < 4 && (16 >> (shift + 1)) >= a.hq) ++shift;
  const int64_t q_groups = ((int64_t)a.rows + (1 << shift) - 1) >> shift;
  if (!grid_holds(grid.x, kThreads) || !grid_holds(q_groups, kThreads)) return -2;
  if (a.format == kQ8E4m3)
    rope_q8_blocks<kQ8E4m3><<<grid, kThreads, 0, stream>>>(a);
  else
    rope_q8_blocks<kQ8Int8><<<grid, kThreads, 0, stream>>>(a);
  if (check_launch() != 0) return -3;
  turn_q_rows<<<dim3((unsigned)q_groups), kThreads, 0, stream>>>(a, shift);
  return check_launch();
}

int launch_decode_q8(DecodeQ8Args a, int rows, hipStream_t stream) {
  // Splits even the rows out themselves (21 rows of 512-5120 keys of 32q/8kv in 512-key
  // splits 28.5 us, 31 so ordered).
  a.per_round = a.splits == 1 && (int64_t)rows * a.hk > kCus ? std::max(kCus / a.hk, 1) : 0;
  while (a.chunk >> a.len_shift >= 64) ++a.len_shift;
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
