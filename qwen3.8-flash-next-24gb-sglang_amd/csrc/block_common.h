// Device helpers of the 8-bit block cache (block_plan.hip, block_store.hip, block_rows.hip, block_tile.hip).
//
// Layout, per layer: codes k8 / v8 [n_blocks, H, B, D], one byte each (e4m3 or int8), B = 16, 32 or 64 tokens; scales
// ks / vs fp32 [n_blocks, H]: the value of a code c is c * s.  A request's position p sits in row p % B of block
// block_table[row][p / B].  The write path stores powers of two as scales, so code * s and x / s are exact and the
// codes of an e4m3 block survive a growing scale unrounded (down to the subnormals); the readers take any scale.
#pragma once

#include "kvt_common.h"

namespace kvt {
namespace blk {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2v __attribute__((ext_vector_type(2)));
typedef uint32_t u4v __attribute__((ext_vector_type(4)));

enum Code : int { kE4M3 = 0, kI8 = 1 };
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxReq = 4096;          // requests of one call (the search below takes two rounds of 64)

// A value that every lane has, in a scalar register (what a uniform address loads is not taken for one by itself).
KVT_DEV int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
KVT_DEV float uniform(float v) { return __uint_as_float((uint32_t)__builtin_amdgcn_readfirstlane((int)__float_as_uint(v))); }

// The smallest power of two s with a / s <= qmax (both codes' qmax = t * 2^p, t in [1, 2)), within 2^-64 .. 2^122.
template <int CODE>
KVT_DEV float pow2_scale(float a) {
  constexpr uint32_t top = CODE == kE4M3 ? 0x600000u : 0x7E0000u;   // fraction bits of 448 = 1.75 * 2^8, 127 = 1.984375 * 2^6
  constexpr int p = CODE == kE4M3 ? 8 : 6;
  const uint32_t b = __float_as_uint(a);
  int e = (int)(b >> 23) - 127 - p + ((b & 0x7FFFFFu) > top ? 1 : 0);
  e = min(max(e, -64), 122);
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// Two fp32 values -> two codes in the low half of a dword.  |x| beyond the codes' range saturates; NaN stays NaN in
// e4m3 and becomes 0 in int8.
KVT_DEV float sat(float x, float top) { return fabsf(x) > top ? copysignf(top, x) : x; }
KVT_DEV uint32_t i8_code(float x) {
  const float r = rintf(sat(x, 127.0f));
  return (uint32_t)(r == r ? (int)r : 0) & 0xFFu;
}
template <int CODE>
KVT_DEV uint32_t pack4(float a, float b, float c, float d) {
  if constexpr (CODE == kE4M3) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(sat(a, 448.0f), sat(b, 448.0f), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(sat(c, 448.0f), sat(d, 448.0f), w, true);
  } else {
    return i8_code(a) | (i8_code(b) << 8) | (i8_code(c) << 16) | (i8_code(d) << 24);
  }
}
template <int CODE>
KVT_DEV void unpack4(uint32_t w, float (&x)[4]) {
  if constexpr (CODE == kE4M3) {
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    x[0] = lo.x, x[1] = lo.y, x[2] = hi.x, x[3] = hi.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)(int8_t)(w >> (8 * i));
  }
}

KVT_DEV h2 as_h2(uint32_t u) { return __builtin_bit_cast(h2, u); }

// Two codes (bytes 0, 1 or 2, 3 of a dword) -> fp16, exact.  e4m3: one conversion.  int8: the byte c + 128 as the low
// byte of 1024 + u, minus 1152 (the caller has flipped the sign bits: flip()).
template <int CODE>
KVT_DEV uint32_t flip(uint32_t w) { return CODE == kI8 ? w ^ 0x80808080u : w; }
template <int CODE, bool HI>
KVT_DEV h2 pair(uint32_t w) {
  if constexpr (CODE == kE4M3) {
    return __builtin_bit_cast(h2, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HI));
  } else {
    const h2 off = {(_Float16)-1152.0f, (_Float16)-1152.0f};
    return as_h2(__builtin_amdgcn_perm(0x64646464u, w, HI ? 0x04030402u : 0x04010400u)) + off;
  }
}
// Eight codes of two dwords in order -> one matrix operand.
template <int CODE>
KVT_DEV h8 operand(uint32_t w0, uint32_t w1) {
  w0 = flip<CODE>(w0), w1 = flip<CODE>(w1);
  const h2 a = pair<CODE, false>(w0), b = pair<CODE, true>(w0), c = pair<CODE, false>(w1), d = pair<CODE, true>(w1);
  return h8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The work items of request r are numbered from first_item(cu[r], r) = floor(cu[r] * mul / div) + per * r on: an upper
// bound of what the requests before it need, so that a launch finds (request, item) from its block index and the prefix
// sums alone, with no list of items.  find_request returns the largest r < n with first_item(r) <= w (0 if none), for n
// <= 4,096: two rounds of one load per lane.  All 64 lanes take part; the result is uniform.
KVT_DEV int64_t first_item(int cu, int r, int mul, int div, int per) {
  return (int64_t)max(cu, 0) * mul / div + (int64_t)per * r;
}
KVT_DEV int find_request(const int32_t* cu, int n, int64_t w, int mul, int div, int per) {
  const int lane = threadIdx.x & 63;
  const int step = (n + 63) >> 6;
  int r = lane * step;
  int below = __popcll(__ballot(r < n && first_item(cu[min(r, n - 1)], r, mul, div, per) <= w));
  int lo = max(below - 1, 0) * step;
  if (step > 1) {
    r = lo + lane;
    below = __popcll(__ballot(lane < step && r < n && first_item(cu[min(r, n - 1)], r, mul, div, per) <= w));
    lo += max(below - 1, 0);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace blk
}  // namespace kvt
