// What the attention kernels of the 8-bit block cache share (block_rows.hip, block_tile.hip): arguments, work items,
// the division of an item's positions into splits, and query rows in operand order.
#pragma once

#include "block_common.h"

namespace kvt {
namespace blk {

constexpr float kLag = 4.0f;     // a row's running maximum moves when a tile exceeds it by more (powers of two)
constexpr float kLift = 10.0f;   // weights are held times 2^10: P = 2^(x - m + 10), at most 2^14, in fp16

struct Attn {
  const void* q;               // [rows, Hq, D]
  const uint8_t* k8;
  const uint8_t* v8;
  const float* ks;
  const float* vs;
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* rows;         // table row of a request (NULL: its number)
  const int32_t* cu;           // NULL: one query per request
  void* out;
  float* part_o;
  float* part_ml;
  int32_t* counters;           // of the items whose splits the launch merges itself (NULL: a launch of its own does)
  int64_t sq_n, sq_h, so_n, so_h, stride;
  float scale_log2;
  int n, n_rows, n_q, H, gs, n_blocks, max_blocks, log2b, splits, causal;
  int item_rows;               // rows of a work item
  int tile, least;             // positions of a tile; the tiles of a split are a multiple of this
  int single;                  // query tiles over one request: (item, KV head) pairs of the launch (else 0)
  int shares, shift;           // decode in equal shares (0: in splits): workgroups; steps of their line are 2^shift tiles
};

// What a workgroup has: request r, query rows [row0, row0 + n_row) of it in (query, q head) order, the query base, and
// the positions that any of its rows sees.
struct Item {
  int r, trow, q0, q_len, row0, n_row, kv, len, limit;
};

// Positions that query qi of the item's request sees.
KVT_DEV int sees(const Attn& P, const Item& t, int qi) {
  return P.causal ? min(t.len, max(t.kv - t.q_len + qi + 1, 0)) : t.len;
}

KVT_DEV Item item_of(const Attn& P, int w) {
  Item t;
  if (P.cu == nullptr) {
    t.r = w, t.q0 = w, t.q_len = 1, t.row0 = 0, t.n_row = P.gs;
  } else {
    t.r = find_request(P.cu, P.n, w, P.gs, P.item_rows, 1);
    const int cu0 = uniform(P.cu[t.r]);
    t.q0 = min(max(cu0, 0), P.n_q);
    t.q_len = min(max(uniform(P.cu[t.r + 1]), t.q0), P.n_q) - t.q0;
    const int64_t row0 = (w - first_item(cu0, t.r, P.gs, P.item_rows, 1)) * P.item_rows;
    const int64_t left = (int64_t)t.q_len * P.gs - row0;
    t.row0 = (int)row0;
    t.n_row = row0 < 0 || left <= 0 ? 0 : (int)min(left, (int64_t)P.item_rows);
  }
  t.trow = P.rows ? uniform(P.rows[t.r]) : t.r;
  t.kv = max(uniform(P.kv_lens[t.r]), 0);
  t.len = (int)min((int64_t)t.kv, (int64_t)P.max_blocks << P.log2b);
  if (t.trow < 0 || t.trow >= P.n_rows) t.len = 0, t.trow = 0;
  t.limit = t.n_row > 0 ? sees(P, t, (t.row0 + t.n_row - 1) / P.gs) : 0;
  return t;
}

// Tiles per split of an item whose rows see `limit` positions.  Splits behind the last tile are empty.  The number of
// splits follows from the table's width, which a short request does not fill, so what a split has at least follows from
// what the rows see: a multiple of `least` tiles, or for query tiles over one request 512 positions, 256 where those
// splits would leave half of the CUs idle (as _TILE_LEAST of block_kv.py has it, where both are measured).  In a table
// of 262,144 positions, us per call, splits of a tile or two / so many: 272 queries behind 3,156 positions (16 / 2
// heads, D 256) 65 / 48, a prompt of 512 36.6 / 33.8, 61 queries behind 1,697 (12 / 1, D 128) 21.6 / 22.5.
KVT_DEV int tiles_of(const Attn& P, int limit) { return (limit + P.tile - 1) / P.tile; }
KVT_DEV int tiles_per_split(const Attn& P, int limit) {
  const int per = (tiles_of(P, limit) + P.splits - 1) / P.splits;
  if (P.single) return max(per, ((int64_t)P.single * ((limit + 511) >> 9) >= 128 ? 512 : 256) / P.tile);
  return max((per + P.least - 1) / P.least, 1) * P.least;
}
// Splits that have tiles (one where there are none: it writes the NaN).  An item of one split is not merged.
KVT_DEV int splits_used(const Attn& P, int limit) {
  const int tps = tiles_per_split(P, limit);
  return P.splits == 1 ? 1 : max((tiles_of(P, limit) + tps - 1) / tps, 1);
}

// fp32 pair -> fp16, to nearest even (one v_cvt_pk_f16_f32)
KVT_DEV h2 h2_rne(float a, float b) { return __builtin_convertvector((f2){a, b}, h2); }

KVT_DEV float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }   // (v_exp_f32: results below 2^-126 are 0)
KVT_DEV float bits_f(uint32_t u) { return __uint_as_float(u); }

// A row that sees a position of a block with a scale that is not finite is NaN, in every channel; to other rows such a
// block is one that is not there, so that no 0 * NaN of a position that they do not see reaches them.  (Scales are >=
// 0.)
KVT_DEV bool finite_scales(float k, float v) { return max(__float_as_uint(k) << 1, __float_as_uint(v) << 1) < 0xFF000000u; }

// NaN codes of V (e4m3) in tiles that some row of a workgroup does not see to their end: a product would take them to
// all of its rows, as 0 * NaN.  They are taken out of the codes, and what remains is the first position where each
// channel has one: a row sees positions 0 .. n - 1, so the channel is NaN for it where that position is below n.
template <int CODE, int D>
struct NanAt {
  int at[CODE == kE4M3 ? D : 1], found;
  KVT_DEV void clear() {                        // (every thread of a workgroup, and a barrier before the first take)
    for (int i = threadIdx.x; i < D; i += 256) at[i] = 0x7FFFFFFF;
    if (threadIdx.x == 0) found = 0;
  }
  KVT_DEV bool any() const { return found != 0; }
  // N dwords of codes: dword i has channels ch + step i .. + 3 of position pos(i).
  template <int N, class Pos>
  KVT_DEV void take(uint32_t (&w)[N], Pos pos, int ch, int step = 0) {
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) any |= (w[i] & 0x7F7F7F7Fu) + 0x01010101u;
    if (!(any & 0x80808080u)) return;
    found = 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t nan = ((w[i] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
#pragma unroll 1
      for (int c = 0; c < 4; ++c)
        if (nan >> (8 * c + 7) & 1) atomicMin(&at[ch + step * i + c], pos(i));
      w[i] &= ~((nan >> 7) * 0xFFu);
    }
  }
  // Converted codes of channels ch .. + 3 in LDS, rows of `pitch` bytes: positions pos .. + 3, + 8 .. + 11.
  KVT_DEV void take_f16(uint8_t* p, int pitch, int pos, int ch) {
    found = 1;
#pragma unroll 1
    for (int k = 0; k < 32; ++k) {
      uint16_t* x = reinterpret_cast<uint16_t*>(p + (k >> 3) * pitch) + (k & 7);
      if ((*x & 0x7FFF) > 0x7C00) {
        atomicMin(&at[ch + (k >> 3)], pos + (k & 7) + (k & 4));
        *x = 0;
      }
    }
  }
};

// O's unit becomes the V scale fv > 0, but no less than 2^-80 of the largest so far (|O| in units of that is below
// 2^40, so it stays finite); returns the factor for O.
KVT_DEV float new_unit(float fv, float& unit, float& peak) {
  peak = fmaxf(peak, fv);
  const float u = fmaxf(fv, peak * 0x1p-80f), a = unit / u;
  unit = u;
  return a;
}

// Four consecutive channels of an output row (rows are 16-byte aligned: the entry points see to it).
KVT_DEV void store_out4(void* out, int ot, int64_t at, float a, float b, float c, float d) {
  if (ot == kF32) {
    *reinterpret_cast<float4*>((float*)out + at) = make_float4(a, b, c, d);
  } else if (ot == kBF16) {
    *reinterpret_cast<uint2*>((uint16_t*)out + at) = make_uint2(bf16x2(a, b), bf16x2(c, d));
  } else {
    const h2 x = h2_rne(a, b), y = h2_rne(c, d);
    *reinterpret_cast<uint2*>((uint16_t*)out + at) = make_uint2(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y));
  }
}

// Eight elements of a query row each at at(k), k < N -> operands.  bf16 rows are scaled by a power of two to fit fp16;
// returns its inverse.  top_of reduces a lane's largest |q| over the lanes that share its row.
template <int QT, int N, class At, class Top>
KVT_DEV float load_q(const void* q, int64_t row, At at, Top top_of, h8 (&out)[N]) {
  uint4 raw[N];
#pragma unroll
  for (int k = 0; k < N; ++k)
    raw[k] = *reinterpret_cast<const uint4*>((const uint16_t*)q + row + at(k));
  if constexpr (QT == kF16) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      asm("" : "+v"(raw[k].x), "+v"(raw[k].y), "+v"(raw[k].z), "+v"(raw[k].w));   // (loaded tuples cost spills)
      out[k] = __builtin_bit_cast(h8, raw[k]);
    }
    return 1.0f;
  } else {
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(bits_f(w[i] << 16)), fabsf(bits_f(w[i] & 0xFFFF0000u))));
    }
    top = top_of(top);
    int e = (int)(__float_as_uint(top) >> 23) - 127;
    e = top > 0.0f && top < __builtin_inff() ? min(max(e, -120), 120) : 0;
    const float f = bits_f((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const uint32_t w[4] = {raw[k].x, raw[k].y, raw[k].z, raw[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        out[k][2 * i] = (_Float16)(bits_f(w[i] << 16) * f);
        out[k][2 * i + 1] = (_Float16)(bits_f(w[i] & 0xFFFF0000u) * f);
      }
    }
    return bits_f((uint32_t)(127 + e) << 23);
  }
}

// Launch of the query-tile kernel (block_tile.hip): one workgroup per (kTileRows rows, KV head, split).
constexpr int kTileRows = 128;
int tile_positions(int D);
void tile_launch(const Attn& P, int code, int qt, int D, int items, int ot, hipStream_t st);

}  // namespace blk
}  // namespace kvt
