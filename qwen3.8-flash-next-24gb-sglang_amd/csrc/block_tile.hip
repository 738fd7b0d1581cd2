// Attention of query chunks over the 8-bit block cache on the matrix cores: the kernel of calls with many rows
// (kvt_block_prefill; block_rows.hip has the mathematics and the calls with few rows).
//
// A row is a (query, q head) pair of one KV head, in that order; one workgroup of 4 wavefronts has 128 of them (32 per
// wavefront) and walks the positions that they see in tiles of T.  The 256 threads convert a tile's codes to fp16 once,
// into LDS, and the four wavefronts multiply from there:
//   S^T = K Q^T on v_mfma_f32_32x32x16_f16 (A = 32 positions from LDS, B = the wavefront's 32 rows in registers).  A
//     lane gets 16 scores of one row, the other 16 of the tile's 32 sit in lane ^ 32: the row maximum takes one
//     cross-lane step.
//   O^T += V^T P^T: the weights stay where they are (register 8 s + j of lane (l, g) is position 16 s + 8 (j / 4) + 4 g
//     + j % 4, its operand's k), and V^T is stored so that these eight positions of a channel are 16 consecutive bytes.
//     Each product covers 16 positions, i.e. one block of the cache, so a block's V scale is one factor for the whole
//     operand.
// Two LDS buffers: a tile's codes are loaded into registers before the products of the tile before, converted and
// stored behind them; one barrier per tile.  Positions' block ids are loaded a tile ahead of the codes.  LDS rows are
// padded by 16 bytes (V^T at D = 256: 16-byte pieces in an order that depends on the channel), which spreads the
// operand reads (16 bytes per lane, 32 consecutive rows) over the banks.  T = 32 positions at D = 256, 64 below: 32 KB
// of fp16 per buffer, so that two workgroups (D = 64: three, 16 KB) fit a CU, whose wavefronts run their softmax under
// each other's products.
//
// Matrix and vector instructions bound it together: causal prompts of 10,001 tokens, 16 / 2 heads, D 256, e4m3 875 us,
// 936 TFLOP/s (a large library product 1,192): the matrix pipes are busy 42 % of the cycles, 7 vector instructions
// stand beside each matrix instruction, a third of the wavefronts' time is waiting (barrier, LDS); 8,192 tokens, 32 / 8
// heads, D 128 620 us, 887 TFLOP/s; 16 / 16, D 64 210 us, 656 TFLOP/s; int8 codes take 2 - 5 % longer.  At D 256 the
// kernels have 252 - 254 of 256 registers, and none is spilled.
#include "block_attn.h"

using namespace kvt;
using namespace kvt::blk;

namespace {

typedef float f16v __attribute__((ext_vector_type(16)));

KVT_DEV f16v mfma(h8 a, h8 b, f16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

KVT_DEV float max_xor32(float v) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(bits_f(b[0]), bits_f(b[1]));
}
KVT_DEV float sum_xor32(float v) {
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return bits_f(b[0]) + bits_f(b[1]);
}

constexpr int kDsRead = 0x100, kMfma = 0x8;   // instruction classes of the scheduling hints
constexpr float kLeast = 0x1p-120f;   // (a factor of 0 would make a masked score, -inf, a NaN)

// The largest of three (one v_maximum3_f32; fmaxf of a matrix product's result costs a canonicalizing v_max_f32 x, x
// each).  Not as asm: the compiler sees no asm read the result of a matrix product, and puts no wait before it.
KVT_DEV float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
// v, where the compiler does not know it: what follows from it is computed here, not kept in registers from further up.
KVT_DEV int again(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

template <int D>
struct Tile {
  static constexpr int T = D == 256 ? 32 : 64;
  static constexpr int KP = 2 * D + 16;         // bytes per K row (a position)
  // V^T rows (a channel each): 16-byte pieces in an order that depends on the channel, where T = 32 (the padding would
  // not leave room for what D = 256 keeps of Q in LDS), else padded
  static constexpr int VP = T == 32 ? 64 : 2 * T + 16;
  static KVT_DEV int piece(int channel, int i) { return T == 32 ? i ^ (channel >> 2 & 3) : i; }
  static constexpr int QL = D == 256 ? 3 : 0;   // operands of Q that are kept in LDS: the registers hold no more than 13
  static constexpr int TPK = 256 / T;           // threads per K row
  static constexpr int NK = D / 16 / TPK;       // 16-byte pieces of a K row per thread
};

template <int D>
struct __align__(16) Buf {
  uint8_t k[Tile<D>::T * Tile<D>::KP];
  uint8_t v[D * Tile<D>::VP];
  // of K in the two halves of 32 positions (-1: no such block, NaN: one with a scale that is not finite), and of V
  float scale[Tile<D>::T / 32][4];
};

// A thread's share of a tile as loaded: pieces of one K row, and 4 channels of 8 positions of V.
template <int D>
struct RawK {
  u4v c[Tile<D>::NK];
};
struct RawV {
  uint32_t c[8];
  float ks, vs;
};

template <int CODE, int QT, int D>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void block_tile_kernel(const Attn P, int items, int ot) {
  using C = Tile<D>;
  constexpr int T = C::T, SUB = T / 32, DT = D / 32;
  constexpr int kAhead = D == 256 ? 2 : 4;     // operands read ahead of their product (what the registers hold)
  __shared__ Buf<D> buf[2];
  __shared__ h8 qlds[C::QL ? C::QL : 1][256];
  __shared__ NanAt<CODE, D> nans;
  const int tid = threadIdx.x, lane = tid & 63, l = lane & 31, g = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // head fastest: with H = 2, 4 or 8 the workgroups of a head share the caches of the same XCDs; the last rows, which
  // see the most positions, first
  const int h = blockIdx.x % P.H, w = items - 1 - (int)(blockIdx.x / P.H), split = blockIdx.y;
  const Item it = item_of(P, w);
  if (it.n_row == 0) return;
  const int tps = tiles_per_split(P, it.limit);
  const int tile0 = split * tps, tile1 = min(tile0 + tps, tiles_of(P, it.limit));
  const int used = splits_used(P, it.limit);
  if (split >= used) return;

  const int fewest = uniform(sees(P, it, it.row0 / P.gs));             // positions that every row of the workgroup sees
  if (CODE == kE4M3) {                         // (the first tile is searched for NaN codes only if it ends behind those)
    nans.clear();
    if (tile0 * T + T > fewest) __syncthreads();
  }
  const int my = it.row0 + 32 * wave + l;
  const bool live = 32 * wave + l < it.n_row;
  constexpr int QR = D / 16 - C::QL;
  h8 Q[D / 16];
  // (rows behind the item's last compute what its first does; nothing is stored of them)
  const int lq = live ? my : it.row0;
  const float qf = load_q<QT>(P.q, (int64_t)(it.q0 + lq / P.gs) * P.sq_n + (int64_t)(h * P.gs + lq % P.gs) * P.sq_h,
                              [g](int k) { return 16 * k + 8 * g; }, max_xor32, Q) * P.scale_log2;
#pragma unroll
  for (int k = 0; k < C::QL; ++k) qlds[k][tid] = Q[QR + k];          // (each lane its own: no barrier)
  const int see = live ? sees(P, it, my / P.gs) : 0;
  const int first_row = it.row0 + 32 * wave, last_row = it.row0 + min(32 * wave + 31, it.n_row - 1);
  const bool any_row = 32 * wave < it.n_row;
  const int all_see = uniform(any_row ? sees(P, it, first_row / P.gs) : 0);   // positions that every row of the wavefront sees
  const int most_see = uniform(any_row ? sees(P, it, last_row / P.gs) : 0);   // and that any of them sees

  // This thread's share of a tile: 16-byte pieces tid % TPK, + TPK, .. of K row tid / TPK; channels vd .. vd + 3 of V
  // rows vrow + {0 .. 3, 8 .. 11}.  A wavefront's rows all lie in the 16 positions `sub` of the tile, i.e. in one
  // block: its id and the addresses' bases are uniform.
  const int sub = T == 32 ? wave >> 1 : wave;
  const int vc = 2 * sub + (lane & 1), vd = 4 * ((lane >> 1) + (T == 32 ? 32 * (wave & 1) : 0));
  const int vrow = 16 * sub + 4 * (lane & 1);
  const bool has_v = vd < D;
  const int32_t* table = P.table + it.trow * P.stride;
  const int bmask = (1 << P.log2b) - 1;
  const int64_t head = (int64_t)h * (D << P.log2b);
  const uint32_t block_bytes = (uint32_t)P.H * (D << P.log2b);        // (of one block: < 2^32, the entry point sees to it)

  // At D = 256 the registers hold only one side of the next tile at a time: K's codes under the first product, V's
  // under the second, and addresses are computed where they are used.
  constexpr bool kApart = D == 256;
  // At D = 64 both halves of a tile are multiplied with Q before the first one's softmax, under which the second
  // product runs (8,192 tokens, 16 heads: 249 -> 220 us, 624 TFLOP/s; at D = 128, whose products are twice as long, 641
  // -> 646).
  constexpr bool kBoth = D == 64;

  // (no branch around a load: the wait for it would move to where the paths join)
  const auto id_at = [&](int tile) { return table[min(tile * T + 16 * sub, it.limit - 1) >> P.log2b]; };
  const auto in_pool = [&](int id) { return (uint32_t)id < (uint32_t)P.n_blocks; };
  const auto offset = [&](int id, int tile) {   // of the wavefront's 16 positions
    return (uint64_t)(in_pool(id) ? (uint32_t)id : 0u) * block_bytes + (uint32_t)((tile * T + 16 * sub) & bmask) * D;
  };
  const auto fetch_k = [&](int tile, int id, RawK<D>& r) {
    const uint8_t* p = P.k8 + head + offset(id, tile);
    const int t = kApart ? again(tid) : tid;
    const uint32_t koff = (uint32_t)(t / C::TPK & 15) * D + 16 * (t % C::TPK);
#pragma unroll
    for (int i = 0; i < C::NK; ++i) r.c[i] = *reinterpret_cast<const u4v*>(p + (koff + 16 * C::TPK * i));
  };
  const auto fetch_v = [&](int tile, int id, RawV& r) {
    const uint8_t* p = P.v8 + head + offset(id, tile);
    const uint32_t voff = 4u * (lane & 1) * D + (has_v ? vd : 0);
#pragma unroll
    for (int i = 0; i < 8; ++i) r.c[i] = *reinterpret_cast<const uint32_t*>(p + (voff + (i + (i & 4)) * D));
    const uint32_t at = (in_pool(id) ? (uint32_t)id : 0u) * (uint32_t)P.H + h;   // (< 2^32: a block and head is 1 KiB at least)
    r.ks = P.ks[at], r.vs = P.vs[at];
  };
  const auto convert_k = [&](const RawK<D>& r, Buf<D>& b) {
    const int t = kApart ? again(tid) : tid;
    uint8_t* kr = b.k + t / C::TPK * C::KP + 32 * (t % C::TPK);
#pragma unroll
    for (int i = 0; i < C::NK; ++i) {
      h8* to = reinterpret_cast<h8*>(kr + 32 * C::TPK * i);
      to[0] = operand<CODE>(r.c[i].x, r.c[i].y);
      to[1] = operand<CODE>(r.c[i].z, r.c[i].w);
    }
  };
  // NaN codes of V in a tile that some row does not see to its end (this thread's share, read back from LDS).
  const auto nans_of = [&](int tile, Buf<D>& b) {
    const int lz = again(lane), d = 4 * ((lz >> 1) + (T == 32 ? 32 * (wave & 1) : 0));
    uint8_t* p = b.v + d * C::VP + 16 * C::piece(d, 2 * sub + (lz & 1));
    uint32_t any = 0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const u4v w = *reinterpret_cast<u4v*>(p + c * C::VP);
#pragma unroll
      for (int i = 0; i < 4; ++i) any |= (w[i] & 0x7FFF7FFFu) + 0x03FF03FFu;
    }
    if (any & 0x80008000u) nans.take_f16(p, C::VP, tile * T + 16 * sub + 4 * (lz & 1), d);
  };
  const auto convert_v = [&](int tile, int id, RawV& r, Buf<D>& b, bool checked) {
    const bool fin = finite_scales(r.ks, r.vs), ok = in_pool(id) && fin;
    if ((T == 64 || !(wave & 1)) && lane == 0) {
      float* to = b.scale[sub >> 1] + (sub & 1);
      to[0] = ok ? r.ks : in_pool(id) ? __builtin_nanf("") : -1.0f;
      to[2] = ok ? r.vs : 0.0f;
    }
    if (!has_v) return;
    const int left = ok ? it.limit - (tile * T + 16 * sub) : 0;   // positions behind the last one, or in no block: 0
    if (left < 16) {
      const int mine = left - (vrow & 15);
#pragma unroll
      for (int i = 0; i < 8; ++i) r.c[i] = i + (i & 4) < mine ? r.c[i] : 0u;
    }
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t a = flip<CODE>(r.c[2 * j]), c = flip<CODE>(r.c[2 * j + 1]);
      lo[j] = __builtin_amdgcn_perm(c, a, 0x05010400u);
      hi[j] = __builtin_amdgcn_perm(c, a, 0x07030602u);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      h2 y[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = c < 2 ? lo[j] : hi[j];
        y[j] = c & 1 ? pair<CODE, true>(u) : pair<CODE, false>(u);
      }
      *reinterpret_cast<h8*>(b.v + (vd + c) * C::VP + 16 * C::piece(vd, vc)) =
          h8{y[0].x, y[0].y, y[1].x, y[1].y, y[2].x, y[2].y, y[3].x, y[3].y};
    }
    if (checked) nans_of(tile, b);
  };

  f16v acc[DT];
#pragma unroll
  for (int c = 0; c < DT; ++c) acc[c] = f16v{};
  float m = -__builtin_inff(), lift = 0x1p120f, sum = 0.0f, part = 0.0f;   // (part: of the sum, in units of ru)
  float unit = 0.0f, peak = 0.0f, ru = 0.0f, log_ru = 0.0f, per_ru = 1.0f;   // uniform, as the next two
  int last = -1, lost = 0;
  int poison = 0x7FFFFFFF;                       // the first position whose block has a scale that is not finite (uniform)

  if (tile0 < tile1) {
    RawK<D> rk;
    RawV rv;
    int id = uniform(id_at(tile0));
    fetch_k(tile0, id, rk);
    fetch_v(tile0, id, rv);
    convert_k(rk, buf[0]);
    convert_v(tile0, id, rv, buf[0], CODE == kE4M3 && tile0 * T + T > fewest);
    int then = id_at(tile0 + 1);
    __syncthreads();
    const auto step = [&](int tile, bool checked) __attribute__((always_inline)) {
      const Buf<D>& b = buf[(tile - tile0) & 1];
      Buf<D>& next = buf[(tile + 1 - tile0) & 1];
      // the next tile's codes (behind the last tile: the block of its last position again, unused)
      id = uniform(then);
      fetch_k(tile + 1, id, rk);
      if (!kApart) fetch_v(tile + 1, id, rv);
      then = id_at(tile + 2);
      f16v scs[kBoth ? SUB : 1];
      f4 scales[kBoth ? SUB : 1];
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        const int p0 = tile * T + 32 * u;
        const bool work = p0 < most_see;
        if (!kApart && !work) continue;
#pragma unroll
        for (int v = u; v < (kBoth ? SUB : u + 1); ++v) {
          if ((kApart && !work) || (kBoth && u > 0)) break;
          f16v& sc = scs[kBoth ? v : 0];
          f4& scale = scales[kBoth ? v : 0];
          sc = f16v{};
          const int lz = kApart ? again(lane) : lane;
          const uint8_t* kb = b.k + (32 * v + (lz & 31)) * C::KP + 16 * (lz >> 5);
          h8 a[kAhead], q[C::QL ? C::QL : 1];
#pragma unroll
          for (int k = 0; k < kAhead; ++k) a[k] = *reinterpret_cast<const h8*>(kb + 32 * k);
          __builtin_amdgcn_sched_group_barrier(kDsRead, kAhead, 0);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            sc = mfma(a[k % kAhead], k < QR ? Q[k < QR ? k : 0] : q[k < QR ? 0 : k - QR], sc);
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            if (k + kAhead < D / 16) {
              a[k % kAhead] = *reinterpret_cast<const h8*>(kb + 32 * (k + kAhead));
              __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
            }
            if (k + kAhead >= QR && k + kAhead < D / 16) {
              q[k + kAhead - QR] = qlds[k + kAhead - QR][tid];
              __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
            }
            if (k + kAhead == D / 16) {
              scale = *reinterpret_cast<const f4*>(b.scale[v]);
              __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
            }
          }
        }
        if (kApart) {
          __builtin_amdgcn_sched_barrier(0);
          convert_k(rk, next);
          __builtin_amdgcn_sched_barrier(0);
          fetch_v(tile + 1, id, rv);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (kApart && !work) continue;
        f16v& sc = scs[kBoth ? u : 0];
        const f4& scale = scales[kBoth ? u : 0];
        const float ks[2] = {uniform(scale[0]), uniform(scale[1])}, vs[2] = {uniform(scale[2]), uniform(scale[3])};
        // (the factors are positive, so the largest score of a half is its largest product times the factor)
        float f[2] = {qf * ks[0], qf * ks[1]};
        if (p0 + 32 > all_see || !(ks[0] >= 0.0f) || !(ks[1] >= 0.0f)) {
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            if (ks[s] != ks[s]) poison = uniform(min(poison, p0 + 16 * s));
            const int seen = ks[s] >= 0.0f ? see : 0;
            f[s] = f[s] >= kLeast ? f[s] : kLeast;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              sc[8 * s + j] = p0 + 16 * s + 8 * (j >> 2) + 4 * g + (j & 3) < seen ? sc[8 * s + j] : -__builtin_inff();
          }
        }
        float top2[2];
#pragma unroll
        for (int s = 0; s < 2; ++s)
          top2[s] = max3(max3(max3(sc[8 * s], sc[8 * s + 1], sc[8 * s + 2]), sc[8 * s + 3], sc[8 * s + 4]),
                         sc[8 * s + 5], __builtin_elementwise_maximum(sc[8 * s + 6], sc[8 * s + 7]));
        const float top = max_xor32(fmaxf(top2[0] * f[0], top2[1] * f[1]));
        const bool rise = top > m + kLag;
        if (__any(rise)) {
          const float m1 = rise ? top : m;
          const float a = m1 == m ? 1.0f : exp2_(m - m1);
          sum *= a, part *= a;
          m = m1;
          lift = kLift - fmaxf(m, -0x1p120f);          // (a row that has seen nothing: 2^-inf is 0 for any of these)
#pragma unroll
          for (int c = 0; c < DT; ++c) acc[c] *= a;
        }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          // V's scale relative to the unit (ru) goes into the exponent: P = 2^(x - m + 10 + log2 ru), and the row sum
          // adds P / ru.  Most halves have the scale of the one before.
          if (__float_as_int(vs[s]) != last) {
            last = __float_as_int(vs[s]);
            if (vs[s] > unit || (vs[s] > 0.0f && vs[s] < 0.25f * unit)) {
              const float a = new_unit(vs[s], unit, peak);
              unit = uniform(unit), peak = uniform(peak);
#pragma unroll
              for (int c = 0; c < DT; ++c) acc[c] *= a;
            }
            ru = uniform(unit > 0.0f ? vs[s] / unit : 0.0f);
            lost = uniform((int)(ru < 0.25f));                       // (a scale of 0, or 2^-80 below the largest)
            const float rs = lost ? 1.0f : ru;
            sum = fmaf(part, per_ru, sum), part = 0.0f;
            log_ru = uniform(__builtin_amdgcn_logf(rs)), per_ru = uniform(1.0f / rs);
          }
          __builtin_amdgcn_sched_barrier(0);
          const float off = log_ru + lift;
          h8 p;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const h2 y = h2_rne(exp2_(fmaf(sc[8 * s + 2 * j], f[s], off)), exp2_(fmaf(sc[8 * s + 2 * j + 1], f[s], off)));
            part = __builtin_amdgcn_fdot2(y, h2{(_Float16)1.0f, (_Float16)1.0f}, part, false);
            p[2 * j] = y.x, p[2 * j + 1] = y.y;
          }
          if (lost) p = p * (_Float16)ru;
          const int lz = kApart ? again(lane) : lane;
          const uint8_t* vb = b.v + (lz & 31) * C::VP + 16 * C::piece(lz, 4 * u + 2 * s + (lz >> 5));
          constexpr int AV = DT < kAhead ? DT : kAhead;
          h8 a[AV];
#pragma unroll
          for (int c = 0; c < AV; ++c) a[c] = *reinterpret_cast<const h8*>(vb + 32 * c * C::VP);
          __builtin_amdgcn_sched_group_barrier(kDsRead, AV, 0);
#pragma unroll
          for (int c = 0; c < DT; ++c) {
            acc[c] = mfma(a[c % AV], p, acc[c]);
            __builtin_amdgcn_sched_group_barrier(kMfma, 1, 0);
            if (c + AV < DT) {
              a[c % AV] = *reinterpret_cast<const h8*>(vb + 32 * (c + AV) * C::VP);
              __builtin_amdgcn_sched_group_barrier(kDsRead, 1, 0);
            }
          }
        }
      }
      if (!kApart) convert_k(rk, next);
      convert_v(tile + 1, id, rv, next, checked);
      __syncthreads();
    };
    // Tiles that some row does not see to their end are the last few: only those (each as the next tile, behind the
    // products) are searched for NaN codes, in a loop of their own.  In one loop the search takes registers that spill
    // at D = 256 (10,001 tokens 912 -> 933 us).
    const int plain = CODE == kE4M3 ? min(max(fewest / T - 1, tile0), tile1) : tile1;
    int tile = tile0;
    for (; tile < plain; ++tile) step(tile, false);
    if (CODE == kE4M3)
      for (; tile < tile1; ++tile) step(tile, true);
  }

  // register i of acc[c]: channel 32 c + 8 (i / 4) + 4 g + i % 4 of row l
  sum = sum_xor32(fmaf(part, per_ru, sum));
  if (poison < see) sum = __builtin_nanf("");
  int row = again(l);                           // (its query and head are computed again: no registers for them till now)
  row += 32 * wave;
  if (row >= it.n_row) return;
  const int qi = (it.row0 + row) / P.gs, hq = h * P.gs + (it.row0 + row) % P.gs;
  const float f = sum == 0.0f ? 0.0f : unit / sum;
  if (CODE == kE4M3 && nans.any()) {
    const int seen = sees(P, it, qi), gz = again(lane) >> 5;
#pragma unroll
    for (int c = 0; c < DT; ++c)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if (nans.at[32 * c + 8 * (i >> 2) + 4 * gz + (i & 3)] < seen) acc[c][i] = __builtin_nanf("");
        if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);
      }
  }
  if (used == 1) {
    const int64_t o = (int64_t)(it.q0 + qi) * P.so_n + (int64_t)hq * P.so_h + 4 * g;
    const float nan = sum == 0.0f ? __builtin_nanf("") : 0.0f;
#pragma unroll
    for (int c = 0; c < DT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        store_out4(P.out, ot, o + 32 * c + 8 * i, acc[c][4 * i] * f + nan, acc[c][4 * i + 1] * f + nan,
                   acc[c][4 * i + 2] * f + nan, acc[c][4 * i + 3] * f + nan);
  } else {
    const int64_t part = (((int64_t)w * P.H + h) * P.splits + split) * kTileRows + row;
#pragma unroll
    for (int c = 0; c < DT; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 o = {acc[c][4 * i], acc[c][4 * i + 1], acc[c][4 * i + 2], acc[c][4 * i + 3]};
        *reinterpret_cast<f4*>(P.part_o + part * D + 32 * c + 8 * i + 4 * g) = o * f;
      }
    if (g == 0) P.part_ml[2 * part] = m, P.part_ml[2 * part + 1] = sum;
  }
}

template <int CODE, int QT, int D>
void launch(const Attn& P, int items, int ot, hipStream_t st) {
  block_tile_kernel<CODE, QT, D><<<dim3(P.H * items, P.splits), 256, 0, st>>>(P, items, ot);
}
template <int CODE, int QT>
void launch_d(const Attn& P, int D, int items, int ot, hipStream_t st) {
  if (D == 64) launch<CODE, QT, 64>(P, items, ot, st);
  else if (D == 128) launch<CODE, QT, 128>(P, items, ot, st);
  else launch<CODE, QT, 256>(P, items, ot, st);
}

}  // namespace

namespace kvt {
namespace blk {

int tile_positions(int D) { return D == 256 ? Tile<256>::T : 64; }

void tile_launch(const Attn& P, int code, int qt, int D, int items, int ot, hipStream_t st) {
  if (code == kE4M3) {
    if (qt == kBF16) launch_d<kE4M3, kBF16>(P, D, items, ot, st);
    else launch_d<kE4M3, kF16>(P, D, items, ot, st);
  } else {
    if (qt == kBF16) launch_d<kI8, kBF16>(P, D, items, ot, st);
    else launch_d<kI8, kF16>(P, D, items, ot, st);
  }
}

}  // namespace blk
}  // namespace kvt
