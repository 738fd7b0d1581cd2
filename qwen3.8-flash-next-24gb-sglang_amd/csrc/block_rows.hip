// Attention of few rows over the 8-bit block cache on the matrix cores: decode (one query token per request) and short
// chunks (kvt_block_decode, and kvt_block_prefill where a call has few rows).
//
//   out[row] = sum_p w_p sv_p vc_p / sum_p w_p,   w_p = exp(scale * sk_p * q . kc_p)
// over the positions p that the row sees; kc, vc are codes, sk, sv the scales of p's block and KV head.  A row is a
// (query, q head) pair of one KV head; 16 of them are one side of a matrix product.
//
// One workgroup of 4 wavefronts per (16 rows, KV head, split of the positions); a wavefront takes every fourth tile of
// 32 positions.  Nothing is staged in LDS: both products take their 8-bit operand from registers as it was loaded.
//   S^T = K Q^T (v_mfma_f32_16x16x32_f16): lane (l, g) (l = lane % 16, g = lane / 16) loads 16 bytes of position l at a
//     time; the k order of the product is the order of the bytes, and Q is loaded in the same order.
//   The result gives a lane four positions (4 g + i) of row l in each of the tile's two halves: these eight weights are
//     the lane's column of P^T in O^T += V^T P^T as they stand.  V^T's operand needs the same eight positions of one
//     channel: a lane loads D / 16 channels of each of them and pairs the bytes of two positions (v_perm_b32) before
//     the conversion.
// Codes are exact in fp16.  The scale of K multiplies the fp32 scores.  The scale of V is folded into P, relative to a
// running unit u: P holds w sv / u and O is kept in units of u, which changes only when a tile's scale leaves [u / 4,
// u] (O is then multiplied by the ratio; two blocks of one tile whose scales differ by more than 4 take a product
// each).  The softmax keeps a running maximum m per row that moves only when a tile exceeds it by more than 4 (in
// powers of two), and P = 2^(x - m + 10): fp16 has weights down to 2^-24 of the largest before they lose bits, and up
// to 2^14 for a row whose maximum lags.  Sums, scores and O are fp32.  bf16 queries are scaled by a power of two per
// row to fit fp16 (exact down to 2^-14 of the row's largest entry, and to 2^-25 of it below).
//
// So two things have fewer bits than 32, both because a matrix operand has 16: the weights, and bf16 queries' smallest
// entries.  The row sums add the weights before that rounding here (they stand in fp32 registers), behind it in
// block_tile.hip (a dot product with ones).  Half a step of fp16 is an eighth of a bf16 output's: against 64 bits those
// are as far off as a form that holds fp32 throughout (relative 1.7e-3); fp16 outputs are 2.3 - 2.5e-4 off against
// 2.1e-4, and fp32 outputs have the weights' error too.
//
// Decode is bound by the cache's bytes, each read once (counted: 269 MB for 262,144 positions of 2 heads, D 256): 45.4
// us there, 5.9 TB/s (a large copy 5.2), where more than half of the wavefronts' time is waiting for memory and the
// vector instructions take 28 %, the matrix instructions 8 % of theirs; e4m3, 32 requests of 16,384 positions and less
// (204 MB) 37.5 us, 5.4 TB/s; int8, 64 requests x 8 heads, D 128 (456 MB) 96.7 us, 4.7 TB/s.  Short calls are launch
// and load latency: 777 positions of 2 heads 12.6 us with the merge in the launch.
#include "block_attn.h"

using namespace kvt;
using namespace kvt::blk;

namespace {

constexpr int kWaves = 4;
constexpr int kTile = 32;
constexpr int kMostSplits = 1024;
// Positions of a table that the kernels take: their 32-bit positions run ahead of an item's last one, by the most in
// block_rows_kernel (a wavefront asks for the block ids of its next 32 tiles, 4,096 positions).
constexpr int64_t kMostPositions = ((int64_t)1 << 31) - 8192;
constexpr int kMostParts = 128;        // parts of a pair, at most, where the launch of equal shares merges them
constexpr int kFew = 16;               // splits that the launch itself may merge, or a merge without LDS

// The parts of an item that the launch merges itself cross XCDs, whose L2s do not see each other: they are written and
// read at device scope (cache policy sc1).
typedef unsigned int b16v __attribute__((vector_size(16)));
typedef unsigned int b8v __attribute__((vector_size(8)));
constexpr int kSc1 = 16;
KVT_DEV __amdgpu_buffer_rsrc_t part_rsrc(float* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(p, 0, bytes, 0x00020000);
}

// A part's weight in the merge of normalized parts, from its maximum and sum and the row's maximum.  Sums are below
// 2^45: times 2^-45 no product with a part is larger than the part, and their sums stay finite.
KVT_DEV float weight_of(float m, float l, float M) { return m == -__builtin_inff() ? 0.0f : exp2_(m - M) * l * 0x1p-45f; }

template <int BYTES> struct Raw { uint32_t w[BYTES / 4]; };
template <int BYTES>
KVT_DEV Raw<BYTES> load(const uint8_t* base, uint32_t off) {
  Raw<BYTES> r;
  if constexpr (BYTES == 16) {
    const u4v x = *reinterpret_cast<const u4v*>(base + off);
    r.w[0] = x.x, r.w[1] = x.y, r.w[2] = x.z, r.w[3] = x.w;
  } else if constexpr (BYTES == 8) {
    const u2v x = *reinterpret_cast<const u2v*>(base + off);
    r.w[0] = x.x, r.w[1] = x.y;
  } else {
    r.w[0] = *reinterpret_cast<const uint32_t*>(base + off);
  }
  return r;
}

KVT_DEV f4 mfma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
KVT_DEV float lane_f(float v, int lane) {
  return bits_f((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}

// The wavefronts' results: O (rows x channels), maximum, sum, unit; NaN codes of V.
template <int CODE, int D>
struct Join {
  float o[kWaves][16][D + 4];
  float m[kWaves][16], l[kWaves][16], u[kWaves];
  float w[16][kFew];           // (weights of the splits of a row, where the launch merges them)
  NanAt<CODE, D> nans;
  int last;
};

// Tiles tile0 .. tile1 - 1 of an item and KV head: into out where they are all that the item has (whole), else as part
// `slot`: its own result with its maximum and sum.  CHUNK: its rows may see different positions.
template <int CODE, int QT, int D, bool CHUNK>
KVT_DEV void attend(const Attn& P, const Item& it, int h, int tile0, int tile1, bool whole, int64_t slot, int ot,
                    Join<CODE, D>& J) {
  constexpr int NC = D / 64;          // 16-byte chunks of a K row per lane
  constexpr int VB = D / 16;          // bytes (channels) of a V row per lane
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const int my = it.row0 + l, qi = my / P.gs;
  const bool live = l < it.n_row;
  h8 Q[D / 32];
  // (chunk c of 64 channels: 16 of them per group g, two operands)
  // (rows behind the item's last compute what its first does; nothing is stored of them)
  const int lq = live ? my : it.row0;
  const float qf = load_q<QT>(P.q, (int64_t)(it.q0 + lq / P.gs) * P.sq_n + (int64_t)(h * P.gs + lq % P.gs) * P.sq_h,
                              [g](int k) { return 64 * (k >> 1) + 16 * g + 8 * (k & 1); }, max_xor16_32, Q) * P.scale_log2;
  const int see = sees(P, it, qi);
  const int all_see = sees(P, it, it.row0 / P.gs);   // (the fewest of the item's rows: positions below it need no comparison)

  f4 acc[VB];
#pragma unroll
  for (int c = 0; c < VB; ++c) acc[c] = f4{0, 0, 0, 0};
  float m = -__builtin_inff(), sum = 0.0f, unit = 0.0f, peak = 0.0f;
  int poison = 0x7FFFFFFF;            // the wavefront's first position of a V scale that is not finite (uniform)

  const uint32_t koff = (uint32_t)l * D + 16u * g, voff = 4u * g * D + (uint32_t)l * VB;
  const int64_t tbl = (int64_t)it.trow * P.stride;

  for (int base = tile0 + wave; base < tile1; base += 32 * kWaves) {
    // blocks and scales of the next 32 tiles: lane 2 i + s has half s of tile base + 4 i
    int id = -1;
    float sk = 0.0f, sv = 0.0f;
    {
      const int p = (base + (lane >> 1) * kWaves) * kTile + 16 * (lane & 1);
      if (p < it.limit) id = P.table[tbl + (p >> P.log2b)];
      if (id < 0 || id >= P.n_blocks) id = -1;
      if (id >= 0) sk = P.ks[(int64_t)id * P.H + h], sv = P.vs[(int64_t)id * P.H + h];
    }
    for (int i = 0; i < 32; ++i) {
      const int tile = base + i * kWaves;
      if (tile >= tile1) break;
      const int p0 = tile * kTile;
      int valid[2];
      const uint8_t *kp[2], *vp[2];
      float fk[2], fv[2];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int b = __builtin_amdgcn_readlane(id, 2 * i + s);
        const int64_t at = ((((int64_t)max(b, 0) * P.H + h) << P.log2b) + ((p0 + 16 * s) & ((1 << P.log2b) - 1))) * D;
        kp[s] = P.k8 + at, vp[s] = P.v8 + at;
        fk[s] = lane_f(sk, 2 * i + s), fv[s] = lane_f(sv, 2 * i + s);
        valid[s] = b < 0 ? 0 : min(max(it.limit - (p0 + 16 * s), 0), 16);
      }
      Raw<16> kr[2][NC];
      Raw<VB> vr[2][4];
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int c = 0; c < NC; ++c) kr[s][c] = load<16>(kp[s], koff + 64u * c);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) vr[s][j] = load<VB>(vp[s], voff + (uint32_t)j * D);

      float x[2][4];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        f4 sc = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          sc = mfma(operand<CODE>(kr[s][c].w[0], kr[s][c].w[1]), Q[2 * c], sc);
          sc = mfma(operand<CODE>(kr[s][c].w[2], kr[s][c].w[3]), Q[2 * c + 1], sc);
        }
        const float f = fmaf(qf, fk[s], fk[s] - fk[s]);            // (NaN for a scale that is not finite)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[s][j] = sc[j] * f;
      }
      if (valid[0] + valid[1] < 32 || p0 + 32 > all_see) {
        // positions past a row's end, in a block that is not there, or stale (their V may hold anything: it counts as
        // 0)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int at = 4 * g + j;
            x[s][j] = at < valid[s] && p0 + 16 * s + at < see ? x[s][j] : -__builtin_inff();
#pragma unroll
            for (int d = 0; d < VB / 4; ++d) vr[s][j].w[d] = at < valid[s] ? vr[s][j].w[d] : 0u;
          }
        if (CHUNK && CODE == kE4M3 && P.causal) {
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              J.nans.template take<VB / 4>(vr[s][j].w, [&](int) { return p0 + 16 * s + 4 * g + j; }, l * VB, 4);
        }
      }
      float top = fmaxf(fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3])),
                        fmaxf(fmaxf(x[1][0], x[1][1]), fmaxf(x[1][2], x[1][3])));
      top = max_xor16_32(top);
      const bool rise = top > m + kLag;
      if (__any(rise)) {
        const float m1 = rise ? top : m;
        const float a = m1 == m ? 1.0f : exp2_(m - m1);             // (m = -inf: 0)
        sum *= a;
        m = m1;
#pragma unroll
        for (int c = 0; c < VB; ++c) acc[c] *= a;
      }
      const float ms = (m == -__builtin_inff() ? 0.0f : m) - kLift;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[s][j] = exp2_(x[s][j] - ms);
          sum += x[s][j];
        }
      // (two blocks whose scales are far apart in one tile: one product for each, so that neither's weights leave fp16)
      const bool far = fminf(fv[0], fv[1]) > 0.0f && (fv[0] < 0.25f * fv[1] || fv[1] < 0.25f * fv[0]);
      for (int pass = 0; pass <= (int)far; ++pass) {
        float big = far ? fv[pass] : __builtin_elementwise_maximum(fv[0], fv[1]);
        if (!(big <= unit) || (big > 0.0f && big < 0.25f * unit)) { // uniform
          if (!finite_scales(big, big)) {
#pragma unroll
            for (int s = 0; s < 2; ++s)
              if (!finite_scales(fv[s], fv[s])) poison = min(poison, p0 + 16 * s), fv[s] = 0.0f;
            big = fmaxf(fv[0], fv[1]);
          }
          if (big > 0.0f) {
            const float a = new_unit(big, unit, peak);
#pragma unroll
            for (int c = 0; c < VB; ++c) acc[c] *= a;
          }
        }
        h8 p;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const float ru = unit > 0.0f && !(far && s != pass) ? fv[s] / unit : 0.0f;
#pragma unroll
          for (int j = 0; j < 4; ++j) p[4 * s + j] = (_Float16)(x[s][j] * ru);
        }
#pragma unroll
        for (int d = 0; d < VB / 4; ++d) {
          uint32_t lo4[4], hi4[4];                                  // {pair (0,1), (2,3) of half 0, of half 1}
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint32_t a = flip<CODE>(vr[s][2 * j].w[d]), b = flip<CODE>(vr[s][2 * j + 1].w[d]);
              lo4[2 * s + j] = __builtin_amdgcn_perm(b, a, 0x05010400u);   // a0 b0 a1 b1
              hi4[2 * s + j] = __builtin_amdgcn_perm(b, a, 0x07030602u);   // a2 b2 a3 b3
            }
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            h2 y[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t u = c < 2 ? lo4[k] : hi4[k];
              y[k] = c & 1 ? pair<CODE, true>(u) : pair<CODE, false>(u);
            }
            const h8 a = {y[0].x, y[0].y, y[1].x, y[1].y, y[2].x, y[2].y, y[3].x, y[3].y};
            acc[4 * d + c] = mfma(a, p, acc[4 * d + c]);
          }
        }
      }
    }
  }

  // the wavefronts' parts -> one: acc[c][i] is channel VB (4 g + i) + c of row l
  sum = sum_xor16_32(sum);
  if (poison < see) sum = __builtin_nanf("");
  if (live) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < VB; c += 4)
        *reinterpret_cast<f4*>(&J.o[wave][l][VB * (4 * g + i) + c]) = f4{acc[c][i], acc[c + 1][i], acc[c + 2][i], acc[c + 3][i]};
    if (g == 0) J.m[wave][l] = m, J.l[wave][l] = sum;
  }
  if (lane == 0) J.u[wave] = unit;
  __syncthreads();
  for (int e = threadIdx.x; e < it.n_row * (D / 4); e += 256) {
    const int row = e / (D / 4), d = 4 * (e % (D / 4));
    float M = -__builtin_inff();
#pragma unroll
    for (int v = 0; v < kWaves; ++v) M = fmaxf(M, J.m[v][row]);
    float L = 0.0f, f[kWaves];
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      f[v] = J.m[v][row] == -__builtin_inff() ? 0.0f : exp2_(J.m[v][row] - M);
      L += f[v] * J.l[v][row];
    }
    // (divided by the sum before the unit comes in: no product is larger than the values themselves)
    f4 O = {0, 0, 0, 0};
    const float per = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) O += *reinterpret_cast<const f4*>(&J.o[v][row][d]) * (f[v] * per) * J.u[v];
    if (CHUNK && CODE == kE4M3 && P.causal && J.nans.any()) {
      const int seen = sees(P, it, (it.row0 + row) / P.gs);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (J.nans.at[d + i] < seen) O[i] = __builtin_nanf("");
    }
    if (whole) {
      const int at = it.row0 + row;
      const int64_t o = (int64_t)(it.q0 + at / P.gs) * P.so_n + (int64_t)(h * P.gs + at % P.gs) * P.so_h + d;
      if (L == 0.0f) O = f4{1, 1, 1, 1} * __builtin_nanf("");
      store_out4(P.out, ot, o, O[0], O[1], O[2], O[3]);
    } else {
      const int64_t part = slot * 16 + row;
      if (P.counters) {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(b16v, O), part_rsrc(P.part_o + slot * 16 * D, 64 * D),
                                               (row * D + d) * 4, 0, kSc1);
        if (d == 0)
          __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(b8v, make_float2(M, L)), part_rsrc(P.part_ml + slot * 32, 128),
                                                row * 8, 0, kSc1);
      } else {
        *reinterpret_cast<f4*>(P.part_o + part * D + d) = O;
        if (d == 0) P.part_ml[2 * part] = M, P.part_ml[2 * part + 1] = L;
      }
    }
  }
}

// The merge of an item's parts by the workgroup that finishes last (counters: zero before and after every call): part 0
// is in slot s0, part k > 0 in slot sb + step k.  Parts cross XCDs, whose L2s do not see each other: they are stored
// and loaded at device scope, and a workgroup counts itself when its stores have arrived.  Nobody waits for another
// workgroup.  The parts are added in their order whoever merges them, as the merge by a second launch does: the same
// bits.
//
// A thread has four channels of a row at a time, and loads them of 16 parts at once: of its first row beside the parts'
// maxima.  Most items have no more parts (MANY: they may, D 64 and 128; at D 256 the registers would spill).
template <int CODE, int D, bool MANY>
KVT_DEV void merge_last(const Attn& P, const Item& it, int h, int64_t item, int parts, int64_t s0, int64_t sb, int step, int ot,
                        Join<CODE, D>& J) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();                                  // every thread's parts have arrived
  if (threadIdx.x == 0) {
    int32_t* c = P.counters + item;
    J.last = __hip_atomic_fetch_add(c, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == parts - 1;
    if (J.last) __hip_atomic_store(c, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!J.last) return;
  const auto ro = part_rsrc(P.part_o + s0 * 16 * D, (step * parts + 1) * 64 * D);
  const auto rml = part_rsrc(P.part_ml + s0 * 32, (step * parts + 1) * 128);
  const int base = (int)(sb - s0), end = it.n_row * (D / 4);   // (slots from here on count from s0)
  const auto slot = [&](int k) { return k ? base + step * k : 0; };
  // (no branch around a load, which would wait for it: what is not there is an offset past the buffer, and reads 0)
  f4 o[kFew];
  const auto load = [&](int e, int k0) {            // row e / (D / 4), channels 4 (e % (D / 4)) ..
#pragma unroll
    for (int k = 0; k < kFew; ++k)
      o[k] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(
                                        ro, k0 + k < parts && e < end ? 64 * D * slot(k0 + k) + 16 * e : -16, 0, kSc1));
  };
  const int row = threadIdx.x >> 4, lane = threadIdx.x & 15;   // 16 rows x 16 parts
  const auto read_ml = [&](int k) {
    const bool is = row < it.n_row && k < parts;
    const float2 ml = __builtin_bit_cast(
        float2, __builtin_amdgcn_raw_buffer_load_b64(rml, is ? (16 * slot(k) + row) * 8 : -8, 0, kSc1));
    return make_float2(is ? ml.x : -__builtin_inff(), ml.y);
  };
  const auto add = [&](int e, f4& O, float& L) {
    const int r = e / (D / 4);
#pragma unroll
    for (int k = 0; k < kFew; ++k) {
      const float f = J.w[r][k];
      L += f;
      O += f * o[k];
    }
  };
  const auto write = [&](int e, const f4& O, float L) {
    const int at = it.row0 + e / (D / 4), d = 4 * (e % (D / 4));
    const f4 y = L == 0.0f ? f4{1, 1, 1, 1} * __builtin_nanf("") : O / L;
    store_out4(P.out, ot, (int64_t)(it.q0 + at / P.gs) * P.so_n + (int64_t)(h * P.gs + at % P.gs) * P.so_h + d, y[0], y[1], y[2],
               y[3]);
  };
  load(threadIdx.x, 0);
  float2 ml = read_ml(lane);
  float M = ml.x;
  if (MANY)
    for (int k = lane + kFew; k < parts; k += kFew) M = fmaxf(M, read_ml(k).x);
  M = group_max<16>(M);
  if (!MANY || parts <= kFew) {
    J.w[row][lane] = weight_of(ml.x, ml.y, M);
    __syncthreads();
    for (int e = threadIdx.x;;) {
      f4 O = {0, 0, 0, 0};
      float L = 0.0f;
      if (e < end) {
        add(e, O, L);
        write(e, O, L);
      }
      e += 256;
      if (e - (int)threadIdx.x >= end) break;
      load(e, 0);
    }
    return;
  }
  constexpr int NE = MANY ? D / 64 : 1;             // 16 rows over 256 threads
  f4 O[NE];
  float L[NE];
#pragma unroll
  for (int n = 0; n < NE; ++n) O[n] = f4{0, 0, 0, 0}, L[n] = 0.0f;
  for (int k0 = 0; k0 < parts; k0 += kFew) {
    if (k0) {
      load(threadIdx.x, k0);
      ml = read_ml(k0 + lane);
    }
    J.w[row][lane] = weight_of(ml.x, ml.y, M);
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NE; ++n) {
      if (n) load(threadIdx.x + 256 * n, k0);
      add(threadIdx.x + 256 * n, O[n], L[n]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < NE; ++n)
    if ((int)threadIdx.x + 256 * n < end) write(threadIdx.x + 256 * n, O[n], L[n]);
}

template <int CODE, int QT, int D>
__global__ __launch_bounds__(256, 2) void block_rows_kernel(const Attn P, int ot) {
  __shared__ Join<CODE, D> J;
  const int split = blockIdx.x, h = blockIdx.y, w = blockIdx.z;
  const Item it = item_of(P, w);
  if (it.n_row == 0) return;
  const int tps = tiles_per_split(P, it.limit);
  const int tile0 = split * tps, tile1 = min(tile0 + tps, tiles_of(P, it.limit));
  const int used = splits_used(P, it.limit);
  if (split >= used) return;                        // (the merge knows which splits there are)
  const int64_t item = (int64_t)w * P.H + h;
  if (CODE == kE4M3 && P.causal) {
    J.nans.clear();
    __syncthreads();
  }
  attend<CODE, QT, D, true>(P, it, h, tile0, tile1, used == 1, item * P.splits + split, ot, J);
  if (P.counters && used > 1) merge_last<CODE, D, false>(P, it, h, item, used, item * P.splits, item * P.splits, 1, ot, J);
}

// Decode in equal shares of all tiles of a call: the (request, KV head) pairs stand in a line, each as long as its
// tiles plus kPad (what beginning with a pair costs, about: Q, the first loads, the join), and workgroup w takes [w
// share, (w + 1) share) of it.  A pair that one workgroup has is written at once; of a pair that several have, each
// leaves a part, which the last of them or a second launch merges.  A workgroup has at most two such pairs, its first
// (slot 2 w) and its last (2 w + 1): 2 slots per workgroup whatever the lengths are.  (With a fixed number of splits
// per pair, workgroups of a ragged batch are short and unequal: 64 requests x 8 heads (D 128), up to 8,191 positions
// 117 us against 98.)
constexpr int kPad = 8;

// A request's table row and length; rows out of range hold nothing.
struct Held {
  int row, len;
};
KVT_DEV Held held(const Attn& P, int r) {
  const int row = P.rows ? P.rows[r] : r, len = (int)min((int64_t)max(P.kv_lens[r], 0), (int64_t)P.max_blocks << P.log2b);
  return row < 0 || row >= P.n_rows ? Held{0, 0} : Held{row, len};
}
KVT_DEV int tiles_in(int len) { return (len + kTile - 1) / kTile; }

// Inclusive sums over the wavefront's lanes (all active).
KVT_DEV uint32_t wave_scan(uint32_t v) {
  int x = (int)v;
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8: within 16 lanes
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);   // lane 15 of rows 0, 2 to rows 1, 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);   // lane 31 to the upper half
  return (uint32_t)x;
}
// The line of a call, per head, in steps of 2^shift tiles (the entry point picks the shift so that 32 bits hold it):
// its length, where request r begins, and what r holds.
struct Line {
  uint32_t total, at;
  int r;
  Held has;
};
KVT_DEV uint32_t steps_of(const Attn& P, int tiles) { return (uint32_t)((tiles + kPad + (1 << P.shift) - 1) >> P.shift); }
// find(total, before, own, r): whether r, which takes `own` steps behind `before`, is the request sought.
template <class Find>
KVT_DEV Line line_of(const Attn& P, Find find) {
  const int lane = threadIdx.x & 63;
  Line s{0, 0, 0, {0, 0}};
  Held has{0, 0};
  uint32_t own = 0, sum = 0;
  const auto look = [&](int c) {
    has = held(P, min(c + lane, P.n - 1));
    own = c + lane < P.n ? steps_of(P, tiles_in(has.len)) : 0u;
    sum = wave_scan(own);
  };
  for (int c = 0; c < P.n; c += 64) {
    look(c);
    s.total += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  }
  uint32_t before = 0;
  for (int c = 0; c < P.n; c += 64) {
    if (P.n > 64) look(c);
    const uint64_t hit = __ballot(c + lane < P.n && find(s.total, before + sum - own, own, c + lane));
    if (hit) {
      const int i = __builtin_ctzll(hit);
      s.r = c + i, s.at = before + (uint32_t)__builtin_amdgcn_readlane((int)(sum - own), i);
      s.has = Held{__builtin_amdgcn_readlane(has.row, i), __builtin_amdgcn_readlane(has.len, i)};
      break;
    }
    before += (uint32_t)__builtin_amdgcn_readlane((int)sum, 63);
  }
  return s;
}
KVT_DEV uint32_t share_of(const Attn& P, uint32_t total) {
  return max((total * P.H + P.shares - 1) / P.shares, (kWaves + (1u << P.shift) - 1) >> P.shift);
}

template <int CODE, int QT, int D>
__global__ __launch_bounds__(256, 2) void block_decode_kernel(const Attn P, int ot) {
  __shared__ Join<CODE, D> J;
  const uint32_t w = blockIdx.x;
  const Line s = line_of(P, [&](uint32_t total, uint32_t before, uint32_t own, int) {
    const uint32_t x = w * share_of(P, total);
    return before * P.H <= x && x < (before + own) * P.H;
  });
  const uint32_t share = share_of(P, s.total), all = s.total * P.H, x0 = w * share, x1 = min(x0 + share, all);
  if (x0 >= x1) return;
  int r = s.r;
  uint32_t at = s.at * P.H;                         // of request r's head 0
  Held has = s.has;
  uint32_t steps = steps_of(P, tiles_in(has.len));
  int h = (int)((x0 - at) / steps);                 // (the first pair)
  for (;;) {
    Item it;
    it.r = r, it.trow = has.row, it.q0 = r, it.q_len = 1, it.row0 = 0, it.n_row = P.gs;
    it.kv = it.len = it.limit = has.len;
    const Held then = held(P, min(r + 1, P.n - 1));  // (the next request's: under this one's work)
    const int tiles = tiles_in(has.len);
    for (; h < P.H; ++h) {
      const uint32_t a = at + (uint32_t)h * steps;
      if (a >= x1) return;
      const int t0 = a < x0 ? (int)min((uint64_t)(x0 - a) << P.shift, (uint64_t)tiles) : 0;
      const int t1 = (int)min((uint64_t)(x1 - a) << P.shift, (uint64_t)tiles);
      if (t0 < t1 || (tiles == 0 && a >= x0)) {
        const bool whole = t0 == 0 && t1 == tiles;
        attend<CODE, QT, D, false>(P, it, h, t0, t1, whole, 2 * (int64_t)w + (a > x0), ot, J);
        if (D < 256 && P.counters && !whole) {      // (at D 256 the merge's registers would spill)
          const int w0 = (int)(a / share), w1 = (int)((a + (uint32_t)((tiles - 1) >> P.shift)) / share);
          merge_last<CODE, D, (D < 256)>(P, it, h, (int64_t)r * P.H + h, w1 - w0 + 1,
                                         2 * (int64_t)w0 + (a > (uint32_t)w0 * share), 2 * (int64_t)w0, 2, ot, J);
        }
        __syncthreads();                            // (J is free again)
      }
    }
    h = 0;
    at += P.H * steps;
    if (++r >= P.n || at >= x1) return;
    has = Held{uniform(then.row), uniform(then.len)};
    steps = steps_of(P, tiles_in(has.len));
  }
}

// The merge of shared decode: pair (blockIdx.z, blockIdx.y)'s parts, where it has several.  D / 4 lanes per row.
template <int D>
__global__ __launch_bounds__(256) void block_decode_merge_kernel(const Attn P, int ot) {
  constexpr int LPR = D / 4;
  const int h = blockIdx.y, r = blockIdx.z, row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, d = 4 * (threadIdx.x % LPR);
  const Line s = line_of(P, [&](uint32_t, uint32_t, uint32_t, int i) { return i == r; });
  const uint32_t share = share_of(P, s.total);
  const int tiles = tiles_in(s.has.len);
  const uint32_t a = s.at * P.H + (uint32_t)h * steps_of(P, tiles);
  const int w0 = (int)(a / share), w1 = (int)((a + (uint32_t)(max(tiles - 1, 0) >> P.shift)) / share);
  if (w0 == w1 || row >= P.gs) return;
  const auto part_of = [&](int w) { return (2 * (int64_t)w + (a > (uint32_t)w * share)) * 16 + row; };
  // (the first eight parts beside their maxima: most pairs have no more; those that are not there are the last again,
  // of no weight)
  constexpr int kNow = 8;
  f4 o[kNow];
  float2 now[kNow];
#pragma unroll
  for (int k = 0; k < kNow; ++k) {
    const int64_t p = part_of(min(w0 + k, w1));
    now[k] = *reinterpret_cast<const float2*>(P.part_ml + 2 * p);
    o[k] = *reinterpret_cast<const f4*>(P.part_o + p * D + d);
  }
  float M = -__builtin_inff(), L = 0.0f;
#pragma unroll
  for (int k = 0; k < kNow; ++k) M = fmaxf(M, now[k].x);
#pragma unroll 8
  for (int w = w0 + kNow; w <= w1; ++w) M = fmaxf(M, P.part_ml[2 * part_of(w)]);
  f4 O = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < kNow; ++k) {
    const float f = weight_of(now[k].x, now[k].y, M);
    L = w0 + k <= w1 ? L + f : L;
    O = w0 + k <= w1 ? O + f * o[k] : O;
  }
#pragma unroll 8
  for (int w = w0 + kNow; w <= w1; ++w) {
    const int64_t p = part_of(w);
    const float2 ml = *reinterpret_cast<const float2*>(P.part_ml + 2 * p);
    const float f = weight_of(ml.x, ml.y, M);
    L += f;
    O += f * *reinterpret_cast<const f4*>(P.part_o + p * D + d);
  }
  O = L == 0.0f ? f4{1, 1, 1, 1} * __builtin_nanf("") : O / L;
  store_out4(P.out, ot, (int64_t)r * P.so_n + (int64_t)(h * P.gs + row) * P.so_h + d, O[0], O[1], O[2], O[3]);
}

// Merge of the splits of a row: one workgroup per (row, 64 channels, KV head and item).  A part is a split's own result
// with its maximum m and sum l; their weights 2^(m - M) l / (the sum of these) go to LDS first, then groups of 16 lanes
// add up every NG-th split, all their loads in flight side by side.
template <int NT>
__global__ __launch_bounds__(NT) void block_merge_kernel(const Attn P, int D, int ot) {
  constexpr int NG = NT / 16;
  __shared__ float wgt[kMostSplits], red[NT / 64], red2[NT / 64];
  __shared__ f4 os[NG][16];
  const int row = blockIdx.x, dc = blockIdx.y, h = blockIdx.z % P.H, w = blockIdx.z / P.H;
  const Item it = item_of(P, w);
  const int used = splits_used(P, it.limit);
  if (row >= it.n_row || used == 1) return;
  const int64_t part = ((int64_t)w * P.H + h) * P.splits * P.item_rows + row;
  float M = -__builtin_inff(), L = 0.0f;
  for (int s = threadIdx.x; s < used; s += NT) M = fmaxf(M, P.part_ml[2 * (part + (int64_t)P.item_rows * s)]);
  M = group_max<64>(M);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = M;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) M = fmaxf(M, red[i]);
  for (int s = threadIdx.x; s < used; s += NT) {
    const float* ml = P.part_ml + 2 * (part + (int64_t)P.item_rows * s);
    const float f = ml[0] == -__builtin_inff() ? 0.0f : exp2_(ml[0] - M);
    wgt[s] = f * ml[1];
    L += wgt[s];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) L += __shfl_xor(L, o, 64);
  if ((threadIdx.x & 63) == 0) red2[threadIdx.x >> 6] = L;
  __syncthreads();
  L = 0.0f;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) L += red2[i];
  const float per = 1.0f / L;
  const int grp = threadIdx.x >> 4, d = 64 * dc + 4 * (threadIdx.x & 15);
  f4 O = {0, 0, 0, 0};
#pragma unroll 4
  for (int s = grp; s < used; s += NG)
    O += (wgt[s] * per) * *reinterpret_cast<const f4*>(P.part_o + (part + (int64_t)P.item_rows * s) * D + d);
  os[grp][threadIdx.x & 15] = O;
  __syncthreads();
  if (grp) return;
  for (int i = 1; i < NG; ++i) O += os[i][threadIdx.x];
  const int at = it.row0 + row;
  const int64_t o = (int64_t)(it.q0 + at / P.gs) * P.so_n + (int64_t)(h * P.gs + at % P.gs) * P.so_h + d;
  if (L == 0.0f) O = f4{1, 1, 1, 1} * __builtin_nanf("");
  store_out4(P.out, ot, o, O[0], O[1], O[2], O[3]);
}
// The same for up to kFew splits: D / 4 lanes per row, which read its parts side by side.
template <int D>
__global__ __launch_bounds__(256) void block_merge_few_kernel(const Attn P, int ot) {
  constexpr int LPR = D / 4;
  const int row = blockIdx.x * (256 / LPR) + threadIdx.x / LPR, d = 4 * (threadIdx.x % LPR), h = blockIdx.y, w = blockIdx.z;
  const Item it = item_of(P, w);
  const int used = splits_used(P, it.limit);
  if (row >= it.n_row || used == 1) return;
  const int64_t part = ((int64_t)w * P.H + h) * P.splits * P.item_rows + row;
  float wgt[kFew], l[kFew], M = -__builtin_inff(), L = 0.0f;
#pragma unroll
  for (int s = 0; s < kFew; ++s) {
    const float2 ml = s < used ? *reinterpret_cast<const float2*>(P.part_ml + 2 * (part + (int64_t)P.item_rows * s))
                               : make_float2(-__builtin_inff(), 0.0f);
    wgt[s] = ml.x, l[s] = ml.y;
  }
#pragma unroll
  for (int s = 0; s < kFew; ++s) M = fmaxf(M, wgt[s]);
#pragma unroll
  for (int s = 0; s < kFew; ++s) {
    wgt[s] = weight_of(wgt[s], l[s], M);
    L += wgt[s];
  }
  f4 O = {0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < kFew; ++s)
    if (s < used) O += wgt[s] * *reinterpret_cast<const f4*>(P.part_o + (part + (int64_t)P.item_rows * s) * D + d);
  const int at = it.row0 + row;
  const int64_t o = (int64_t)(it.q0 + at / P.gs) * P.so_n + (int64_t)(h * P.gs + at % P.gs) * P.so_h + d;
  O = L == 0.0f ? f4{1, 1, 1, 1} * __builtin_nanf("") : O / L;
  store_out4(P.out, ot, o, O[0], O[1], O[2], O[3]);
}
template <int D>
void merge(const Attn& P, int items, int rows, int ot, hipStream_t st) {
  if (P.splits <= kFew) {
    block_merge_few_kernel<D><<<dim3((rows * (D / 4) + 255) / 256, P.H, items), 256, 0, st>>>(P, ot);
  } else {
    const dim3 grid(rows, D / 64, P.H * items);
    if (P.splits > 64) block_merge_kernel<1024><<<grid, 1024, 0, st>>>(P, D, ot);
    else block_merge_kernel<256><<<grid, 256, 0, st>>>(P, D, ot);
  }
}

template <int CODE, int QT, int D>
void launch(const Attn& P, int items, int ot, hipStream_t st) {
  if (!P.shares) {
    block_rows_kernel<CODE, QT, D><<<dim3(P.splits, P.H, items), 256, 0, st>>>(P, ot);
    if (P.splits > 1 && !P.counters) merge<D>(P, items, P.cu ? 16 : P.gs, ot, st);
    return;
  }
  block_decode_kernel<CODE, QT, D><<<P.shares, 256, 0, st>>>(P, ot);
  if (P.shares > 1 && !P.counters)
    block_decode_merge_kernel<D><<<dim3((P.gs * (D / 4) + 255) / 256, P.H, P.n), 256, 0, st>>>(P, ot);
}
template <int CODE, int QT>
void launch_d(const Attn& P, int D, int items, int ot, hipStream_t st) {
  if (D == 64) launch<CODE, QT, 64>(P, items, ot, st);
  else if (D == 128) launch<CODE, QT, 128>(P, items, ot, st);
  else launch<CODE, QT, 256>(P, items, ot, st);
}
void launch_all(const Attn& P, int code, int qt, int D, int items, int ot, hipStream_t st) {
  if (code == kE4M3) {
    if (qt == kBF16) launch_d<kE4M3, kBF16>(P, D, items, ot, st);
    else launch_d<kE4M3, kF16>(P, D, items, ot, st);
  } else {
    if (qt == kBF16) launch_d<kI8, kBF16>(P, D, items, ot, st);
    else launch_d<kI8, kF16>(P, D, items, ot, st);
  }
}

int check(const Attn& P, int Hq, int D, int block, int code, int qt, int ot) {
  if (P.n < 1 || P.n > kMaxReq || P.H < 1 || Hq < P.H || Hq % P.H || Hq / P.H > 16 || P.n_rows < 1 || P.n_blocks < 1 ||
      P.max_blocks < 1 || P.stride < P.max_blocks || (!P.rows && P.n_rows < P.n) || P.splits < 1 ||
      !(P.scale_log2 > 0.0f))
    return KVT_EINVAL;
  if ((D != 64 && D != 128 && D != 256) || (block != 16 && block != 32 && block != 64)) return KVT_EINVAL;
  if ((code != kE4M3 && code != kI8) || (qt != kBF16 && qt != kF16) || (ot != kBF16 && ot != kF16 && ot != kF32))
    return KVT_EINVAL;
  if ((uintptr_t)P.q & 15 || P.sq_n % 8 || P.sq_h % 8 || ((uintptr_t)P.k8 | (uintptr_t)P.v8) & 15) return KVT_EINVAL;
  const int out8 = ot == kF32 ? 4 : 8;   // 16-byte aligned output rows
  if ((uintptr_t)P.out & 15 || P.so_n % out8 || P.so_h % out8) return KVT_EINVAL;
  if (P.H > 65535 || P.splits > kMostSplits || (int64_t)P.max_blocks * block > kMostPositions ||
      (int64_t)P.H * block * D > 0xFFFFFFFFll) return KVT_ERANGE;
  return KVT_OK;
}

}  // namespace

extern "C" int kvt_block_decode(const void* q, int64_t sq_n, int64_t sq_h, int q_type, const void* kv_lens, int n, int H,
                                int Hq, int D, int code, const void* k8, const void* v8, const void* ks, const void* vs,
                                int n_blocks, int block, const void* block_table, int64_t bt_stride, int n_rows,
                                int max_blocks, const void* rows, float scale, int n_splits, void* part_o,
                                void* part_ml, void* counters, void* out, int out_type, int64_t so_n, int64_t so_h,
                                void* stream) {
  Attn P;
  P.q = q, P.k8 = (const uint8_t*)k8, P.v8 = (const uint8_t*)v8, P.ks = (const float*)ks, P.vs = (const float*)vs;
  P.table = (const int32_t*)block_table, P.kv_lens = (const int32_t*)kv_lens, P.rows = (const int32_t*)rows;
  // One workgroup merges a pair's parts inside the launch: up to kFew splits, or kMostParts parts, which is about the
  // most that a pair can have of equal shares (one long request among short ones).  us per call, by a second launch /
  // inside: 64 requests x 8 heads (D 128), up to 8,191 positions 103 / 100, 32 x 8 up to 3,000 29.8 / 27.7, 32 x 4 up
  // to 16,000 51.5 / 46.8; of one of them alone among short ones 20.9 / 16.3, 16.4 / 11.4, 21.7 / 23.0; 32 x 1 (16 q
  // heads, 512 parts) 29.3 / 43.5.
  const bool few = n_splits > 1 ? n_splits <= kFew : n_splits < -1 && D < 256 && -(n_splits / (H > 0 ? H : 1)) <= kMostParts;
  P.counters = few ? (int32_t*)counters : nullptr;
  P.cu = nullptr, P.out = out, P.part_o = (float*)part_o, P.part_ml = (float*)part_ml;
  P.sq_n = sq_n, P.sq_h = sq_h, P.so_n = so_n, P.so_h = so_h, P.stride = bt_stride, P.scale_log2 = scale * kLog2e;
  P.n = n, P.n_rows = n_rows, P.n_q = n, P.H = H, P.gs = H > 0 ? Hq / H : 0, P.n_blocks = n_blocks;
  P.max_blocks = max_blocks, P.log2b = block == 16 ? 4 : block == 32 ? 5 : 6, P.causal = 0;
  P.splits = n_splits >= 0 ? n_splits : 1, P.shares = n_splits >= 0 ? 0 : -max(n_splits, -65536);
  P.item_rows = 16, P.tile = kTile, P.least = kWaves, P.single = 0, P.shift = 0;
  const double longest = (double)max_blocks * block / kTile + kPad;
  while (P.shift < 31 && (double)n * H * (longest / (1 << P.shift) + 2) + P.shares > 2e9) ++P.shift;
  const int st = check(P, Hq, D, block, code, q_type, out_type);
  if (st != KVT_OK) return st;
  if ((P.splits > 1 || P.shares > 1) && (!part_o || !part_ml)) return KVT_EINVAL;
  if (P.shares > 65535 || (n_splits > 1 && (int64_t)n * H > 65535)) return KVT_ERANGE;
  launch_all(P, code, q_type, D, n, out_type, (hipStream_t)stream);
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}

extern "C" int kvt_block_prefill(const void* q, int64_t sq_n, int64_t sq_h, int q_type, const void* cu_q, int n_q,
                                 const void* kv_lens, int n, int H, int Hq, int D, int code, const void* k8,
                                 const void* v8, const void* ks, const void* vs, int n_blocks, int block,
                                 const void* block_table, int64_t bt_stride, int n_rows, int max_blocks,
                                 const void* rows, int causal, float scale, int item_rows, int n_splits, void* part_o,
                                 void* part_ml, void* counters, void* out, int out_type, int64_t so_n, int64_t so_h,
                                 void* stream) {
  Attn P;
  P.q = q, P.k8 = (const uint8_t*)k8, P.v8 = (const uint8_t*)v8, P.ks = (const float*)ks, P.vs = (const float*)vs;
  P.table = (const int32_t*)block_table, P.kv_lens = (const int32_t*)kv_lens, P.rows = (const int32_t*)rows;
  P.counters = n_splits > 1 && n_splits <= kFew && item_rows == 16 ? (int32_t*)counters : nullptr;
  P.cu = (const int32_t*)cu_q, P.out = out, P.part_o = (float*)part_o, P.part_ml = (float*)part_ml;
  P.sq_n = sq_n, P.sq_h = sq_h, P.so_n = so_n, P.so_h = so_h, P.stride = bt_stride, P.scale_log2 = scale * kLog2e;
  P.n = n, P.n_rows = n_rows, P.n_q = n_q, P.H = H, P.gs = H > 0 ? Hq / H : 0, P.n_blocks = n_blocks;
  P.max_blocks = max_blocks, P.log2b = block == 16 ? 4 : block == 32 ? 5 : 6, P.splits = n_splits;
  P.causal = causal, P.shares = 0;
  const bool tiled = item_rows == kTileRows;
  P.item_rows = item_rows, P.tile = tiled ? tile_positions(D) : kTile;
  // (requests of several lengths: splits of a multiple of 512 positions, or 256 where the call asks for that many of
  // the table's width, so that the long requests' splits are not much longer than the others', and a short one is not
  // split: 8 x 20 heads (D 64), 448 ragged queries over 1,500 ragged positions 52.5 -> 45.5 us)
  const int grain = (int64_t)max_blocks * block <= (int64_t)n_splits * 256 ? 256 : 512;
  P.least = !tiled ? kWaves : grain / P.tile;
  P.single = 0;
  const int st = check(P, Hq, D, block, code, q_type, out_type);
  if (st != KVT_OK) return st;
  if (!cu_q || n_q < 0 || (item_rows != 16 && !tiled) || (n_splits > 1 && (!part_o || !part_ml))) return KVT_EINVAL;
  if (n_q == 0) return KVT_OK;
  const int64_t items = (int64_t)n_q * P.gs / item_rows + n;
  if (items > (tiled ? 0xFFFFFF / P.H : 65535) || (n_splits > 1 && items * P.H > 65535)) return KVT_ERANGE;
  if (tiled) {
    if (n == 1) P.single = (int)(((int64_t)n_q * P.gs + kTileRows - 1) / kTileRows * P.H);
    tile_launch(P, code, q_type, D, (int)items, out_type, (hipStream_t)stream);
    if (n_splits > 1) {
      if (D == 64) merge<64>(P, (int)items, kTileRows, out_type, (hipStream_t)stream);
      else if (D == 128) merge<128>(P, (int)items, kTileRows, out_type, (hipStream_t)stream);
      else merge<256>(P, (int)items, kTileRows, out_type, (hipStream_t)stream);
    }
  } else {
    launch_all(P, code, q_type, D, (int)items, out_type, (hipStream_t)stream);
  }
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}
