// Attention weight of a step's queries per cache entry of the 8-bit block cache (kvt_block_weigh).
//
//   out[row, h, p] = prior[row, h, p] + sum over the request's queries i that see p and the q heads g of KV head h of
//                    exp(x_igp - M_ig) / L_ig,   x_igp = scale * sk_p * q_ig . kc_p
// with M and L the maximum and the sum of exponentials of (i, g)'s scores: the column sums of softmax(Q K^T), whose
// rows have to be complete before any column can be.
//
// One query per request (a (request, KV head) has at most 16 rows): the scores are formed once, by 16 x 16 products
// with K's codes from registers as they were loaded, and kept as fp32; a second launch joins the splits' maxima and sums
// and adds up the columns.  With gs q heads a KV head they are 8 gs bytes an entry, written and read back, against D bytes
// of codes for a second read of K: less up to gs 8 at D 64 and 16 at D 128, where they are as much; twice as much at D 64
// with gs 16, which is served alike.  Bytes bound both: 32 requests x 2 heads, D 256, up to 16,384 entries (103 MB of codes,
// 19 MB of scores written and read) 31 + 9 us; int8, 64 x 8 heads, D 128, blocks of 16 (195 + 49 MB) 60 + 17, 4.1 TB/s;
// 32 requests of 8,000, 4 heads of gs 8, D 64 (66 MB of codes, 33 of scores) 32 together.  (Tiles of 64 positions a
// wavefront instead of 32: 57 -> 64; of 16: 59.)
//
// Chunks: a row has too many scores to keep, so they are formed twice.  The first launch holds 256 rows of Q in
// registers (64 a wavefront) and streams K through LDS for maxima and sums; each lane keeps them for a row of its own,
// over the positions that it sees, so that nothing crosses lanes in the loop.  The second one holds 256 positions of K
// in registers and streams Q; a lane adds up the weights of its position.  Splits are joined in their order by launches
// of their own: no atomics, the same bits for every call.  64 rows (positions) a wavefront, which halve the reads of the
// streamed tile against 32, are about what 256 registers hold at D 256 with two wavefronts a SIMD, and 168 at D 128 with
// three: the second kernel spills two registers at both (four with int8 and fp16).  A prompt of 10,001 tokens, 16 / 2
// heads, D 256 (410 GFLOP a launch): 424 + 488 us, 967 and 840 TFLOP/s (a large library product 1,241); the steps
// there: 856 + 1,405 with one wavefront a SIMD, 64-bit divisions for the rows and masks for every tile; 497 + 541
// without the first two; 460 + 495 with operands read ahead of their products and Q copied straight to LDS; 429 with
// masks by wavefront.  Vector instructions (6.5 and 7.4 a product at D 256, 13 at D 128, exponentials at a quarter of
// the rate among them) take about as long as the products at D 256, and more than twice as long at D 128: they bound it
// there and at D 64.
//
// Operands have q's type (codes of 8 bits are exact in bf16 and fp16); scores, maxima, sums and weights are fp32.
#include <type_traits>

#include "block_common.h"

using namespace kvt;
using namespace kvt::blk;

namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f16v __attribute__((ext_vector_type(16)));

constexpr float kInf = __builtin_inff();
constexpr int kTileRows = 256;         // rows (query, q head) of a workgroup of the first chunk launch
constexpr int kTilePos = 256;          // positions of a workgroup's step of the second one
constexpr int kStep = 64;              // positions (rows) of a streamed tile
constexpr int kMostSplits = 1024;
constexpr int64_t kMostPositions = ((int64_t)1 << 31) - 8192;

struct Weigh {
  const void* q;
  const uint8_t* k8;
  const float* ks;
  const int32_t* table;
  const int32_t* kv_lens;
  const int32_t* rows;
  const int32_t* cu;           // NULL: one query per request
  const int32_t* since;        // entries from here on start from zero (NULL: those of the call's queries)
  const float* prior;
  float* out;
  float* scores;               // decode: [n * H, gs, cap]
  float2* part;                // (maximum, sum): decode [n * H, splits, 16]; chunks [splits, H, n_q * gs]
  float2* norm;                // chunks: (maximum, 1 / sum) [H, n_q * gs]
  float* sums;                 // chunks: [row_splits, n * H, cap]
  int64_t sq_n, sq_h, stride, sw_r, sw_h, so_r, so_h;
  float scale_log2;
  uint32_t per_gs;             // ceil(2^31 / gs): row / gs is the high half of a product, exact for rows below 2^27
  int n, n_rows, n_q, H, gs, n_blocks, max_blocks, log2b, splits, row_splits, groups;
  int fit, most;               // chunks: workgroups that the chip holds at once, and of a launch, about
};

KVT_DEV float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
KVT_DEV float lane_f(float v, int lane) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}

// Two codes (bytes 0, 1 or 2, 3 of a dword) -> two operand halves, exact.
template <int CODE, int QT, bool HI>
KVT_DEV uint32_t two(uint32_t w) {
  if constexpr (QT == kF16) {
    return __builtin_bit_cast(uint32_t, pair<CODE, HI>(w));
  } else if constexpr (CODE == kE4M3) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  } else {
    return bf16x2((float)(int8_t)(w >> (HI ? 16 : 0)), (float)(int8_t)(w >> (HI ? 24 : 8)));
  }
}
// Eight codes in order -> an operand.
template <int CODE, int QT>
KVT_DEV u4v eight(uint32_t w0, uint32_t w1) {
  if constexpr (QT == kF16) w0 = flip<CODE>(w0), w1 = flip<CODE>(w1);
  return u4v{two<CODE, QT, false>(w0), two<CODE, QT, true>(w0), two<CODE, QT, false>(w1), two<CODE, QT, true>(w1)};
}
template <int QT>
KVT_DEV f4 mfma16(u4v a, u4v b, f4 c) {
  if constexpr (QT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
template <int QT>
KVT_DEV f16v mfma32(u4v a, u4v b, f16v c) {
  if constexpr (QT == kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}

// K's scale times the softmax scale in powers of two; NaN for a scale that is not finite (>= 0).
KVT_DEV float factor(const Weigh& P, float sk) { return fmaf(P.scale_log2, sk, sk - sk); }

KVT_DEV int query_of(const Weigh& P, int row) { return (int)__umulhi((uint32_t)row << 1, P.per_gs); }

struct Req {
  int trow, q0, q_len, kv, len;      // table row, first query, queries, entries, entries of the table
};
KVT_DEV Req request(const Weigh& P, int r) {
  Req t;
  t.q0 = r, t.q_len = 1;
  if (P.cu) {
    t.q0 = min(max(uniform(P.cu[r]), 0), P.n_q);
    t.q_len = min(max(uniform(P.cu[r + 1]), t.q0), P.n_q) - t.q0;
  }
  t.trow = P.rows ? uniform(P.rows[r]) : r;
  t.kv = max(uniform(P.kv_lens[r]), 0);
  t.len = (int)min((int64_t)t.kv, (int64_t)P.max_blocks << P.log2b);
  if (t.trow < 0 || t.trow >= P.n_rows) t.len = 0, t.trow = 0;
  return t;
}
// Element offset of the q row of the request's row (query, q head of KV head h).
KVT_DEV int64_t q_offset(const Weigh& P, const Req& t, int h, int row) {
  const int i = query_of(P, row);
  return (int64_t)(t.q0 + i) * P.sq_n + (int64_t)(h * P.gs + row - i * P.gs) * P.sq_h;
}
// Entries that query i of the request sees.
KVT_DEV int sees(const Req& t, int i) {
  return (int)min((int64_t)t.len, max((int64_t)t.kv - t.q_len + i + 1, (int64_t)0));
}

// The request, KV head and part of a workgroup.  Parts that a request has no use for are the last ones, so parts are the
// slow index: the workgroups at work are the first ones, on all CUs alike (the hardware deals them out in turn; with
// parts as the fast index 32 short requests in a wide table ran on 2 CUs of 32: 25 us against 13).  With 8 heads, or a
// multiple, every XCD has a head of each request, whose scores stay in its L2; otherwise the pairs move on by one from part
// to part, so that a long request is not all on one or two XCDs (32 ragged requests x 2 heads 41 us, 48 without; 16 x 8
// pairs of 2,000 entries 16.6 us with it, 15.4 without).
struct Part { int r, h, k; };
KVT_DEV Part part_of(const Weigh& P) {
  const int pairs = P.n * P.H, k = blockIdx.x / pairs;
  const int pair = ((int)blockIdx.x - k * pairs + (P.H % 8 ? k : 0)) % pairs;
  return {uniform(pair / P.H), uniform(pair % P.H), uniform(k)};
}

// x and its maximum and sum: a running pair takes another one.
KVT_DEV void join(float& m, float& l, float m2, float l2) {
  const float M = fmaxf(m, m2);
  l = (m == -kInf ? l : l * exp2_(m - M)) + (m2 == -kInf ? l2 : l2 * exp2_(m2 - M));
  m = M;
}

KVT_DEV void finish(const Weigh& P, const Req& t, int r, int h, int p, float sum) {
  const int since = P.since ? P.since[r] : t.kv - t.q_len;
  if (p < since) sum += P.prior[t.trow * P.sw_r + h * P.sw_h + p];
  P.out[t.trow * P.so_r + h * P.so_h + p] = sum;
}

// ------------------------------------------------------------------------------------------- one query per request
// Positions per split: equal shares in multiples of 128 (a tile of 32 for each wavefront), 256 at least.
KVT_DEV int per_split(int len, int splits) { return max(((len + splits - 1) / splits + 127) & ~127, 256); }

template <int CODE, int QT, int D>
__global__ __launch_bounds__(256) void weigh_rows_kernel(const Weigh P) {
  constexpr int NC = D / 64;
  __shared__ float2 J[4][16];
  __shared__ u4v Qs[D / 32][64];
  const auto [r, h, split] = part_of(P);
  const Req t = request(P, r);
  const int per = per_split(t.len, P.splits);
  const int64_t from = (int64_t)split * per;
  if (from >= t.len) return;
  const int p_begin = (int)from, p_end = (int)min(from + per, (int64_t)t.len);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 15, g = lane >> 4;
  const bool live = l < P.gs;
  const uint16_t* qrow = (const uint16_t*)P.q + (int64_t)t.q0 * P.sq_n + (int64_t)(h * P.gs + (live ? l : 0)) * P.sq_h;
  if (wave == 0) {
#pragma unroll
    for (int k = 0; k < D / 32; ++k)
      Qs[k][lane] = *reinterpret_cast<const u4v*>(qrow + 64 * (k >> 1) + 16 * g + 8 * (k & 1));
  }
  const int64_t pair_id = (int64_t)r * P.H + h, cap = (int64_t)P.max_blocks << P.log2b;
  float* score = P.scores + (pair_id * P.gs + l) * cap;
  const uint32_t koff = (uint32_t)l * D + 16u * g;
  const int64_t tbl = (int64_t)t.trow * P.stride;
  float m = -kInf, sum = 0.0f;
  __syncthreads();

  for (int base = p_begin + 32 * wave; base < p_end; base += 32 * 128) {
    // blocks and scales of the next 32 tiles: lane 2 i + s has half s of the tile at base + 128 i
    int id = -1;
    float sk = 0.0f;
    const int mine = base + (lane >> 1) * 128 + 16 * (lane & 1);
    if (mine < p_end) id = P.table[tbl + (mine >> P.log2b)];
    if (id < 0 || id >= P.n_blocks) id = -1;
    if (id >= 0) sk = P.ks[(int64_t)id * P.H + h];
    for (int i = 0; i < 32; ++i) {
      const int p0 = base + 128 * i;
      if (p0 >= p_end) break;
      int valid[2];
      float f[2];
      u4v kr[2][NC];
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const int b = __builtin_amdgcn_readlane(id, 2 * i + s);
        const int64_t at = ((((int64_t)max(b, 0) * P.H + h) << P.log2b) + ((p0 + 16 * s) & ((1 << P.log2b) - 1))) * D;
        f[s] = factor(P, lane_f(sk, 2 * i + s));
        valid[s] = b < 0 ? 0 : min(max(p_end - (p0 + 16 * s), 0), 16);
#pragma unroll
        for (int c = 0; c < NC; ++c) kr[s][c] = *reinterpret_cast<const u4v*>(P.k8 + at + koff + 64u * c);
      }
      float x[2][4];
      f4 accs[2] = {};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const u4v q0 = Qs[2 * c][lane], q1 = Qs[2 * c + 1][lane];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          accs[s] = mfma16<QT>(eight<CODE, QT>(kr[s][c][0], kr[s][c][1]), q0, accs[s]);
          accs[s] = mfma16<QT>(eight<CODE, QT>(kr[s][c][2], kr[s][c][3]), q1, accs[s]);
        }
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const f4 acc = accs[s];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[s][j] = 4 * g + j < valid[s] ? acc[j] * f[s] : -kInf;
        if (live && p0 + 16 * s < p_end)
          *reinterpret_cast<f4*>(score + p0 + 16 * s + 4 * g) = f4{x[s][0], x[s][1], x[s][2], x[s][3]};
      }
      float top = m;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) top = fmaxf(top, x[s][j]);
      const float ref = top == -kInf ? 0.0f : top;
      sum *= exp2_(m - ref);
      m = top;
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += exp2_(x[s][j] - ref);
    }
  }
  const float M = max_xor16_32(m);
  sum = sum_xor16_32(m == -kInf ? sum : sum * exp2_(m - M));
  if (g == 0) J[wave][l] = make_float2(M, sum);
  __syncthreads();
  if (threadIdx.x < 16) {
    float2 a = J[0][l];
#pragma unroll
    for (int v = 1; v < 4; ++v) join(a.x, a.y, J[v][l].x, J[v][l].y);
    P.part[(pair_id * P.splits + split) * 16 + l] = a;
  }
}

// Maximum and 1 / sum of the pair's rows from the splits' parts, then the columns of 1,024 positions at a time, four
// per thread.
__global__ __launch_bounds__(256) void weigh_columns_kernel(const Weigh P) {
  __shared__ float2 J[16][16];
  __shared__ float2 norm[16];
  const auto [r, h, split] = part_of(P);
  const Req t = request(P, r);
  if ((int64_t)split * 1024 >= t.len) return;
  const int64_t pair_id = (int64_t)r * P.H + h, cap = (int64_t)P.max_blocks << P.log2b;
  const int per = per_split(t.len, P.splits), used = (t.len + per - 1) / per;
  const float* scores = P.scores + pair_id * P.gs * cap;
  // four rows' scores of four positions, and the positions' block
  f4 x[4];
  int id = -1;
  auto load = [&](int p, int g) {
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = *reinterpret_cast<const f4*>(scores + min(g + k, P.gs - 1) * cap + p);
  };
  int64_t base = (int64_t)split * 1024;
  const int first = min((int)base + 4 * (int)threadIdx.x, (t.len - 1) & ~3);
  load(first, 0);                                 // (asked for before the parts)
  id = P.table[(int64_t)t.trow * P.stride + (first >> P.log2b)];
  {
    const int l = threadIdx.x & 15, c = threadIdx.x >> 4;
    float m = -kInf, s = 0.0f;
#pragma unroll 4
    for (int i = c; i < used; i += 16) {
      const float2 a = P.part[(pair_id * P.splits + i) * 16 + l];
      join(m, s, a.x, a.y);
    }
    J[c][l] = make_float2(m, s);
  }
  __syncthreads();
  if (threadIdx.x < 16) {
    float2 a = J[0][threadIdx.x];
#pragma unroll
    for (int c = 1; c < 16; ++c) join(a.x, a.y, J[c][threadIdx.x].x, J[c][threadIdx.x].y);
    // (rows behind the last one: nothing)
    norm[threadIdx.x] = (int)threadIdx.x < P.gs ? make_float2(a.x, 1.0f / a.y) : make_float2(kInf, 0.0f);
  }
  __syncthreads();
  for (bool again = false; base < t.len; base += (int64_t)P.groups * 1024, again = true) {
    const int p = (int)base + 4 * threadIdx.x;
    if (p >= t.len) break;
    if (again) {
      load(p, 0);
      id = P.table[(int64_t)t.trow * P.stride + (p >> P.log2b)];      // (four positions of one block)
    }
    float sum[4] = {0, 0, 0, 0};
    for (int g = 0; g < P.gs; g += 4) {
      if (g) load(p, g);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 a = norm[g + k];
        if (g + k < P.gs)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] = fmaf(exp2_(x[k][i] - a.x), a.y, sum[i]);
      }
    }
    const bool there = id >= 0 && id < P.n_blocks;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + i < t.len) finish(P, t, r, h, p + i, there ? sum[i] : 0.0f);
  }
}

// ------------------------------------------------------------------------------------------------------------- chunks
// A streamed tile in LDS: kStep rows of D halves, padded so that 32 rows' 16-byte reads spread over the banks.
template <int D> constexpr int kPitch = 2 * D + 16;

// Operand k of a streamed row: with a held operand whose lanes have 16 codes in a row (K in registers), channels
// 32 k' + 16 hl + 8 (k & 1); else 16 k + 8 hl.
template <bool SIXTEEN>
KVT_DEV int channel(int k, int hl) { return SIXTEEN ? 32 * (k >> 1) + 16 * hl + 8 * (k & 1) : 16 * k + 8 * hl; }

// BYTES per lane from each lane's address into lds + BYTES * lane.  The caller waits: vmcnt(0) and a barrier.
template <int BYTES>
KVT_DEV void copy_to_lds(const void* from, void* lds) {
  const auto* g = (const __attribute__((address_space(1))) void*)from;
  auto* l = (__attribute__((address_space(3))) void*)lds;
  if constexpr (BYTES == 16) __builtin_amdgcn_global_load_lds(g, l, 16, 0, 0);
  else __builtin_amdgcn_global_load_lds(g, l, 4, 0, 0);
}

// The products of a streamed tile of 32 rows, whose operand k is read(k), with two held ones: operands are read a batch
// ahead of their products.  (By itself the compiler reads each one into the registers of the last, and every two
// products wait for LDS.)
template <int QT, int KS, class Read>
KVT_DEV void products(Read read, const u4v (&held)[2][KS], f16v (&acc)[2]) {
  constexpr int N = KS > 4 ? 2 : 4;           // (registers)
  u4v a[2][N];
#pragma unroll
  for (int i = 0; i < N; ++i) a[0][i] = read(i);
#pragma unroll
  for (int b = 0; b < KS / N; ++b) {
    if (b + 1 < KS / N) {
#pragma unroll
      for (int i = 0; i < N; ++i) a[(b + 1) & 1][i] = read(N * (b + 1) + i);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) acc[c] = mfma32<QT>(a[b & 1][i], held[c][N * b + i], acc[c]);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// Row (of 32) that register i of a 32 x 32 product has in lanes of half hl.
KVT_DEV int prow(int i, int hl) { return 8 * (i >> 2) + 4 * hl + (i & 3); }

// The host knows the table's width only, which a short request does not fill: how an item's positions, and a request's
// rows, are divided follows from its own lengths, within what the launch has.
//
// Positions of a split of an item whose rows see `limit`: splits of 512 at least, or smaller ones, of 128 at least, as
// long as the launch does not fill the chip.
constexpr int kLeast = 9;
KVT_DEV int per_norm_split(const Weigh& P, int limit, int items) {
  const int many = max(P.fit / (items * P.H), limit >> kLeast), used = max(min(min(many, P.splits), (limit + 127) >> 7), 1);
  return max(((limit + kStep - 1) / kStep + used - 1) / used, 1) * kStep;
}

// Maxima and sums of 256 rows over a split of the positions.  (The reference in the place of the running maximum: 52 of
// some 290 vector instructions per 64 x 64 scores less, 429 -> 411 us.)
template <int CODE, int QT, int D>
__global__ __launch_bounds__(256, 2) void weigh_norm_kernel(const Weigh P, int items) {
  constexpr int KS = D / 16, NL = D / 64;     // products per tile of 32; 16-byte loads per thread and tile
  constexpr int TPR = D / 16;                 // threads per streamed row
  __shared__ __attribute__((aligned(16))) uint8_t tile[2][kStep * kPitch<D>];
  // (the last items see the most: they begin first)
  const int item = items - 1 - blockIdx.x % items, w = blockIdx.x / items, h = w % P.H, split = w / P.H;
  const int r = find_request(P.cu, P.n, item, P.gs, kTileRows, 1);
  const Req t = request(P, r);
  const int64_t begin = (item - first_item(uniform(P.cu[r]), r, P.gs, kTileRows, 1)) * kTileRows;
  const int n_rows = t.q_len * P.gs;
  if (begin < 0 || begin >= n_rows) return;
  const int row0 = (int)begin, live = min(n_rows - row0, kTileRows);
  const int limit = sees(t, query_of(P, row0 + live - 1));
  const int per = per_norm_split(P, limit, items);
  if (split > 0 && (int64_t)split * per >= limit) return;
  const int p_begin = (int)min((int64_t)split * per, (int64_t)limit);
  const int p_end = (int)min((int64_t)p_begin + per, (int64_t)limit);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l = lane & 31, hl = lane >> 5;

  u4v Q[2][KS];
  int see[2];
  float m[2] = {-kInf, -kInf}, sum[2] = {0, 0};
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int mine = 64 * wave + 32 * c + l, row = row0 + (mine < live ? mine : 0);
    see[c] = sees(t, query_of(P, row));
    const uint16_t* p = (const uint16_t*)P.q + q_offset(P, t, h, row);
#pragma unroll
    for (int k = 0; k < KS; ++k) Q[c][k] = *reinterpret_cast<const u4v*>(p + channel<false>(k, hl));
  }
  // what all of the wavefront's rows see, and any of them
  const bool idle = 64 * wave >= live;
  const int all_see = idle ? 0 : uniform(sees(t, query_of(P, row0 + 64 * wave)));
  const int any_see = idle ? 0 : uniform(sees(t, query_of(P, row0 + min(64 * wave + 63, live - 1))));
  const int64_t tbl = (int64_t)t.trow * P.stride;

  int id = -1;
  float sk = 0.0f;
  // blocks and scales of the next 16 tiles: lane 4 i + s has quarter s of tile base / 64 + i
  auto ids = [&](int base) {
    const int p = base + 16 * lane;
    id = p < p_end ? P.table[tbl + (p >> P.log2b)] : -1;
    if (id < 0 || id >= P.n_blocks) id = -1;
    sk = id >= 0 ? P.ks[(int64_t)id * P.H + h] : 0.0f;
  };
  u4v raw[NL];
  const int tr = threadIdx.x / TPR, tc = threadIdx.x % TPR;
  auto load = [&](int p0, int i) {
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      const int row = tr + k * (256 / TPR);             // (a wavefront's rows are of one quarter)
      const int b = max(__builtin_amdgcn_readlane(id, 4 * i + uniform(row >> 4)), 0);
      raw[k] = *reinterpret_cast<const u4v*>(
          P.k8 + ((((int64_t)b * P.H + h) << P.log2b) + ((p0 + row) & ((1 << P.log2b) - 1))) * D + 16 * tc);
    }
  };
  if (p_begin < p_end) {
    ids(p_begin);
    load(p_begin, 0);
  }
  int buf = 0, slot = 0;
  for (int p0 = p_begin; p0 < p_end; p0 += kStep, buf ^= 1) {
    uint8_t* T = tile[buf];
#pragma unroll
    for (int k = 0; k < NL; ++k) {
      u4v* o = reinterpret_cast<u4v*>(T + (tr + k * (256 / TPR)) * kPitch<D> + 32 * tc);
      o[0] = eight<CODE, QT>(raw[k][0], raw[k][1]);
      o[1] = eight<CODE, QT>(raw[k][2], raw[k][3]);
    }
    float f[4];
    int valid[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      f[s] = factor(P, lane_f(sk, 4 * slot + s));
      valid[s] = __builtin_amdgcn_readlane(id, 4 * slot + s) < 0 ? 0 : min(max(p_end - (p0 + 16 * s), 0), 16);
    }
    const bool edge = valid[0] + valid[1] + valid[2] + valid[3] < kStep || p0 + kStep > all_see;
    ++slot;
    if (p0 + kStep < p_end) {
      if (slot == 16) ids(p0 + kStep), slot = 0;
      load(p0 + kStep, slot);
    }
    __syncthreads();
    auto take = [&](auto masked) {
      constexpr bool EDGE = decltype(masked)::value;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        f16v acc[2] = {};
        products<QT, KS>(
            [&](int k) {
              return *reinterpret_cast<const u4v*>(T + (32 * s + l) * kPitch<D> + 2 * channel<false>(k, hl));
            }, Q, acc);
        float f0 = f[2 * s], f1 = f[2 * s + 1];
        if constexpr (EDGE) {
#pragma unroll
          for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const int at = prow(i, hl);
              const bool is = (at & 15) < valid[2 * s + (i >> 3)] && p0 + 32 * s + at < see[c];
              acc[c][i] = is ? acc[c][i] * (i < 8 ? f0 : f1) : -kInf;
            }
          f0 = f1 = 1.0f;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          auto exps = [&](float ref) {
            float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              s0 += exp2_(fmaf(acc[c][i], f0, -ref));
              s1 += exp2_(fmaf(acc[c][8 + i], f1, -ref));
            }
            return s0 + s1;
          };
          // The reference m need not be the maximum: it stays while no sum leaves 2^90 (-inf at first: no sum is a
          // number)
          float more = EDGE ? kInf : exps(m[c]);
          if (EDGE || __any(!(more <= 0x1p90f))) {
            // (scales are >= 0: the largest score of a block is its largest product's)
            float t0 = acc[c][0], t1 = acc[c][8];
#pragma unroll
            for (int i = 1; i < 8; ++i) t0 = fmaxf(t0, acc[c][i]), t1 = fmaxf(t1, acc[c][8 + i]);
            const float top = fmaxf(m[c], fmaxf(t0 * f0, t1 * f1)), ref = top == -kInf ? 0.0f : top;
            more = exps(ref);
            sum[c] *= exp2_(m[c] - ref);
            m[c] = top;
          }
          sum[c] += more;
        }
      }
    };
    if (p0 < any_see) {
      if (__builtin_expect(edge, 0)) {
        asm volatile("");                     // (a branch: without it the masks are computed for every tile)
        take(std::true_type{});
      } else {
        take(std::false_type{});
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const float m2 = __shfl_xor(m[c], 32, 64), s2 = __shfl_xor(sum[c], 32, 64);
    join(m[c], sum[c], m2, s2);
    const int mine = 64 * wave + 32 * c + l;
    if (hl == 0 && mine < live) {
      const int64_t at = ((int64_t)h * P.n_q + t.q0) * P.gs + row0 + mine;
      // (for the join: how many parts the row has)
      if (split == 0)
        P.norm[at] = P.splits == 1 ? make_float2(m[c], 1.0f / sum[c]) : make_float2(__int_as_float((limit + per - 1) / per), 0);
      if (P.splits > 1) P.part[split * ((int64_t)P.H * P.n_q * P.gs) + at] = make_float2(m[c], sum[c]);
    }
  }
}

// Joins the splits' maxima and sums: LANES lanes per row.
template <int LANES>
__global__ __launch_bounds__(256) void weigh_join_kernel(const Weigh P) {
  constexpr int R = 64 / LANES;               // rows of a wavefront
  const int per_head = P.n_q * P.gs, h = blockIdx.y, lane = threadIdx.x & 63;
  const int i = blockIdx.x * 4 * R + (threadIdx.x >> 6) * R + lane % R;
  const int64_t total = (int64_t)P.H * per_head, at = (int64_t)h * per_head + i;
  const bool is = i < per_head && query_of(P, i) < P.cu[P.n];      // (padding has no parts)
  float m = -kInf, s = 0.0f;
  if (is) {
    const int parts = min(max(__float_as_int(P.norm[at].x), 1), P.splits);  // (rows of no request: anything)
#pragma unroll 4
    for (int k = lane / R; k < parts; k += LANES) {
      const float2 a = P.part[k * total + at];
      join(m, s, a.x, a.y);
    }
  }
#pragma unroll
  for (int o = R; o < 64; o <<= 1) {
    const float m2 = __shfl_xor(m, o, 64), s2 = __shfl_xor(s, o, 64);
    join(m, s, m2, s2);
  }
  if (is && lane < R) P.norm[at] = make_float2(m, 1.0f / s);
}

// How a request's (positions, rows) are divided over the workgroups that it has per KV head: rows in equal splits of
// multiples of 64, 512 at least, or smaller ones, of 128 at least, as long as the launch does not fill the chip; positions
// in steps of 256 over `groups` workgroups for each of them.
struct Cut { int splits, per, groups; };
KVT_DEV Cut cut(const Weigh& P, const Req& t) {
  const int n_rows = t.q_len * P.gs, tiles = max((t.len + kTilePos - 1) / kTilePos, 1);
  Cut c = {1, max((n_rows + 63) & ~63, 64), min(P.groups, tiles)};
  if (P.row_splits == 1 || n_rows <= 128) return c;
  const int each = (int)min((int64_t)P.n * P.H * tiles, (int64_t)1 << 30);        // (32-bit divisions)
  const int many = max(P.fit / each, min(P.most / each, n_rows >> kLeast));
  c.splits = max(min(min(many, P.row_splits), P.groups / tiles), 1);
  c.per = max(((n_rows + c.splits - 1) / c.splits + 63) & ~63, 128);
  c.splits = max((n_rows + c.per - 1) / c.per, 1);
  c.groups = min(P.groups / c.splits, tiles);
  return {uniform(c.splits), uniform(c.per), uniform(c.groups)};
}

// Column sums of 256 positions over a split of the request's rows.  Q's tiles are copied to LDS without a detour by
// registers: 16-byte chunk c of row i goes to place c ^ (i & 15) (D 64: & 7), so that a column of chunks is spread over
// the banks.
template <int CODE, int QT, int D>
__global__ __launch_bounds__(256, D == 256 ? 2 : 3) void weigh_sums_kernel(const Weigh P) {
  constexpr int KS = D / 16, NL = D / 32;     // products per tile of 32 rows; 16-byte copies per thread and tile of Q
  constexpr int TPR = D / 8, SW = TPR < 16 ? TPR - 1 : 15;
  // (arrays of their own, and a loop of two steps: the compiler makes a read of one buffer wait for copies into it
  // only)
  __shared__ __attribute__((aligned(16))) uint8_t tile0[kStep * 2 * D], tile1[kStep * 2 * D];
  __shared__ __attribute__((aligned(16))) float2 norms0[kStep], norms1[kStep];
  // (a request's workgroups follow each other, positions first: 16 pairs of 24,000 rows 171 us, with part_of's order 183)
  const int each = P.H * P.groups, r = blockIdx.x / each, mine = blockIdx.x - r * each;
  const Req t = request(P, r);
  const Cut c = cut(P, t);
  const int w = mine / c.groups, split = mine - w * c.groups, h = w % P.H, rs = w / P.H;
  if (rs >= c.splits) return;
  const int n_rows = t.q_len * P.gs, r_begin = min(rs * c.per, n_rows), r_end = min(r_begin + c.per, n_rows);
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), l = lane & 31, hl = lane >> 5;
  const int64_t cap = (int64_t)P.max_blocks << P.log2b;
  const int tr = threadIdx.x / TPR, tc = threadIdx.x % TPR;
  const float2* norm = P.norm + ((int64_t)h * P.n_q + t.q0) * P.gs;
  const int splits = c.splits;
  const int older = t.kv - t.q_len;           // entries before the queries' own (negative: some queries see nothing)
  // the first row that sees position p (the number of rows where none does)
  auto row_of = [&](int64_t p) { return (int)min(max(p - older, (int64_t)0), (int64_t)t.q_len) * P.gs; };

  for (int64_t p0 = (int64_t)split * kTilePos; p0 < t.len; p0 += (int64_t)c.groups * kTilePos) {
    u4v K[2][KS];
    float f[2], sum[2] = {0, 0};
    int first[2];               // the first row that sees the lane's position
    bool there[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int64_t p = p0 + 64 * wave + 32 * c + l;
      const int id = p < t.len ? P.table[(int64_t)t.trow * P.stride + (p >> P.log2b)] : -1;
      there[c] = id >= 0 && id < P.n_blocks;
      f[c] = there[c] ? factor(P, P.ks[(int64_t)id * P.H + h]) : 0.0f;
      first[c] = row_of(p);
      const int64_t row = (((int64_t)(there[c] ? id : 0) * P.H + h) << P.log2b) + (p & ((1 << P.log2b) - 1));
      const uint8_t* kp = P.k8 + row * D + 16 * hl;
#pragma unroll
      for (int k = 0; k < KS / 2; ++k) {
        const u4v v = *reinterpret_cast<const u4v*>(kp + 32 * k);
        K[c][2 * k] = eight<CODE, QT>(v[0], v[1]);
        K[c][2 * k + 1] = eight<CODE, QT>(v[2], v[3]);
      }
    }
    // the first rows that see any of the workgroup's positions, any of the wavefront's, and all of those
    const int64_t pw = p0 + 64 * wave;
    const int begin = max(row_of(p0), r_begin) & ~(kStep - 1);
    const int some = pw < t.len ? row_of(pw) : r_end, all = row_of(min(pw + 64, (int64_t)t.len) - 1);
    auto copy = [&](int r0, uint8_t* tile, float2* norms) {
#pragma unroll
      for (int k = 0; k < NL; ++k) {
        const int at = tr + k * (256 / TPR), row = min(r0 + at, r_end - 1);   // (those behind the last count for nothing)
        const uint16_t* from = (const uint16_t*)P.q + q_offset(P, t, h, row) + 8 * (tc ^ (at & SW));
        copy_to_lds<16>(from, tile + 4096 * k + 1024 * wave);
      }
      if (wave < 2) {
        const float* from = (const float*)(norm + min(r0 + 32 * wave + (lane >> 1), r_end - 1)) + (lane & 1);
        copy_to_lds<4>(from, norms + 32 * wave);
      }
    };
    if (begin < r_end) copy(begin, tile0, norms0);
    auto step = [&](int r0, const uint8_t* T, const float2* norms, uint8_t* next_tile, float2* next_norms) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // (the tile's copies)
      __syncthreads();
      if (r0 + kStep < r_end) copy(r0 + kStep, next_tile, next_norms);
      auto take = [&](auto masked) {
        constexpr bool EDGE = decltype(masked)::value;
        float more[2] = {0, 0};               // (a tile's own sum: long columns lose less)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          f16v acc[2] = {};
          products<QT, KS>(
              [&](int k) {
                const int chunk = channel<true>(k, hl) / 8;
                return *reinterpret_cast<const u4v*>(T + (32 * s + l) * 2 * D + 16 * (chunk ^ (l & SW)));
              }, K, acc);
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const f4 n2 = *reinterpret_cast<const f4*>(norms + 32 * s + prow(i, hl));
            const int row = r0 + 32 * s + prow(i, hl);
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float x = fmaf(acc[c][i + j], f[c], -n2[2 * j]), li = n2[2 * j + 1];
                if constexpr (EDGE) {
                  const bool is = (row + j >= first[c]) & (row + j < r_end);
                  x = is ? x : -kInf, li = is ? li : 0.0f;
                }
                more[c] = fmaf(exp2_(x), li, more[c]);
              }
          }
        }
        sum[0] += more[0], sum[1] += more[1];
      };
      if (r0 + kStep > some) {
        if (__builtin_expect(r0 < all || r0 + kStep > r_end, 0)) {
          asm volatile("");
          take(std::true_type{});
        } else {
          take(std::false_type{});
        }
      }
    };
    for (int r0 = begin; r0 < r_end; r0 += 2 * kStep) {
      step(r0, tile0, norms0, tile1, norms1);
      if (r0 + kStep < r_end) step(r0 + kStep, tile1, norms1, tile0, norms0);
    }
    __syncthreads();            // (the next positions' first tile goes where this one's last may still be read)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int64_t p = p0 + 64 * wave + 32 * c + l;
      float v = sum[c] + __shfl_xor(sum[c], 32, 64);
      if (!there[c]) v = 0.0f;
      if (hl != 0 || p >= t.len) continue;
      if (splits == 1) finish(P, t, r, h, (int)p, v);
      else P.sums[((int64_t)rs * P.n * P.H + (int64_t)r * P.H + h) * cap + p] = v;
    }
  }
}

__global__ __launch_bounds__(256) void weigh_add_kernel(const Weigh P) {
  const auto [r, h, split] = part_of(P);
  const Req t = request(P, r);
  const int used = cut(P, t).splits;
  if (used == 1) return;                      // (done)
  const int64_t cap = (int64_t)P.max_blocks << P.log2b, step = (int64_t)P.n * P.H * cap;
  for (int64_t p = (int64_t)split * 256 + threadIdx.x; p < t.len; p += (int64_t)P.groups * 256) {
    float s = 0.0f;
    for (int k = 0; k < used; ++k) s += P.sums[k * step + ((int64_t)r * P.H + h) * cap + p];
    finish(P, t, r, h, (int)p, s);
  }
}

template <int CODE, int QT, int D>
int launch(Weigh P, int at_once, hipStream_t st) {
  if (!P.cu) {
    // as many requests at once as the workspace holds scores of
    for (int n = P.n; n > 0; n -= P.n) {
      P.n = min(n, at_once);
      weigh_rows_kernel<CODE, QT, D><<<P.n * P.H * P.splits, 256, 0, st>>>(P);
      KVT_CHECK_LAUNCH();
      weigh_columns_kernel<<<P.n * P.H * P.groups, 256, 0, st>>>(P);
      KVT_CHECK_LAUNCH();
      P.q = (const uint16_t*)P.q + P.n * P.sq_n, P.kv_lens += P.n;
      if (P.since) P.since += P.n;
      if (P.rows) {
        P.rows += P.n;
      } else {                                // (request j's row is j)
        P.table += P.n * P.stride, P.prior += P.n * P.sw_r, P.out += P.n * P.so_r, P.n_rows -= P.n;
      }
    }
    return KVT_OK;
  }
  const int items = (int)((int64_t)P.n_q * P.gs / kTileRows) + P.n;
  weigh_norm_kernel<CODE, QT, D><<<items * P.H * P.splits, 256, 0, st>>>(P, items);
  KVT_CHECK_LAUNCH();
  if (P.splits > 1 && P.n_q > 0) {
    const int rows = P.n_q * P.gs;
    if (P.splits <= 8) weigh_join_kernel<4><<<dim3((rows + 63) / 64, P.H), 256, 0, st>>>(P);
    else weigh_join_kernel<32><<<dim3((rows + 7) / 8, P.H), 256, 0, st>>>(P);
    KVT_CHECK_LAUNCH();
  }
  weigh_sums_kernel<CODE, QT, D><<<P.n * P.H * P.groups, 256, 0, st>>>(P);
  KVT_CHECK_LAUNCH();
  if (P.row_splits > 1) {
    weigh_add_kernel<<<P.n * P.H * P.groups, 256, 0, st>>>(P);
    KVT_CHECK_LAUNCH();
  }
  return KVT_OK;
}
template <int CODE, int QT>
int launch_d(const Weigh& P, int D, int at_once, hipStream_t st) {
  return D == 64 ? launch<CODE, QT, 64>(P, at_once, st)
                 : D == 128 ? launch<CODE, QT, 128>(P, at_once, st) : launch<CODE, QT, 256>(P, at_once, st);
}

// Floats of the workspace's parts: scores or norm, part, sums.
struct Space { int64_t scores, part, norm, sums; };
Space space(int n, int n_q, int H, int gs, int64_t cap, bool chunk, int splits, int row_splits) {
  if (!chunk) return {(int64_t)n * H * gs * cap, (int64_t)n * H * splits * 32, 0, 0};
  const int64_t rows = (int64_t)H * n_q * gs;
  return {0, splits > 1 ? splits * rows * 2 : 0, rows * 2, row_splits > 1 ? (int64_t)row_splits * n * H * cap : 0};
}

}  // namespace

extern "C" int kvt_block_weigh(const void* q, int64_t sq_n, int64_t sq_h, int q_type, const void* cu_q, int n_q,
                               const void* kv_lens, int n, int H, int Hq, int D, int code, const void* k8, const void* ks,
                               int n_blocks, int block, const void* block_table, int64_t bt_stride, int n_rows,
                               int max_blocks, const void* rows, float scale, const void* since, const void* weights,
                               int64_t sw_r, int64_t sw_h, void* out, int64_t so_r, int64_t so_h, int splits,
                               int row_splits, int groups, int fit, int most, void* work, int64_t work_floats, void* stream) {
  if (n < 1 || n > kMaxReq || H < 1 || Hq < H || Hq % H || Hq / H > 16 || n_q < 0 || n_blocks < 1 || n_rows < 1 ||
      max_blocks < 1 || bt_stride < max_blocks || (!rows && n_rows < n) || (!cu_q && n_q < n))
    return KVT_EINVAL;
  if ((D != 64 && D != 128 && D != 256) || (block != 16 && block != 32 && block != 64)) return KVT_EINVAL;
  if ((code != kE4M3 && code != kI8) || (q_type != kBF16 && q_type != kF16) || !(scale > 0.0f)) return KVT_EINVAL;
  if (((uintptr_t)q | (uintptr_t)k8 | (uintptr_t)work) & 15 || (sq_n | sq_h) & 7) return KVT_EINVAL;
  if (splits < 1 || splits > kMostSplits || row_splits < 1 || row_splits > kMostSplits || groups < 1 || fit < 0 || most < 0)
    return KVT_EINVAL;
  const int gs = Hq / H;
  const int64_t cap = (int64_t)max_blocks * block;
  if (cap > kMostPositions) return KVT_ERANGE;
  // requests of a launch, and the tiles of rows of a chunk
  const Space one = space(1, n_q, H, gs, cap, false, splits, row_splits);
  const int at_once = cu_q ? n : (int)min((int64_t)n, work_floats / (one.scores + one.part));
  const int64_t items = (int64_t)n_q * gs / kTileRows + n;
  const int64_t top = 1 << 24;                                      // (2^32 threads of a launch)
  if (at_once < 1) return KVT_EINVAL;
  if ((cu_q ? items : (int64_t)at_once) * H * splits >= top || (int64_t)at_once * H * groups >= top ||
      (int64_t)n_q * gs >= top * 8 || H > 65535)
    return KVT_ERANGE;
  const Space s = space(at_once, n_q, H, gs, cap, cu_q != nullptr, splits, row_splits);
  if (s.scores + s.part + s.norm + s.sums > work_floats) return KVT_EINVAL;
  Weigh P;
  P.q = q, P.k8 = (const uint8_t*)k8, P.ks = (const float*)ks, P.table = (const int32_t*)block_table;
  P.kv_lens = (const int32_t*)kv_lens, P.rows = (const int32_t*)rows, P.cu = (const int32_t*)cu_q;
  P.since = (const int32_t*)since, P.prior = (const float*)weights, P.out = (float*)out;
  float* x = (float*)work;
  P.scores = x, P.part = (float2*)(x + s.scores), P.norm = (float2*)(x + s.scores + s.part);
  P.sums = x + s.scores + s.part + s.norm;
  P.sq_n = sq_n, P.sq_h = sq_h, P.stride = bt_stride, P.sw_r = sw_r, P.sw_h = sw_h, P.so_r = so_r, P.so_h = so_h;
  P.scale_log2 = scale * kLog2e;
  P.n = n, P.n_rows = n_rows, P.n_q = n_q, P.H = H, P.gs = gs, P.n_blocks = n_blocks, P.max_blocks = max_blocks;
  P.log2b = block == 16 ? 4 : block == 32 ? 5 : 6;
  P.per_gs = (uint32_t)((((uint64_t)1 << 31) + gs - 1) / gs);
  P.splits = splits, P.row_splits = row_splits, P.groups = groups, P.fit = fit, P.most = most;
  hipStream_t st = (hipStream_t)stream;
  if (code == kE4M3) return q_type == kBF16 ? launch_d<kE4M3, kBF16>(P, D, at_once, st) : launch_d<kE4M3, kF16>(P, D, at_once, st);
  return q_type == kBF16 ? launch_d<kI8, kBF16>(P, D, at_once, st) : launch_d<kI8, kF16>(P, D, at_once, st);
}
