// Quantizing write of a step's K/V rows into 8-bit blocks with one scale per (block, KV head) and side
// (kvt_block_store).
//
// With a = max |x| over the rows that the call writes into a block (finite ones), need = the smallest power of two with
// a / need <= Q (448 for e4m3, 127 for int8), within 2^-64 .. 2^122:
//   s    = need where the call opens the block, else max(need, s_old) (an s_old that is not finite stays)
//   old codes (rows that the request held in the block) -> rne(code * s_old / s) where s grew
//   new codes = rne(x / s)
// Powers of two, because a block fills up over many calls: x / s is exact, a growing scale moves the exponent of an
// e4m3 code and rounds nothing but subnormals (with s = a / Q every growth would round every code again), and the
// readers' products with the scale are exact.  The price is up to one bit of int8's range.
//
// Bytes bound it: the rows are read once and the codes written once.  An item is a (request's block, KV head, side): a
// request's tokens are consecutive, so a cache block is written by one workgroup or wavefront and its maximum needs no
// atomics.  Which (request, block) an item is follows from the prefix sums of the token counts (find_request).  A
// thread keeps its eight channels of NP rows as they are in memory between the maximum and the codes.  32,000 rows of
// 1,024 channels (197 MB of bf16 or fp16 rows and codes) take 38 - 41 us for every block size and head length, 4.8 -
// 5.2 TB/s, a large copy's rate; fp32 rows (328 MB) 62 - 65.
//
// Up to 4,096 values a block an item is a wavefront, and a workgroup takes four heads of a block, whose rows are side
// by side in memory; more values need the registers of four wavefronts.  With 256 threads for every item, heads apart:
// blocks of 16 x 64 101 us, 16 x 128 59, 64 x 256 53.  Heads before blocks in the grid's order, for the same reason.
// Magnitudes are compared as bits, two at a time, and finite rows are converted without clamps: int8 from fp16 38 us,
// with three instructions per value for the maximum and a clamp 51.
//
// Calls of a few rows per request (decode steps) take a wavefront per item and a loop over its rows, read twice: 256
// requests x 8 heads, blocks of 64 x 128, one row each 5.8 us against 12.9 with 256 threads, four rows 6.6 / 12.9; 32 x
// 2 heads (64 x 256) 3.4 / 3.6.  From eight rows on a request writes more than the loop's lanes hold, and blocks of 16
// gain nothing (6.2 / 6.0).
#include "block_common.h"

using namespace kvt;
using namespace kvt::blk;

namespace {

constexpr int kFewRows = 4;            // rows per request, on average, up to which a call takes the loop

struct Store {
  const void* x[2];            // K, V rows [N, H, D]
  int64_t sn[2], sh[2];        // element strides of token and head
  uint8_t* codes[2];
  float* scale[2];
  const int32_t* cu;
  const int32_t* kv_lens;
  const int32_t* table;
  const int32_t* rows;         // table row of a request (NULL: its number)
  int64_t stride;
  int n, n_rows, n_tokens, H, n_blocks, max_blocks, log2b;
};

// Eight elements of a row as they are in memory: packed pairs of 16 bits, or fp32.
template <int DT> struct Raw {
  static constexpr int N = DT == kF32 ? 8 : 4;
  uint32_t w[N];
};
template <int DT>
KVT_DEV Raw<DT> load8(const void* base, int64_t at) {
  Raw<DT> r;
#pragma unroll
  for (int i = 0; i < Raw<DT>::N; i += 4) {
    const u4v a = *reinterpret_cast<const u4v*>((const char*)base + at * (DT == kF32 ? 4 : 2) + 4 * i);
    r.w[i] = a.x, r.w[i + 1] = a.y, r.w[i + 2] = a.z, r.w[i + 3] = a.w;
  }
  return r;
}
template <int DT>
KVT_DEV float elem(const Raw<DT>& r, int i) {
  if constexpr (DT == kF32) return __uint_as_float(r.w[i]);
  const uint32_t w = r.w[i >> 1];
  if constexpr (DT == kBF16) return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
  return (float)as_h2(w)[i & 1];
}

// Magnitudes are ordered as their bits are (NaN above infinity): the largest one's bits, two at a time where they are
// 16.
typedef uint16_t us2 __attribute__((ext_vector_type(2)));
template <int DT> constexpr uint32_t kInfBits = DT == kBF16 ? 0x7F80u : DT == kF16 ? 0x7C00u : 0x7F800000u;
template <int DT>
KVT_DEV uint32_t top(uint32_t t, uint32_t w) {
  if constexpr (DT == kF32) return max(t, w & 0x7FFFFFFFu);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, t),
                                                                __builtin_bit_cast(us2, w & 0x7FFF7FFFu)));
}
template <int DT>
KVT_DEV float magnitude(uint32_t bits) {            // (of one element)
  if constexpr (DT == kF32) return __uint_as_float(bits);
  if constexpr (DT == kBF16) return __uint_as_float(bits << 16);
  return f16_bits_to_f32((uint16_t)bits);
}

KVT_DEV uint32_t group_umax(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, 64));
  return v;
}

// Codes of finite x, which are in range (|x * inv| <= 448 or 127; the largest fp32 is less than 127 * 2^122): no clamp.
// int8: the sum with 1.5 * 2^23 is rounded to an integer, to even, whose low byte is the code.
template <int CODE>
KVT_DEV uint32_t pack4_plain(float a, float b, float c, float d, float inv) {
  if constexpr (CODE == kE4M3) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
  } else {
    constexpr float k = 12582912.0f;
    const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(fmaf(b, inv, k)), __float_as_uint(fmaf(a, inv, k)), 0x0C0C0400u);
    return lo | __builtin_amdgcn_perm(__float_as_uint(fmaf(d, inv, k)), __float_as_uint(fmaf(c, inv, k)), 0x04000C0Cu);
  }
}

// T threads per item (64: one wavefront, 256 / T heads per workgroup; 256: a workgroup).  NP rows of a thread, kept in
// registers; NP = 0: any number, each read twice.
template <int DT, int CODE, int D, int T, int NP>
__global__ __launch_bounds__(256) void block_store_kernel(const Store P) {
  constexpr int TPR = D / 8;          // threads per row
  constexpr int RPP = T / TPR;        // rows per pass
  constexpr int HPW = 256 / T;
  __shared__ uint32_t part[4];
  const int B = 1 << P.log2b, side = blockIdx.y;
  const int hg = (P.H + HPW - 1) / HPW;
  const int64_t w = blockIdx.x / hg;
  const int h = uniform((int)(blockIdx.x % hg) * HPW + (T == 64 ? (int)threadIdx.x >> 6 : 0));
  const int r = find_request(P.cu, P.n, w, 1, B, 2);
  const int t0 = min(max(P.cu[r], 0), P.n_tokens), t1 = min(max(P.cu[r + 1], t0), P.n_tokens);
  const int64_t len = P.kv_lens[r], old = len - (t1 - t0);
  const int64_t item = w - first_item(P.cu[r], r, 1, B, 2);
  const int64_t lp = (old >> P.log2b) + item;
  const int row = P.rows ? P.rows[r] : r;
  if (h >= P.H || t1 == t0 || item < 0 || old < 0 || lp * B >= len || lp >= P.max_blocks || row < 0 || row >= P.n_rows) return;
  const int block = P.table[row * P.stride + lp];
  if (block < 0 || block >= P.n_blocks) return;
  const int held = (int)max(old - lp * B, (int64_t)0);              // rows of the block that the request holds already
  const int end = (int)min(len - lp * B, (int64_t)B);
  const int64_t tok = t0 + (lp * B - old);                          // token of the block's row 0 (may lie before t0)
  const int lane = threadIdx.x % T, tr = lane / TPR, ch = 8 * (lane % TPR);
  const int64_t at = (int64_t)block * P.H + h;
  const float was = held ? P.scale[side][at] : 0.0f;

  Raw<DT> x[NP ? NP : 1];
  auto read = [&](int q) { return load8<DT>(P.x[side], (tok + q) * P.sn[side] + h * P.sh[side] + ch); };
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int q = i * RPP + tr;
    if (q >= held && q < end) x[i] = read(q);
    else x[i] = Raw<DT>{};
  }
  auto each = [&](auto f) {                                         // f(row of the block, its elements)
    if constexpr (NP == 0) {
      for (int q = held + tr; q < end; q += RPP) f(q, read(q));
    } else {
#pragma unroll
      for (int i = 0; i < NP; ++i) f(i * RPP + tr, x[i]);
    }
  };
  // the largest magnitude's bits over the item (T == 256: also the barrier before which every thread has read the
  // scale)
  auto widest = [&](uint32_t t) {
    t = group_umax(t);
    if constexpr (T == 256) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = t;
      __syncthreads();
      t = max(max(part[0], part[1]), max(part[2], part[3]));
    }
    return (uint32_t)uniform((int)t);
  };
  uint32_t t = 0;
  each([&](int, const Raw<DT>& v) {
#pragma unroll
    for (int c = 0; c < Raw<DT>::N; ++c) t = top<DT>(t, v.w[c]);
  });
  if constexpr (DT != kF32) t = max(t & 0xFFFFu, t >> 16);
  t = widest(t);
  const bool finite = t < kInfBits<DT>;
  if (!finite) {                                                    // (infinities and NaN set no scale)
    t = 0;
    each([&](int, const Raw<DT>& v) {
#pragma unroll
      for (int c = 0; c < Raw<DT>::N; ++c) {
        const uint32_t u = v.w[c];
        if constexpr (DT == kF32) {
          t = max(t, (u & 0x7FFFFFFFu) < kInfBits<DT> ? u & 0x7FFFFFFFu : 0u);
        } else {
          t = max(t, (u & 0x7FFFu) < kInfBits<DT> ? u & 0x7FFFu : 0u);
          t = max(t, (u >> 16 & 0x7FFFu) < kInfBits<DT> ? u >> 16 & 0x7FFFu : 0u);
        }
      }
    });
    t = widest(t);
  }
  float s = pow2_scale<CODE>(magnitude<DT>(t));
  if (held && !(was <= s)) s = was;                                 // (a NaN stays: the rows held are NaN with it)
  const float inv = 1.0f / s;
  uint8_t* out = P.codes[side] + ((at << P.log2b) * D);
  if (held && s > was) {
    const float f = was * inv;
    for (int i = lane; i < held * (D / 8); i += T) {
      u2v* p = reinterpret_cast<u2v*>(out) + i;
      u2v c = *p;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float y[4];
        unpack4<CODE>(c[k], y);
        c[k] = pack4<CODE>(y[0] * f, y[1] * f, y[2] * f, y[3] * f);
      }
      *p = c;
    }
  }
  if (lane == 0) P.scale[side][at] = s;
  auto write = [&](auto pack) {
    each([&](int q, Raw<DT> v) {
      if (q < held || q >= end) return;
#pragma unroll
      for (int c = 0; c < Raw<DT>::N; ++c) asm volatile("" : "+v"(v.w[c]));   // (converted here, not all rows ahead)
      u2v c;
      c.x = pack(elem<DT>(v, 0), elem<DT>(v, 1), elem<DT>(v, 2), elem<DT>(v, 3));
      c.y = pack(elem<DT>(v, 4), elem<DT>(v, 5), elem<DT>(v, 6), elem<DT>(v, 7));
      *reinterpret_cast<u2v*>(out + q * D + ch) = c;
    });
  };
  if (finite) write([&](float p, float q, float u, float v) { return pack4_plain<CODE>(p, q, u, v, inv); });
  else write([&](float p, float q, float u, float v) { return pack4<CODE>(p * inv, q * inv, u * inv, v * inv); });
}

template <int DT, int CODE, int D, int T, int NP>
int launch(const Store& P, int64_t items, hipStream_t st) {
  constexpr int HPW = 256 / T;
  const int64_t groups = items * ((P.H + HPW - 1) / HPW);
  if (groups >= 1 << 24) return KVT_ERANGE;         // (2^32 threads)
  block_store_kernel<DT, CODE, D, T, NP><<<dim3((uint32_t)groups, 2), 256, 0, st>>>(P);
  return KVT_OK;
}
template <int DT, int CODE, int D>
int launch_b(const Store& P, int64_t items, hipStream_t st) {
  if (P.n_tokens <= kFewRows * P.n) return launch<DT, CODE, D, 64, 0>(P, items, st);
  if (P.log2b == 4) return launch<DT, CODE, D, 64, D / 32>(P, items, st);
  if constexpr (D == 256) {
    if (P.log2b == 5) return launch<DT, CODE, D, 256, 4>(P, items, st);
    return launch<DT, CODE, D, 256, 8>(P, items, st);
  } else {
    if (P.log2b == 5) return launch<DT, CODE, D, 64, D / 16>(P, items, st);
    if constexpr (D == 128) return launch<DT, CODE, D, 256, 4>(P, items, st);
    else return launch<DT, CODE, D, 64, 8>(P, items, st);
  }
}
template <int DT, int CODE>
int launch_d(const Store& P, int D, int64_t items, hipStream_t st) {
  if (D == 64) return launch_b<DT, CODE, 64>(P, items, st);
  if (D == 128) return launch_b<DT, CODE, 128>(P, items, st);
  return launch_b<DT, CODE, 256>(P, items, st);
}
template <int DT>
int launch_c(const Store& P, int code, int D, int64_t items, hipStream_t st) {
  return code == kE4M3 ? launch_d<DT, kE4M3>(P, D, items, st) : launch_d<DT, kI8>(P, D, items, st);
}

}  // namespace

extern "C" int kvt_block_store(const void* k, const void* v, int dtype, int64_t sk_n, int64_t sk_h, int64_t sv_n,
                               int64_t sv_h, int n_tokens, int H, int D, const void* cu, const void* kv_lens, int n,
                               const void* rows, const void* block_table, int64_t bt_stride, int n_rows,
                               int max_blocks, int code, void* k8, void* v8, void* ks, void* vs, int n_blocks,
                               int block, void* stream) {
  if (n < 1 || n > kMaxReq || n_tokens < 0 || H < 1 || n_rows < 1 || max_blocks < 1 || bt_stride < max_blocks ||
      n_blocks < 1 || (!rows && n_rows < n))
    return KVT_EINVAL;
  if ((D != 64 && D != 128 && D != 256) || (block != 16 && block != 32 && block != 64)) return KVT_EINVAL;
  if ((code != kE4M3 && code != kI8) || (dtype != kBF16 && dtype != kF16 && dtype != kF32)) return KVT_EINVAL;
  const int per16 = dtype == kF32 ? 4 : 8;   // 16-byte row loads
  if (((uintptr_t)k | (uintptr_t)v) & 15 || sk_n % per16 || sk_h % per16 || sv_n % per16 || sv_h % per16) return KVT_EINVAL;
  if (((uintptr_t)k8 | (uintptr_t)v8) & 15) return KVT_EINVAL;
  if (H > 65535 || n_tokens > (1 << 30)) return KVT_ERANGE;
  if (n_tokens == 0) return KVT_OK;
  Store P;
  P.x[0] = k, P.x[1] = v, P.sn[0] = sk_n, P.sn[1] = sv_n, P.sh[0] = sk_h, P.sh[1] = sv_h;
  P.codes[0] = (uint8_t*)k8, P.codes[1] = (uint8_t*)v8, P.scale[0] = (float*)ks, P.scale[1] = (float*)vs;
  P.cu = (const int32_t*)cu, P.kv_lens = (const int32_t*)kv_lens, P.table = (const int32_t*)block_table;
  P.rows = (const int32_t*)rows, P.stride = bt_stride;
  P.n = n, P.n_rows = n_rows, P.n_tokens = n_tokens, P.H = H, P.n_blocks = n_blocks, P.max_blocks = max_blocks;
  P.log2b = block == 16 ? 4 : block == 32 ? 5 : 6;
  const int64_t items = n_tokens / block + 2 * n;
  hipStream_t st = (hipStream_t)stream;
  const int rc = dtype == kBF16 ? launch_c<kBF16>(P, code, D, items, st)
                 : dtype == kF16 ? launch_c<kF16>(P, code, D, items, st) : launch_c<kF32>(P, code, D, items, st);
  if (rc != KVT_OK) return rc;
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}
