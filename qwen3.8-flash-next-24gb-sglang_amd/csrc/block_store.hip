// Quantizing write of a step's K/V rows into 8-bit blocks with one scale per (block, KV head) and side (kvt_block_store).
//
// With a = max |x| over the rows that the call writes into a block (finite ones), need = the smallest power of two with
// a / need <= Q (448 for e4m3, 127 for int8), within 2^-64 .. 2^122:
//   s    = need where the call opens the block, else max(need, s_old)
//   old codes (rows that the request held in the block) -> rne(code * s_old / s) where s grew
//   new codes = rne(x / s)
// Powers of two, because a block fills up over many calls: x / s is exact, a growing scale moves the exponent of an e4m3
// code and rounds nothing but subnormals (with s = a / Q every growth would round every code again), and the readers'
// products with the scale are exact.  The price is up to one bit of int8's range.
//
// One block of 256 threads per (request's block, KV head, side): a request's tokens are consecutive, so a cache block is
// written by one workgroup and its maximum needs no atomics.  A thread keeps its 8 channels of B / (256 / (D / 8)) rows in
// registers between the maximum and the codes, so the rows are read once.  Which (request, block) a workgroup has
// follows from the prefix sums of the token counts (find_request).
#include "block_common.h"

using namespace kvt;
using namespace kvt::blk;

namespace {

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

// 8 elements at p (16-byte aligned) as fp32
template <int DT>
KVT_DEV void load8(const void* base, int64_t at, float (&x)[8]) {
  if constexpr (DT == kF32) {
    const float4 a = *reinterpret_cast<const float4*>((const float*)base + at);
    const float4 b = *reinterpret_cast<const float4*>((const float*)base + at + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>((const uint16_t*)base + at);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == kBF16) {
        x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      } else {
        x[2 * i] = f16_bits_to_f32((uint16_t)w[i]), x[2 * i + 1] = f16_bits_to_f32((uint16_t)(w[i] >> 16));
      }
    }
  }
}

// NP: rows of a thread (B / rows per pass, at least 1)
template <int DT, int CODE, int D, int NP>
__global__ __launch_bounds__(256) void block_store_kernel(const Store P) {
  constexpr int TPR = D / 8;          // threads per row
  constexpr int RPP = 256 / TPR;      // rows per pass
  __shared__ float part[4];
  const int B = 1 << P.log2b, h = blockIdx.y, side = blockIdx.z;
  const int64_t w = blockIdx.x;
  const int r = find_request(P.cu, P.n, w, 1, B, 2);
  const int t0 = min(max(P.cu[r], 0), P.n_tokens), t1 = min(max(P.cu[r + 1], t0), P.n_tokens);
  const int64_t len = P.kv_lens[r], old = len - (t1 - t0);
  const int64_t item = w - first_item(P.cu[r], r, 1, B, 2);
  const int64_t lp = (old >> P.log2b) + item;
  const int row = P.rows ? P.rows[r] : r;
  if (t1 == t0 || item < 0 || old < 0 || lp * B >= len || lp >= P.max_blocks || row < 0 || row >= P.n_rows) return;
  const int block = P.table[row * P.stride + lp];
  if (block < 0 || block >= P.n_blocks) return;
  const int held = (int)max(old - lp * B, (int64_t)0);              // rows of the block that the request holds already
  const int end = (int)min(len - lp * B, (int64_t)B);
  const int64_t tok = t0 + (lp * B - old);                          // token of the block's row 0 (may lie before t0)
  const int tr = threadIdx.x / TPR, ch = 8 * (threadIdx.x % TPR);

  float x[NP][8], a = 0.0f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int q = i * RPP + tr;
    if (q >= held && q < end) {
      load8<DT>(P.x[side], (tok + q) * P.sn[side] + h * P.sh[side] + ch, x[i]);
    } else {
#pragma unroll
      for (int c = 0; c < 8; ++c) x[i][c] = 0.0f;
    }
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const float m = fabsf(x[i][c]);
      a = m < __builtin_inff() ? fmaxf(a, m) : a;                   // (infinities and NaN set no scale)
    }
  }
  a = group_max<64>(a);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = a;
  __syncthreads();
  a = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
  const int64_t at = (int64_t)block * P.H + h;
  float s = pow2_scale<CODE>(a), was = 0.0f;
  if (held) {
    was = P.scale[side][at];
    s = fmaxf(s, was);
  }
  __syncthreads();                                                  // every thread has read the old scale
  const float inv = 1.0f / s;
  uint8_t* out = P.codes[side] + ((at << P.log2b) * D);
  if (held && s > was) {
    const float f = was * inv;
    for (int i = threadIdx.x; i < held * (D / 8); i += 256) {
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
  if (threadIdx.x == 0) P.scale[side][at] = s;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int q = i * RPP + tr;
    if (q >= held && q < end) {
      u2v c;
      c.x = pack4<CODE>(x[i][0] * inv, x[i][1] * inv, x[i][2] * inv, x[i][3] * inv);
      c.y = pack4<CODE>(x[i][4] * inv, x[i][5] * inv, x[i][6] * inv, x[i][7] * inv);
      *reinterpret_cast<u2v*>(out + q * D + ch) = c;
    }
  }
}

template <int DT, int CODE, int D>
void launch(const Store& P, dim3 grid, hipStream_t st) {
  const int np = (1 << P.log2b) * (D / 8) / 256;
  if (np <= 1) block_store_kernel<DT, CODE, D, 1><<<grid, 256, 0, st>>>(P);
  else if (np == 2) block_store_kernel<DT, CODE, D, 2><<<grid, 256, 0, st>>>(P);
  else if (np == 4) block_store_kernel<DT, CODE, D, 4><<<grid, 256, 0, st>>>(P);
  else if constexpr (D == 256) block_store_kernel<DT, CODE, D, 8><<<grid, 256, 0, st>>>(P);
}
template <int DT, int CODE>
void launch_d(const Store& P, int D, dim3 grid, hipStream_t st) {
  if (D == 64) launch<DT, CODE, 64>(P, grid, st);
  else if (D == 128) launch<DT, CODE, 128>(P, grid, st);
  else launch<DT, CODE, 256>(P, grid, st);
}
template <int DT>
void launch_c(const Store& P, int code, int D, dim3 grid, hipStream_t st) {
  if (code == kE4M3) launch_d<DT, kE4M3>(P, D, grid, st);
  else launch_d<DT, kI8>(P, D, grid, st);
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
  const dim3 grid(n_tokens / block + 2 * n, H, 2);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == kBF16) launch_c<kBF16>(P, code, D, grid, st);
  else if (dtype == kF16) launch_c<kF16>(P, code, D, grid, st);
  else launch_c<kF32>(P, code, D, grid, st);
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}
