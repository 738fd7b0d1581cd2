// Rotary positions of a step's queries and keys (kvt_rope).
//
// The first `rot` channels of a head are pairs (a, b): channels (i, i + rot / 2), or (2 i, 2 i + 1) where they are
// interleaved.  With theta = position * inv_freq[i] and a factor c (long-context schemes scale cosine and sine):
//   a' = c (a cos theta - b sin theta),   b' = c (b cos theta + a sin theta)
// -theta gives the transpose, which is the gradient.  Channels from rot on are copied, or left alone in place.
//
// Angles: theta and its fraction of a turn are formed in 64 bits (in 32, position 262,144 at frequency 1 would be off
// by 0.02 rad); what remains, within an eighth of a turn, goes through the Taylor series of sine and cosine in 32 bits
// (to x^9 and x^10: the next terms are below 2e-9 for |x| <= pi / 4).  Products are fp32, rounded once.
//
// A workgroup takes one token: its pairs' cosines and sines go to LDS once and serve all heads of q and k.  Bytes bound
// it: every element is read once and written once, 16 bytes a lane (7,115 tokens of 64 + 8 heads x 128, fp16,
// interleaved, out of one projection's output: 262 MB in 46 us, 5.7 TB/s).  64 tokens of 26 heads, a quarter of D 256:
// 5.4 us, launch and load latency.  Where rot / 2 (rot, interleaved), the rows or D are no multiples of 16 bytes, the whole
// head goes by single elements: 4,096 tokens of 26 heads, D 256, rot 20 48 us, rot 64 25 (109 MB); of 40 heads, D 96, rot 24
// 33, rot 48 19 (63 MB).
#include "block_common.h"

using namespace kvt;
using namespace kvt::blk;

namespace {

constexpr int kThreads = 256;

struct Rope {
  const void* x[2];            // q, k [N, heads, D] (k may be missing: no heads)
  void* out[2];
  int64_t sn[2], sh[2], on[2], oh[2];
  const void* positions;
  const double* inv_freq;
  const int32_t* cu;           // NULL: a position per token
  const int32_t* rows;
  const int32_t* ahead;
  float scale;
  int heads[2], copy[2];       // copy: channels behind rot are written too
  int n, n_rows, D, rot, wide, sign;
};

// Rounded value in a type of at most 32 bits.
template <int DT>
KVT_DEV uint32_t store_bits(float v) {
  if constexpr (DT == kBF16) return bf16_rne(v);
  if constexpr (DT == kF16) return f32_to_f16_bits(v);
  return __float_as_uint(v);
}

// E elements in 16 bytes, or one.
template <int DT, bool VEC>
struct Unit {
  static constexpr int SIZE = DT == kF32 ? 4 : 2, E = VEC ? 16 / SIZE : 1;
  float v[E];
  KVT_DEV void load(const char* p) {
    if constexpr (VEC) {
      const u4v w = *reinterpret_cast<const u4v*>(p);
#pragma unroll
      for (int i = 0; i < E; ++i) {
        if constexpr (DT == kF32) v[i] = __uint_as_float(w[i]);
        else if constexpr (DT == kBF16) v[i] = __uint_as_float(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16);
        else v[i] = (float)as_h2(w[i >> 1])[i & 1];
      }
    } else {
      v[0] = load_in<DT>(p, 0);
    }
  }
  KVT_DEV void store(char* p) const {
    if constexpr (VEC) {
      u4v w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (DT == kF32) w[i] = __float_as_uint(v[i]);
        else if constexpr (DT == kBF16) w[i] = bf16x2(v[2 * i], v[2 * i + 1]);
        else w[i] = store_bits<DT>(v[2 * i]) | store_bits<DT>(v[2 * i + 1]) << 16;
      }
      *reinterpret_cast<u4v*>(p) = w;
    } else if constexpr (DT == kF32) {
      *reinterpret_cast<float*>(p) = v[0];
    } else {
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)store_bits<DT>(v[0]);
    }
  }
};

// c cos and c sin of `pos` turns at a frequency.
KVT_DEV float2 turn(double pos, double freq, float c) {
  const double t = pos * freq * 0.15915494309189535;          // (1 / 2 pi)
  const double f = t - rint(t), k = rint(4.0 * f);
  const float x = (float)((f - 0.25 * k) * 6.283185307179586), y = x * x;
  const float s0 = x * fmaf(y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
  const float c4 = fmaf(y, fmaf(y, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720);
  const float c0 = fmaf(y, fmaf(y, fmaf(y, c4, 1.0f / 24), -0.5f), 1.0f);
  const int q = (int)k & 3;
  const float sn = q == 0 ? s0 : q == 1 ? c0 : q == 2 ? -s0 : -c0, cs = q == 0 ? c0 : q == 1 ? -s0 : q == 2 ? -c0 : s0;
  return make_float2(c * cs, c * sn);
}

template <int DT, bool VEC, bool INTER>
__global__ __launch_bounds__(kThreads) void rope_kernel(const Rope P) {
  using U = Unit<DT, VEC>;
  constexpr int E = U::E, SIZE = U::SIZE;
  __shared__ float2 cs[128];
  const int t = blockIdx.x, half = P.rot >> 1;
  int64_t pos;
  if (P.cu) {
    const int r = find_request(P.cu, P.n, t, 1, 1, 0);
    const int t0 = P.cu[r], t1 = P.cu[r + 1];
    const int row = P.rows ? P.rows[r] : r;
    if (t < t0 || t >= t1) return;                            // (padding behind the last request)
    pos = (int64_t)((const int32_t*)P.positions)[r] - (t1 - t);
    if (P.ahead && row >= 0 && row < P.n_rows) pos += P.ahead[row];
  } else {
    pos = P.wide ? ((const int64_t*)P.positions)[t] : ((const int32_t*)P.positions)[t];
  }
  if ((int)threadIdx.x < half) cs[threadIdx.x] = turn((double)(P.sign * pos), P.inv_freq[threadIdx.x], P.scale);
  __syncthreads();

  // units of a head: rotated ones (two places of E channels each, or one where the pairs are side by side and E > 1),
  // then copied ones
  constexpr bool ONE = INTER && VEC;
  const int turned = ONE ? P.rot / E : half / E;
  const int units = turned + (P.copy[0] | P.copy[1] ? (P.D - P.rot) / E : 0);
  const int u = threadIdx.x % units, first = threadIdx.x / units, step = kThreads / units;
  if (first >= step) return;
  const bool turns = u < turned;
  // channel of the unit, and of its second place
  const int at = !turns ? P.rot + (u - turned) * E : ONE ? u * E : INTER ? 2 * u : u * E;
  const int other = INTER ? at + 1 : at + half;
  float2 w[ONE ? (E > 1 ? E / 2 : 1) : E];
  if (turns) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(w) / sizeof(w[0])); ++i) w[i] = cs[ONE ? at / 2 + i : u * E + i];
  }
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    if (!turns && !P.copy[side]) continue;
    const char* in = (const char*)P.x[side] + (t * P.sn[side]) * SIZE;
    char* out = (char*)P.out[side] + (t * P.on[side]) * SIZE;
#pragma unroll 4
    for (int h = first; h < P.heads[side]; h += step) {
      const char* p = in + (h * P.sh[side]) * SIZE;
      char* o = out + (h * P.oh[side]) * SIZE;
      U a;
      a.load(p + at * SIZE);
      if (!turns) {
        a.store(o + at * SIZE);
      } else if constexpr (ONE) {
        U y;
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          y.v[2 * i] = fmaf(a.v[2 * i], w[i].x, -a.v[2 * i + 1] * w[i].y);
          y.v[2 * i + 1] = fmaf(a.v[2 * i + 1], w[i].x, a.v[2 * i] * w[i].y);
        }
        y.store(o + at * SIZE);
      } else {
        U b, y, z;
        b.load(p + other * SIZE);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          y.v[i] = fmaf(a.v[i], w[i].x, -b.v[i] * w[i].y);
          z.v[i] = fmaf(b.v[i], w[i].x, a.v[i] * w[i].y);
        }
        y.store(o + at * SIZE);
        z.store(o + other * SIZE);
      }
    }
  }
}

template <int DT>
void launch(const Rope& P, int n_tokens, bool vec, bool inter, hipStream_t st) {
  if (vec && inter) rope_kernel<DT, true, true><<<n_tokens, kThreads, 0, st>>>(P);
  else if (vec) rope_kernel<DT, true, false><<<n_tokens, kThreads, 0, st>>>(P);
  else if (inter) rope_kernel<DT, false, true><<<n_tokens, kThreads, 0, st>>>(P);
  else rope_kernel<DT, false, false><<<n_tokens, kThreads, 0, st>>>(P);
}

}  // namespace

extern "C" int kvt_rope(const void* q, int64_t sq_n, int64_t sq_h, int Hq, void* out_q, int64_t oq_n, int64_t oq_h,
                        const void* k, int64_t sk_n, int64_t sk_h, int Hk, void* out_k, int64_t ok_n, int64_t ok_h,
                        int dtype, int n_tokens, int D, int rot, const void* inv_freq, const void* positions,
                        int positions_are_int64, const void* cu, int n, const void* rows, const void* ahead, int n_rows,
                        float scale, int interleaved, int inverse, void* stream) {
  if (D < 2 || D > 256 || rot < 2 || rot > D || rot & 1 || Hq < 1 || Hk < 0 || n_tokens < 0) return KVT_EINVAL;
  if (dtype != kBF16 && dtype != kF16 && dtype != kF32) return KVT_EINVAL;
  if (cu && (n < 1 || n > kMaxReq || positions_are_int64 || (ahead && n_rows < 1))) return KVT_EINVAL;
  if (!cu && ahead) return KVT_EINVAL;
  if (n_tokens >= 1 << 24) return KVT_ERANGE;                 // (2^32 threads)
  if (n_tokens == 0) return KVT_OK;
  const int size = dtype == kF32 ? 4 : 2, e = 16 / size;
  Rope P;
  P.x[0] = q, P.x[1] = k, P.out[0] = out_q, P.out[1] = out_k;
  P.sn[0] = sq_n, P.sn[1] = sk_n, P.sh[0] = sq_h, P.sh[1] = sk_h;
  P.on[0] = oq_n, P.on[1] = ok_n, P.oh[0] = oq_h, P.oh[1] = ok_h;
  P.heads[0] = Hq, P.heads[1] = k ? Hk : 0;
  bool vec = D % e == 0 && rot % e == 0 && (interleaved || (rot >> 1) % e == 0);
  for (int s = 0; s < 2; ++s) {
    P.copy[s] = P.heads[s] > 0 && rot < D && P.x[s] != P.out[s];
    if (P.heads[s] == 0) continue;
    if (P.x[s] == P.out[s] && (P.sn[s] != P.on[s] || P.sh[s] != P.oh[s])) return KVT_EINVAL;
    vec = vec && !(((uintptr_t)P.x[s] | (uintptr_t)P.out[s]) & 15) &&
          !((P.sn[s] | P.sh[s] | P.on[s] | P.oh[s]) & (e - 1));
  }
  P.positions = positions, P.inv_freq = (const double*)inv_freq, P.cu = (const int32_t*)cu;
  P.rows = (const int32_t*)rows, P.ahead = (const int32_t*)ahead, P.scale = scale;
  P.n = n, P.n_rows = n_rows, P.D = D, P.rot = rot, P.wide = positions_are_int64, P.sign = inverse ? -1 : 1;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == kBF16) launch<kBF16>(P, n_tokens, vec, interleaved, st);
  else if (dtype == kF16) launch<kF16>(P, n_tokens, vec, interleaved, st);
  else launch<kF32>(P, n_tokens, vec, interleaved, st);
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}
