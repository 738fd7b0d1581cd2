// Eviction from the 8-bit block cache by accumulated attention weight: which entries stay (kvt_block_keep), their move
// into the places of those that go (kvt_block_evict), and the blocks behind the budget back to the free list
// (kvt_block_trim).
//
// Attention does not ask for the order of a cache's entries (keys are rotated to their positions before they are
// written), so nothing is compacted: of the `budget` entries that stay, those below the budget stay where they are, and
// those behind it, in order, take the free places, in order.  Sources lie behind the budget, which is a multiple of the
// block size, and destinations before it: no launch reads what it writes, and a row moves at most once per eviction.
// What the order no longer says, pos does: entry e >= held was never moved and sits at position e + evicted.
#include "block_common.h"

using namespace kvt;
using namespace kvt::blk;

namespace {

// ---------------------------------------------------------------------------------------------------------------- keep
constexpr int kKeepThreads = 1024, kWaves = kKeepThreads / 64;

struct Keep {
  const float* weights;
  const int32_t* kv_lens;
  const int32_t* rows;
  const int32_t* pos;
  const int32_t* held;
  const int32_t* evicted;
  int32_t* src;
  int32_t* list;               // [n * H, budget]: entries that move
  int64_t sw_r, sw_h, sp_r, sp_h, cap;
  int n, n_rows, H, budget, recent, sinks;
};

// Weights in the order of unsigned numbers: NaN below all, -0 as 0.
KVT_DEV uint32_t ordered(float w) {
  const uint32_t b = __float_as_uint(w + 0.0f);
  return w != w ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sum over lanes before this one, and over all (a block of 16 wavefronts; sums: 16 entries).
KVT_DEV int before(int v, int* sums, int& all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(x, o, 64);
    if (lane >= o) x += u;
  }
  __syncthreads();
  if (lane == 63) sums[w] = x;
  __syncthreads();
  int b = 0;
  all = 0;
  for (int i = 0; i < kWaves; ++i) {
    if (i < w) b += sums[i];
    all += sums[i];
  }
  return b + x - v;
}

// The keys' budget-th largest by radix select, 11 + 11 + 10 bits, each pass a histogram in LDS; ties to the lowest entry.
// One workgroup per (request, KV head).
__global__ __launch_bounds__(kKeepThreads) void keep_kernel(const Keep P) {
  __shared__ int hist[2048], sums[kWaves], found[2];
  const int h = blockIdx.x % P.H, j = blockIdx.x / P.H, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row = P.rows ? P.rows[j] : j;
  const bool bad = row < 0 || row >= P.n_rows;
  const int len = bad ? 0 : (int)min((int64_t)max(P.kv_lens[j], 0), P.cap);
  int32_t* src = P.src + ((int64_t)j * P.H + h) * P.budget;
  int32_t* list = P.list + ((int64_t)j * P.H + h) * P.budget;
  if (len <= P.budget) {
    for (int e = tid; e < P.budget; e += kKeepThreads) src[e] = e < len ? e : -1;
    return;
  }
  const float* w = P.weights + row * P.sw_r + h * P.sw_h;
  const int32_t* pos = P.pos ? P.pos + row * P.sp_r + h * P.sp_h : nullptr;
  const int held = pos ? min(max(P.held[row], 0), len) : 0;
  const int64_t evicted = pos ? P.evicted[row] : 0, last = (int64_t)len + evicted - P.recent;
  auto key = [&](int e) {
    const int64_t at = e < held ? (int64_t)pos[e] : e + evicted;
    return e < P.sinks || at >= last ? 0xFFFFFFFFu : ordered(w[e]);
  };

  uint32_t prefix = 0, mask = 0;
  int k = P.budget;
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    __syncthreads();
    for (int i = tid; i < 2048; i += kKeepThreads) hist[i] = 0;
    __syncthreads();
    for (int e = tid; e < len; e += kKeepThreads) {
      const uint32_t u = key(e);
      if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift) & ((1 << bits) - 1)], 1);
    }
    __syncthreads();
    // bins from the highest on: thread t has bins 2047 - 2 t and 2046 - 2 t
    const int a = hist[2047 - 2 * tid], b = hist[2046 - 2 * tid];
    int all;
    const int above = before(a + b, sums, all);
    if (above < k && k <= above + a) found[0] = 2047 - 2 * tid, found[1] = k - above;
    else if (above + a < k && k <= above + a + b) found[0] = 2046 - 2 * tid, found[1] = k - above - a;
    __syncthreads();
    prefix |= (uint32_t)found[0] << shift;
    mask |= (uint32_t)((1 << bits) - 1) << shift;
    k = found[1];
  }

  // wavefront v has entries v * seg ..: the k first ties stay; ranks by ballots
  const int seg = (((len + kWaves - 1) / kWaves) + 63) & ~63;
  const int e0 = min(wave * seg, len), e1 = min(e0 + seg, len);
  const uint64_t lower = ((uint64_t)1 << lane) - 1;
  int count = 0, all;
  for (int e = e0 + lane; e < e1; e += 64) count += key(e) == prefix;
  int ties = before(count, sums, all);
  ties = __shfl(ties, 0, 64);
  auto walk = [&](auto f) {                 // f(entry, whether it stays), every lane of the wavefront in step
    int t = ties;
    for (int base = e0; base < e1; base += 64) {
      const int e = base + lane;
      const uint32_t u = e < e1 ? key(e) : 0u;
      const bool tie = e < e1 && u == prefix;
      const uint64_t b = __ballot(tie);
      const bool stays = e < e1 && (u > prefix || (tie && t + __popcll(b & lower) < k));
      t += __popcll(b);
      f(e, stays);
    }
  };
  int moves = 0, frees = 0;
  walk([&](int e, bool stays) {
    moves += __popcll(__ballot(stays && e >= P.budget));
    frees += __popcll(__ballot(!stays && e < P.budget && e < e1));
  });
  int m = __shfl(before(lane == 0 ? moves : 0, sums, all), 0, 64);
  int f = __shfl(before(lane == 0 ? frees : 0, sums, all), 0, 64);
  walk([&](int e, bool stays) {
    const uint64_t b = __ballot(stays && e >= P.budget);
    if (stays && e >= P.budget) list[m + __popcll(b & lower)] = e;
    m += __popcll(b);
  });
  __syncthreads();
  walk([&](int e, bool stays) {
    const bool free = !stays && e < P.budget && e < e1;
    const uint64_t b = __ballot(free);
    if (e < P.budget && e < e1) src[e] = free ? list[f + __popcll(b & lower)] : e;
    f += __popcll(b);
  });
}

// --------------------------------------------------------------------------------------------------------------- evict
struct Evict {
  const int32_t* src;
  const int32_t* kv_lens;
  const int32_t* rows;
  const int32_t* table;
  const int32_t* held;
  const int32_t* evicted;
  uint8_t* codes[2];
  float* scale[2];
  float* weights;
  int32_t* pos;
  int64_t stride, sw_r, sw_h, sp_r, sp_h, cap;
  int n, n_rows, H, n_blocks, max_blocks, log2b, budget;
};

// The largest finite magnitude of four codes.
template <int CODE>
KVT_DEV float magnitude(uint32_t w) {
  if constexpr (CODE == kE4M3) {
    uint32_t m = w & 0x7F7F7F7Fu;
    m &= ~((((m + 0x01010101u) & 0x80808080u) >> 7) * 0xFFu);          // (NaN codes count as 0)
    const uint32_t a = max(m & 0xFFu, m >> 8 & 0xFFu), b = max(m >> 16 & 0xFFu, m >> 24);
    return __builtin_amdgcn_cvt_f32_fp8((int)max(a, b), 0);            // (magnitudes are ordered as their codes are)
  } else {
    float x[4];
    unpack4<CODE>(w, x);
    return fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));
  }
}

// One workgroup per (request, KV head, block below the budget).  A block of which every row stays is left as it is.
// Another one's scale is the smallest power of two that holds its rows' values, as if they were stored anew; a row that
// stays is written again only if the scale changed.
template <int CODE, int D>
__global__ __launch_bounds__(256) void evict_kernel(const Evict P) {
  constexpr int TPR = D / 16;                 // threads per row
  constexpr int RPP = 256 / TPR;              // rows per pass
  constexpr int NP = 64 / RPP > 0 ? 64 / RPP : 1;
  __shared__ int from[64], moved[64];         // pool row of each row; whether it moves
  __shared__ float scales[2][64];
  __shared__ float part[4];
  const int B = 1 << P.log2b, nb = P.budget >> P.log2b;
  const int lp = blockIdx.x % nb, w = blockIdx.x / nb, h = w % P.H, j = w / P.H;
  const int row = P.rows ? P.rows[j] : j;
  if (row < 0 || row >= P.n_rows) return;
  const int len = (int)min((int64_t)max(P.kv_lens[j], 0), P.cap);
  if (len <= P.budget) return;
  const int64_t tbl = row * P.stride;
  const int block = P.table[tbl + lp];
  const bool there = block >= 0 && block < P.n_blocks;
  const int t = threadIdx.x;
  int moves = 0;
  if (t < B) {
    const int e = (lp << P.log2b) + t;
    const int s = P.src[((int64_t)j * P.H + h) * P.budget + e];
    int b = s >= P.budget && s < len ? P.table[tbl + (s >> P.log2b)] : -1;
    moves = b >= 0 && b < P.n_blocks && there;
    if (P.weights && moves) {
      float* x = P.weights + row * P.sw_r + h * P.sw_h;
      x[e] = x[s];
    }
    if (P.pos) {
      int32_t* x = P.pos + row * P.sp_r + h * P.sp_h;
      const int held = P.held[row], gone = P.evicted[row], at = moves ? s : e;
      if (moves || e >= held) x[e] = at < held ? x[at] : at + gone;
    }
    moved[t] = moves;
    if (!moves) b = block;
    from[t] = there ? (b << P.log2b) + ((moves ? s : e) & (B - 1)) : 0;
    if (there) {
      const int64_t at = (int64_t)b * P.H + h;
      scales[0][t] = P.scale[0][at], scales[1][t] = P.scale[1][at];
    }
  }
  if (!__syncthreads_or(moves)) return;
  const int tr = t / TPR, tc = t % TPR;
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    uint8_t* codes = P.codes[side];
    u4v raw[NP];
    float top = 0.0f;
    bool fine = true;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = tr + i * RPP;
      if (r >= B) continue;
      const int at = from[r];
      raw[i] = *reinterpret_cast<const u4v*>(
          codes + ((((int64_t)(at >> P.log2b) * P.H + h) << P.log2b) + (at & (B - 1))) * D + 16 * tc);
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = tr + i * RPP;
      if (r >= B) continue;
      float m = 0.0f;
#pragma unroll
      for (int c = 0; c < 4; ++c) m = fmaxf(m, magnitude<CODE>(raw[i][c]));
      const float s = scales[side][r];
      fine = fine && s - s == 0.0f;
      top = fmaxf(top, m * s);
    }
    top = group_max<64>(fine ? fminf(top, 3.402823466e38f) : __builtin_inff());   // (infinity: a scale that is not finite)
    __syncthreads();
    if ((t & 63) == 0) part[t >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
    const bool finite = top < __builtin_inff();
    const float size = finite ? pow2_scale<CODE>(top) : __builtin_nanf("");
    const float inv = 1.0f / size;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int r = tr + i * RPP;
      if (r >= B) continue;
      const float s = scales[side][r];
      if (!moved[r] && (!finite || s == size)) continue;
      u4v o = raw[i];
      if (finite && s != size) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float y[4];
          unpack4<CODE>(raw[i][c], y);
          o[c] = pack4<CODE>(y[0] * s * inv, y[1] * s * inv, y[2] * s * inv, y[3] * s * inv);
        }
      }
      *reinterpret_cast<u4v*>(codes + ((((int64_t)block * P.H + h) << P.log2b) + r) * D + 16 * tc) = o;
    }
    if (t == 0) P.scale[side][(int64_t)block * P.H + h] = size;
  }
}

template <int CODE>
void evict_launch(const Evict& P, int D, int grid, hipStream_t st) {
  if (D == 64) evict_kernel<CODE, 64><<<grid, 256, 0, st>>>(P);
  else if (D == 128) evict_kernel<CODE, 128><<<grid, 256, 0, st>>>(P);
  else evict_kernel<CODE, 256><<<grid, 256, 0, st>>>(P);
}

// ---------------------------------------------------------------------------------------------------------------- trim
constexpr int kMaxTrim = 1024, kStamps = 4096;
enum { kBadRow = 8, kFreeOver = 16 };

struct Trim {
  const int32_t* seqs;
  int32_t* seq_lens;
  int32_t* table;
  int32_t* free_list;
  int32_t* free_head;
  int32_t* held;
  int32_t* evicted;
  int32_t* kv_lens;
  int32_t* next_head;
  int32_t* status;
  int64_t stride;
  int n, rows, max_blocks, n_free, log2b, budget, commit;
};

// One workgroup: a thread per request finds its length and whether an earlier request has its row, a wavefront per request
// counts the blocks that it gives back, and after a scan writes them in request order.
__global__ __launch_bounds__(1024) void trim_kernel(const Trim P) {
  __shared__ int rows[kMaxTrim], lens[kMaxTrim], count[kMaxTrim], stamp[kStamps], sums[kWaves], flags;
  const int j = threadIdx.x, lane = j & 63, wave = j >> 6;
  if (j == 0) flags = 0;
  for (int i = j; i < kStamps; i += 1024) stamp[i] = kMaxTrim;
  int row = -1;
  if (j < P.n) {
    row = P.seqs[j];
    if (row < 0 || row >= P.rows) row = -1;
    rows[j] = row;
  }
  __syncthreads();
  if (row >= 0) atomicMin(&stamp[row & (kStamps - 1)], j);
  __syncthreads();
  bool bad = j < P.n && row < 0;
  if (row >= 0) {
    const int w = stamp[row & (kStamps - 1)];
    if (w != j) {
      bool twice = rows[w] == row;
      if (!twice)                // (more than 4,096 table rows: another row has the stamp)
        for (int i = 0; i < j && !twice; ++i) twice = rows[i] == row;
      bad = twice;
    }
  }
  __syncthreads();
  if (bad) rows[j] = row = -1;
  int len = 0;
  if (j < P.n) {
    len = row >= 0 ? max(P.seq_lens[row], 0) : 0;
    lens[j] = len;
    P.kv_lens[j] = min(len, P.budget);
    if (bad) atomicOr(&flags, kBadRow);
  }
  __syncthreads();
  const int first = P.budget >> P.log2b;
  auto blocks = [&](int r, auto f) {                  // f(table entry, its id, whether it is a block)
    const int last = (int)min(((int64_t)lens[r] + (1 << P.log2b) - 1) >> P.log2b, (int64_t)P.max_blocks);
    for (int base = first; base < last; base += 64) {
      int32_t* at = P.table + rows[r] * P.stride + base + lane;
      const int id = base + lane < last ? *at : -1;
      f(at, id >= 0 && id < P.n_free, id, base + lane < last);
    }
  };
  for (int r = wave; r < P.n; r += kWaves) {
    int c = 0;
    if (rows[r] >= 0) blocks(r, [&](int32_t*, bool is, int, bool) { c += __popcll(__ballot(is)); });
    if (lane == 0) count[r] = c;
  }
  __syncthreads();
  int total;
  const int c = j < P.n ? count[j] : 0;
  const int at = before(c, sums, total);
  const int head = min(max(*P.free_head, 0), P.n_free);
  __syncthreads();
  if (j < P.n) count[j] = at;
  if (j == 0) {
    *P.next_head = max(head - total, 0);
    if (total > head) atomicOr(&flags, kFreeOver);
  }
  __syncthreads();
  for (int r = wave; r < P.n; r += kWaves) {
    if (rows[r] < 0) continue;
    int to = head - total + count[r];
    blocks(r, [&](int32_t* p, bool is, int id, bool in) {
      const uint64_t b = __ballot(is);
      const int k = to + __popcll(b & (((uint64_t)1 << lane) - 1));
      if (is && k >= 0) P.free_list[k] = id;
      if (in && P.commit) *p = -1;
      to += __popcll(b);
    });
  }
  if (P.commit && row >= 0 && len > P.budget) {
    P.seq_lens[row] = P.budget;
    if (P.evicted) P.evicted[row] += len - P.budget, P.held[row] = P.budget;
  }
  if (j == 0) {
    if (P.commit) *P.free_head = max(head - total, 0);
    if (P.status && flags) atomicOr(P.status, flags);
  }
}

}  // namespace

extern "C" int kvt_block_keep(const void* weights, int64_t sw_r, int64_t sw_h, const void* kv_lens, int n, int H,
                              int n_rows, const void* rows, int64_t cap, int budget, int recent, int sinks, const void* pos,
                              int64_t sp_r, int64_t sp_h, const void* held, const void* evicted, void* src, void* work,
                              void* stream) {
  if (n < 1 || H < 1 || n_rows < 1 || cap < 1 || budget < 1 || recent < 0 || sinks < 0 || (!rows && n_rows < n))
    return KVT_EINVAL;
  if ((int64_t)recent + sinks > budget || !pos != !held || !pos != !evicted) return KVT_EINVAL;
  if (cap > ((int64_t)1 << 31) - 8192 || (int64_t)n * H >= 1 << 22) return KVT_ERANGE;
  Keep P;
  P.weights = (const float*)weights, P.kv_lens = (const int32_t*)kv_lens, P.rows = (const int32_t*)rows;
  P.pos = (const int32_t*)pos, P.held = (const int32_t*)held, P.evicted = (const int32_t*)evicted;
  P.src = (int32_t*)src, P.list = (int32_t*)work, P.sw_r = sw_r, P.sw_h = sw_h, P.sp_r = sp_r, P.sp_h = sp_h, P.cap = cap;
  P.n = n, P.n_rows = n_rows, P.H = H, P.budget = budget, P.recent = recent, P.sinks = sinks;
  keep_kernel<<<n * H, kKeepThreads, 0, (hipStream_t)stream>>>(P);
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}

extern "C" int kvt_block_evict(const void* src, const void* kv_lens, int n, int H, int D, int code, void* k8, void* v8,
                               void* ks, void* vs, int n_blocks, int block, const void* block_table, int64_t bt_stride,
                               int n_rows, int max_blocks, const void* rows, int budget, void* weights, int64_t sw_r,
                               int64_t sw_h, void* pos, int64_t sp_r, int64_t sp_h, const void* held, const void* evicted,
                               void* stream) {
  if (n < 1 || H < 1 || n_blocks < 1 || n_rows < 1 || max_blocks < 1 || bt_stride < max_blocks || (!rows && n_rows < n))
    return KVT_EINVAL;
  if ((D != 64 && D != 128 && D != 256) || (block != 16 && block != 32 && block != 64)) return KVT_EINVAL;
  if ((code != kE4M3 && code != kI8) || budget < block || budget % block || budget / block > max_blocks) return KVT_EINVAL;
  if (((uintptr_t)k8 | (uintptr_t)v8) & 15 || (pos && (!held || !evicted))) return KVT_EINVAL;
  const int64_t grid = (int64_t)n * H * (budget / block);
  if (grid >= 1 << 24 || (int64_t)max_blocks * block > ((int64_t)1 << 31) - 8192 ||
      (int64_t)n_blocks * block > (int64_t)1 << 31)
    return KVT_ERANGE;
  Evict P;
  P.src = (const int32_t*)src, P.kv_lens = (const int32_t*)kv_lens, P.rows = (const int32_t*)rows;
  P.table = (const int32_t*)block_table, P.held = (const int32_t*)held, P.evicted = (const int32_t*)evicted;
  P.codes[0] = (uint8_t*)k8, P.codes[1] = (uint8_t*)v8, P.scale[0] = (float*)ks, P.scale[1] = (float*)vs;
  P.weights = (float*)weights, P.pos = (int32_t*)pos, P.stride = bt_stride;
  P.sw_r = sw_r, P.sw_h = sw_h, P.sp_r = sp_r, P.sp_h = sp_h, P.cap = (int64_t)max_blocks * block;
  P.n = n, P.n_rows = n_rows, P.H = H, P.n_blocks = n_blocks, P.max_blocks = max_blocks;
  P.log2b = block == 16 ? 4 : block == 32 ? 5 : 6, P.budget = budget;
  if (code == kE4M3) evict_launch<kE4M3>(P, D, (int)grid, (hipStream_t)stream);
  else evict_launch<kI8>(P, D, (int)grid, (hipStream_t)stream);
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}

extern "C" int kvt_block_trim(int n, const void* seqs, void* seq_lens, int rows, void* block_table, int64_t bt_stride,
                              int max_blocks, void* free_list, int n_free, void* free_head, int block, int budget,
                              void* held, void* evicted, void* kv_lens, void* next_head, void* status, int commit,
                              void* stream) {
  if (n < 1 || n > kMaxTrim || rows < 1 || max_blocks < 1 || bt_stride < max_blocks || n_free < 0) return KVT_EINVAL;
  if ((block != 16 && block != 32 && block != 64) || budget < block || budget % block || !held != !evicted) return KVT_EINVAL;
  Trim P;
  P.seqs = (const int32_t*)seqs, P.seq_lens = (int32_t*)seq_lens, P.table = (int32_t*)block_table;
  P.free_list = (int32_t*)free_list, P.free_head = (int32_t*)free_head, P.held = (int32_t*)held;
  P.evicted = (int32_t*)evicted, P.kv_lens = (int32_t*)kv_lens, P.next_head = (int32_t*)next_head;
  P.status = (int32_t*)status, P.stride = bt_stride, P.n = n, P.rows = rows, P.max_blocks = max_blocks;
  P.n_free = n_free, P.log2b = block == 16 ? 4 : block == 32 ? 5 : 6, P.budget = budget, P.commit = commit;
  trim_kernel<<<1, 1024, 0, (hipStream_t)stream>>>(P);
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}
