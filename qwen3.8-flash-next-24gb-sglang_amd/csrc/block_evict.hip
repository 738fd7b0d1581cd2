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
//
// The budget-th largest key of a (request, KV head) by radix select (11 + 11 + 10 bits, histograms in LDS), ties to the
// lowest entry, and the places of what moves, from ranks by ballots.  Up to kSmall entries (kFew: one of 512 threads) one
// workgroup does it all with the keys in registers, read once.  Longer ones take a launch per step, with kMostChunks
// workgroups a pair at most: three histograms (joined by integer atomics: their order does not matter), counts per
// chunk, places.  Lengths are on the device, so a wide table takes all launches, and each leaves the pairs alone that are
// not its own.  us a call, calls in a row: 64 x 8 pairs of 4,160 entries to 4,096 13.6 (14.2 with positions; by the kernel
// of 1,024 threads 31), in tables of 16,384 16.4, of 65,536 38; nothing over the budget 3.6 and 28; two pairs of 8,192 13.3,
// of 8,256 20, of 32,768 33, of 32,769 36; of 262,144 to 16,384 40 (one workgroup a pair, which reads the keys seven times,
// 742); 64 x 8 of 16,384 47, of 32,768 68, of 32,769 236 (every key read seven times, by one or two workgroups a pair).
constexpr int kKeepThreads = 1024, kWaves = kKeepThreads / 64;
constexpr int kFew = 8192, kSmall = 32768, kChunk = 4096, kMostChunks = 256, kBins = 2048;
constexpr int64_t kChunkBlocks = 1024;        // workgroups of a step's launch, about

struct Keep {
  const float* weights;
  const int32_t* kv_lens;
  const int32_t* rows;
  const int32_t* pos;
  const int32_t* held;
  const int32_t* evicted;
  int32_t* src;
  int32_t* work;               // per pair: 3 histograms, 4 counts per chunk, a Found per pass, sources, free places
  int64_t sw_r, sw_h, sp_r, sp_h, cap;
  int n, n_rows, H, budget, recent, sinks, chunks;
};
struct Found { int prefix, k, moves, pad; };
KVT_DEV int64_t work_size(const Keep& P) { return 3 * kBins + 4 * P.chunks + 12 + 2 * (((int64_t)P.budget + 1) & ~1); }

// Weights in the order of unsigned numbers: NaN (1) below all, -0 as 0; 0 is no key.
KVT_DEV uint32_t ordered(float w) {
  const uint32_t b = __float_as_uint(w + 0.0f);
  return w != w ? 1u : b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sum over the threads before this one, and over all (a block of 16 wavefronts; sums: 16 entries).
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
#pragma unroll
  for (int i = 0; i < kWaves; ++i) {
    const int s = sums[i];
    b += i < w ? s : 0;
    all += s;
  }
  return b + x - v;
}

// A (request, KV head): its entries' keys.
struct Pair {
  const float* w;
  const int32_t* pos;
  int32_t* src;
  uint32_t evicted, last;      // (positions are below 2^32)
  int len, held, sinks;
  // of an entry's weight and, if it is one of those held, position (both loads without a branch around them)
  KVT_DEV int place(int e) const { return pos ? pos[e] : 0; }
  KVT_DEV uint32_t key(int e, float weight, int place) const {
    const uint32_t at = e < held ? (uint32_t)place : e + evicted;
    return e < sinks || at >= last ? 0xFFFFFFFFu : ordered(weight);
  }
  KVT_DEV uint32_t key(int e) const { return key(e, w[e], place(e)); }
};
KVT_DEV Pair pair_of(const Keep& P, int id) {
  const int h = id % P.H, j = id / P.H, row = P.rows ? P.rows[j] : j;
  const bool bad = row < 0 || row >= P.n_rows;
  Pair t;
  t.len = bad ? 0 : (int)min((int64_t)max(P.kv_lens[j], 0), P.cap);
  t.src = P.src + ((int64_t)j * P.H + h) * P.budget;
  const int64_t r = bad ? 0 : row;
  t.w = P.weights + r * P.sw_r + h * P.sw_h;
  t.pos = P.pos ? P.pos + r * P.sp_r + h * P.sp_h : nullptr;
  t.held = P.pos ? min(max(P.held[r], 0), t.len) : 0;
  t.evicted = P.pos ? max(P.evicted[r], 0) : 0;
  t.last = (uint32_t)max((int64_t)t.len + t.evicted - P.recent, (int64_t)0);
  t.sinks = P.sinks;
  return t;
}

// Where the k-th largest of a histogram's keys is: its bin and the k that is left within it.  found: two entries.
KVT_DEV void find_bin(const int* hist, int k, int* sums, int* found, int& bin, int& left) {
  // bins from the highest on: thread t has bins 2047 - 2 t and 2046 - 2 t
  const int t = threadIdx.x, a = hist[kBins - 1 - 2 * t], b = hist[kBins - 2 - 2 * t];
  int all;
  const int above = before(a + b, sums, all);
  if (above < k && k <= above + a) found[0] = kBins - 1 - 2 * t, found[1] = k - above;
  else if (above + a < k && k <= above + a + b) found[0] = kBins - 2 - 2 * t, found[1] = k - above - a;
  __syncthreads();
  bin = found[0], left = found[1];
}
KVT_DEV int shift_of(int pass) { return pass == 0 ? 21 : pass == 1 ? 10 : 0; }
KVT_DEV int bins_of(int pass) { return pass == 2 ? 1024 : 2048; }

// The same by every wavefront for itself: lane l has bins 2047 - 32 l and the 31 below.  Four words lie between those
// of two lanes (padded), so that their 16-byte reads are spread over the banks.
constexpr int kPadded = kBins + kBins / 8;
KVT_DEV int padded(int bin) { return bin + (bin >> 5) * 4; }
KVT_DEV int wave_before(int v) {                  // sum over the lanes up to this one
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    v += lane >= o ? u : 0;
  }
  return v;
}
KVT_DEV void find_bin_wave(const int* hist, int k, int& bin, int& left) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int4 v = *reinterpret_cast<const int4*>(hist + 36 * (63 - lane) + 4 * i);
    sum += v.x + v.y + v.z + v.w;
  }
  int x = wave_before(sum);
  const int from = __ffsll((unsigned long long)__ballot(x - sum < k && k <= x)) - 1;
  k -= __builtin_amdgcn_readlane(x - sum, from);
  const int n = lane < 32 ? hist[36 * (63 - from) + 31 - lane] : 0;       // its bins, from the highest on
  x = wave_before(n);
  const int at = __ffsll((unsigned long long)__ballot(x - n < k && k <= x)) - 1;
  bin = kBins - 1 - 32 * from - at, left = k - __builtin_amdgcn_readlane(x - n, at);
}

// One workgroup of T threads per pair of more than OVER and no more than T R entries: wavefront v has entries v * seg ..,
// key i of a lane that of entry v * seg + 64 i + lane.  Latency and its instructions bound it: 512 x 4,160 entries, keys
// re-read from memory by 1,024 threads 39 us, in registers 26, every wavefront finding a histogram's bin for itself
// instead of three barriers more, 512 threads, 16 (256 threads 20, 1,024 19).  More than 8,192 entries: 101 registers at
// 1,024 threads, so one workgroup a CU and nothing behind its barriers (512 x 32,768 entries 68, 67 MB of weights).
template <int T, int R, int OVER>
__global__ __launch_bounds__(T) void keep_kernel(const Keep P) {
  __shared__ __attribute__((aligned(16))) int hist[3][kPadded];
  __shared__ int sums[2][T / 64];
  __shared__ uint16_t list[T * R / 2];          // (no more than half of the entries can move)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Pair t = pair_of(P, blockIdx.x);
  if (OVER == 0 && t.len <= P.budget) {
    for (int e = tid; e < P.budget; e += T) t.src[e] = e < t.len ? e : -1;
    return;
  }
  if (OVER > 0 && t.len > kSmall && t.len > P.budget) {                 // (the launches behind begin with zeros)
    int32_t* w = P.work + blockIdx.x * work_size(P);
    for (int i = tid; i < 3 * kBins; i += T) w[i] = 0;
    return;
  }
  if (t.len <= P.budget || t.len <= OVER || t.len > T * R) return;      // (another launch's)
  const int steps = (t.len + T - 1) / T, e0 = wave * 64 * steps + lane;
  uint32_t key[R];
  int place[R];
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i < steps) key[i] = __float_as_uint(t.w[min(e0 + 64 * i, t.len - 1)]);
  if (t.held) {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (i < steps) place[i] = t.pos[min(e0 + 64 * i, t.len - 1)];
  }
  for (int i = tid; i < 3 * kPadded; i += T) hist[0][i] = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = e0 + 64 * i;
    key[i] = i < steps && e < t.len ? t.key(e, __uint_as_float(key[i]), place[i]) : 0u;
  }
  __syncthreads();
  uint32_t prefix = 0, mask = 0;
  int k = P.budget;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = shift_of(pass);
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (key[i] && (key[i] & mask) == prefix)
        atomicAdd(&hist[pass][padded((key[i] >> shift) & (bins_of(pass) - 1))], 1);
    __syncthreads();
    int bin;
    find_bin_wave(hist[pass], k, bin, k);
    prefix |= (uint32_t)bin << shift;
    mask |= (uint32_t)(bins_of(pass) - 1) << shift;
  }

  // what the wavefronts before this one have
  auto earlier = [&](int v, int* s) {
    if (lane == 0) s[wave] = v;
    __syncthreads();
    int b = 0;
#pragma unroll
    for (int i = 0; i < T / 64; ++i) b += i < wave ? s[i] : 0;
    return b;
  };
  const uint64_t lower = ((uint64_t)1 << lane) - 1;
  int count = 0;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i < steps) count += __popcll(__ballot(key[i] == prefix));
  int ties = earlier(count, sums[0]), all_ties = 0;
#pragma unroll
  for (int i = 0; i < T / 64; ++i) all_ties += sums[0][i];
  uint32_t stays = 0;                           // bit i: entry of key i stays
  int moves = 0, frees = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = e0 + 64 * i;
    if (i < steps) {
      bool is = key[i] >= prefix;
      if (all_ties > k) {                       // (not all of the ties stay)
        const bool tie = key[i] == prefix;
        const uint64_t b = __ballot(tie);
        is = key[i] > prefix || (tie && ties + __popcll(b & lower) < k);
        ties += __popcll(b);
      }
      stays |= (uint32_t)is << i;
      moves += __popcll(__ballot(is && e >= P.budget));
      frees += __popcll(__ballot(!is && e < P.budget));
    }
  }
  // (both counts in one sum: neither leaves 16 bits)
  const int at = earlier(moves << 16 | frees, sums[1]);
  int m = at >> 16, f = at & 0xFFFF;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = e0 + 64 * i;
    if (i < steps) {
      const bool is = (stays >> i & 1) && e >= P.budget;
      const uint64_t b = __ballot(is);
      if (is) list[m + __popcll(b & lower)] = (uint16_t)e;
      m += __popcll(b);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int e = e0 + 64 * i;
    if (i < steps) {
      const bool free = !(stays >> i & 1) && e < P.budget;
      const uint64_t b = __ballot(free);
      if (e < P.budget) t.src[e] = free ? (int)list[f + __popcll(b & lower)] : e;
      f += __popcll(b);
    }
  }
}

// Pairs of more than kSmall entries.  Chunk c of a pair has entries c * per .. (a multiple of 1,024).
struct Long {
  int32_t* hist;
  int32_t* counts;             // of a chunk: keys above the threshold below the budget and behind it, ties likewise
  Found* found;
  int32_t* list;
  int32_t* places;
  int begin, end;
};
KVT_DEV bool long_of(const Keep& P, int id, const Pair& t, int c, Long& L) {
  if (t.len <= P.budget || t.len <= kSmall) return false;
  int32_t* w = P.work + id * work_size(P);
  L.hist = w, L.counts = w + 3 * kBins, L.found = (Found*)(L.counts + 4 * P.chunks);
  L.list = (int32_t*)(L.found + 3), L.places = L.list + P.budget;
  const int per = ((t.len + P.chunks - 1) / P.chunks + 1023) & ~1023;
  L.begin = (int)min((int64_t)c * per, (int64_t)t.len), L.end = (int)min((int64_t)L.begin + per, (int64_t)t.len);
  return true;
}

// What pass `pass` found so far: read, or for the pass before formed from its histogram and written (by chunk 0).
KVT_DEV Found found_before(const Keep& P, const Long& L, int pass, int c, int* sums, int* found) {
  Found f = {0, P.budget, 0, 0};
  if (pass == 0) return f;
  if (pass > 1) f = L.found[pass - 2];
  int bin;
  find_bin(L.hist + (pass - 1) * kBins, f.k, sums, found, bin, f.k);
  f.prefix |= (int)((uint32_t)bin << shift_of(pass - 1));
  if (c == 0 && threadIdx.x == 0) L.found[pass - 1] = f;
  return f;
}

__global__ __launch_bounds__(kKeepThreads) void keep_hist_kernel(const Keep P, int pass) {
  __shared__ int hist[kBins], sums[kWaves], found[2];
  const int c = blockIdx.x % P.chunks, id = blockIdx.x / P.chunks, tid = threadIdx.x;
  const Pair t = pair_of(P, id);
  Long L;
  if (!long_of(P, id, t, c, L)) return;
  const Found f = found_before(P, L, pass, c, sums, found);
  if (L.begin >= L.end) return;
  const uint32_t prefix = (uint32_t)f.prefix, mask = pass == 0 ? 0u : ~0u << shift_of(pass - 1);
  for (int i = tid; i < kBins; i += kKeepThreads) hist[i] = 0;
  __syncthreads();
#pragma unroll 4
  for (int e = L.begin + tid; e < L.end; e += kKeepThreads) {
    const uint32_t u = t.key(e);
    if ((u & mask) == prefix) atomicAdd(&hist[(u >> shift_of(pass)) & (bins_of(pass) - 1)], 1);
  }
  __syncthreads();
  for (int i = tid; i < kBins; i += kKeepThreads)
    if (hist[i]) atomicAdd(&L.hist[pass * kBins + i], hist[i]);
}

__global__ __launch_bounds__(kKeepThreads) void keep_count_kernel(const Keep P) {
  __shared__ int sums[kWaves], found[2], counts[4];
  const int c = blockIdx.x % P.chunks, id = blockIdx.x / P.chunks, tid = threadIdx.x;
  const Pair t = pair_of(P, id);
  Long L;
  if (!long_of(P, id, t, c, L)) return;
  const uint32_t T = (uint32_t)found_before(P, L, 3, c, sums, found).prefix;
  if (tid < 4) counts[tid] = 0;
  __syncthreads();
  int n[4] = {0, 0, 0, 0};
#pragma unroll 4
  for (int e = L.begin + tid; e < L.end; e += kKeepThreads) {
    const uint32_t u = t.key(e);
    const bool behind = e >= P.budget;
    n[0] += u > T && !behind, n[1] += u > T && behind, n[2] += u == T && !behind, n[3] += u == T && behind;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int o = 32; o; o >>= 1) n[i] += __shfl_xor(n[i], o, 64);
    if ((tid & 63) == 0) atomicAdd(&counts[i], n[i]);
  }
  __syncthreads();
  if (tid < 4) L.counts[4 * c + tid] = counts[tid];
}

// Entries that stay below the budget, and the lists of those that move and of the places that are free.
__global__ __launch_bounds__(kKeepThreads) void keep_list_kernel(const Keep P) {
  __shared__ int sums[kWaves], start[3];
  const int c = blockIdx.x % P.chunks, id = blockIdx.x / P.chunks, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Pair t = pair_of(P, id);
  Long L;
  if (!long_of(P, id, t, c, L)) return;
  const uint32_t T = (uint32_t)L.found[2].prefix;
  const int k = L.found[2].k;
  if (wave == 0) {
    // ties, moves and free places before the chunk: the ties that stay follow from the number of ties before
    int ties = 0, moves = 0, frees = 0, total = 0;
    for (int base = 0; base < P.chunks; base += 64) {
      const int i = base + lane;
      const int4 n = i < P.chunks ? *reinterpret_cast<const int4*>(L.counts + 4 * i) : make_int4(0, 0, 0, 0);
      int x = n.z + n.w;                        // (ties are taken below the budget first: entries in order)
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(x, o, 64);
        if (lane >= o) x += u;
      }
      const int first = ties + x - n.z - n.w;
      const int low = min(max(k - first, 0), n.z), high = min(max(k - first - n.z, 0), n.w);
      const int per = ((t.len + P.chunks - 1) / P.chunks + 1023) & ~1023;
      const int64_t b = (int64_t)i * per;
      const int64_t has = i < P.chunks ? min((int64_t)per, max((int64_t)t.len - b, (int64_t)0)) : 0;
      const int below = (int)min(max((int64_t)P.budget - b, (int64_t)0), has);
      int mv = n.y + high, fr = below - n.x - low;
      total += mv;
      if (i >= c) mv = fr = 0;
      int tb = i < c ? n.z + n.w : 0;
#pragma unroll
      for (int o = 32; o; o >>= 1) {
        mv += __shfl_xor(mv, o, 64);
        fr += __shfl_xor(fr, o, 64);
        tb += __shfl_xor(tb, o, 64);
      }
      moves += mv, frees += fr;
      if (base <= c && c < base + 64 && lane == 0) start[0] = ties + tb;
      ties += __shfl(x, 63, 64);
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o, 64);
    if (lane == 0) {
      start[1] = moves, start[2] = frees;
      if (c == 0) L.found[2].moves = total;
    }
  }
  __syncthreads();
  if (L.begin >= L.end) return;
  const int seg = ((L.end - L.begin + kKeepThreads - 1) / kKeepThreads) * 64;
  const int e0 = min(L.begin + wave * seg, L.end), e1 = min(e0 + seg, L.end);
  const uint64_t lower = ((uint64_t)1 << lane) - 1;
  int count = 0, all;
#pragma unroll 4
  for (int e = e0 + lane; e < e1; e += 64) count += t.key(e) == T;
  int ties = start[0] + __shfl(before(count, sums, all), 0, 64);
  auto walk = [&](auto f) {                     // f(entry, whether it is one, whether it stays), the wavefront in step
    int n = ties;
    for (int base = e0; base < e1; base += 256) {             // (four loads under way at once)
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = base + 64 * i + lane < e1 ? t.key(base + 64 * i + lane) : 0u;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = base + 64 * i + lane;
        const bool tie = e < e1 && u[i] == T;
        const uint64_t b = __ballot(tie);
        f(e, e < e1, e < e1 && (u[i] > T || (tie && n + __popcll(b & lower) < k)));
        n += __popcll(b);
      }
    }
  };
  int moves = 0, frees = 0;
  walk([&](int e, bool is, bool stays) {
    moves += __popcll(__ballot(stays && e >= P.budget));
    frees += __popcll(__ballot(is && !stays && e < P.budget));
  });
  int m = start[1] + __shfl(before(lane == 0 ? moves : 0, sums, all), 0, 64);
  int f = start[2] + __shfl(before(lane == 0 ? frees : 0, sums, all), 0, 64);
  walk([&](int e, bool is, bool stays) {
    const bool move = stays && e >= P.budget, free = is && !stays && e < P.budget;
    const uint64_t b = __ballot(move), g = __ballot(free);
    if (move) L.list[m + __popcll(b & lower)] = e;
    if (free) L.places[f + __popcll(g & lower)] = e;
    if (is && stays && e < P.budget) t.src[e] = e;
    m += __popcll(b), f += __popcll(g);
  });
}

__global__ __launch_bounds__(256) void keep_place_kernel(const Keep P, int blocks) {
  const int id = blockIdx.x / blocks;
  const Pair t = pair_of(P, id);
  Long L;
  if (!long_of(P, id, t, 0, L)) return;
  const int moves = L.found[2].moves;
  for (int i = (blockIdx.x % blocks) * 256 + threadIdx.x; i < moves; i += blocks * 256) t.src[L.places[i]] = L.list[i];
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

// The largest finite magnitude of sixteen codes, two bytes of a dword at a time.
typedef int16_t s2 __attribute__((ext_vector_type(2)));
template <int CODE>
KVT_DEV float magnitude(u4v v) {
  if constexpr (CODE == kE4M3) {
    // (magnitudes are ordered as their codes are, NaN, 0x7F, above all)
    s2 lo = {0, 0}, hi = {0, 0};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      lo = __builtin_elementwise_max(lo, __builtin_bit_cast(s2, v[c] & 0x007F007Fu));
      hi = __builtin_elementwise_max(hi, __builtin_bit_cast(s2, v[c] & 0x7F007F00u));
    }
    const auto low = __builtin_bit_cast(uint32_t, lo), high = __builtin_bit_cast(uint32_t, hi) >> 8;
    uint32_t top = max(max(low & 0xFFFFu, low >> 16), max(high & 0xFFu, high >> 16));
    if (top == 0x7Fu) {                       // (NaN codes count as 0)
      top = 0;
#pragma unroll
      for (int c = 0; c < 16; ++c) {
        const uint32_t x = v[c >> 2] >> (8 * (c & 3)) & 0x7Fu;
        top = max(top, x == 0x7Fu ? 0u : x);
      }
    }
    return __builtin_amdgcn_cvt_f32_fp8((int)top, 0);
  } else {
    s2 up = {0, 0}, down = {0, 0};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t w = v[c];                // (a bit cast of an element itself takes the first one)
      const s2 even = __builtin_bit_cast(s2, w << 8) >> 8, odd = __builtin_bit_cast(s2, w) >> 8;
      up = __builtin_elementwise_max(__builtin_elementwise_max(up, even), odd);
      down = __builtin_elementwise_min(__builtin_elementwise_min(down, even), odd);
    }
    return (float)max(max((int)up.x, (int)up.y), -min((int)down.x, (int)down.y));
  }
}

// One wavefront per (request, KV head, block below the budget, side).  A block of which every row stays is left as it
// is. Another one's scale is the smallest power of two that holds its rows' values, as if they were stored anew; a row
// that stays is written again only if the scale changed.
//
// Bytes and latency bound it.  Lane r has row r's source and scale (K's wavefronts: its weight and position); then 16
// bytes of a row at a time.  64 requests x 8 heads, D 128, 4,160 entries cut to 4,096, e4m3 (some 186 MB): 47 us, 4.0
// TB/s; with a workgroup of 256 threads per block, one side after the other 74, both sides at once 69, a wavefront for
// both sides 56.
template <int CODE, int D, int B>
__global__ __launch_bounds__(256) void evict_kernel(const Evict P) {
  constexpr int LOG2B = B == 16 ? 4 : B == 32 ? 5 : 6;
  constexpr int TPR = D / 16, NP = B * TPR / 64;             // lanes per row; units of a lane and side
  const int lane = threadIdx.x & 63, w = blockIdx.x * 4 + uniform((int)threadIdx.x >> 6);
  const int h = blockIdx.y, j = blockIdx.z;
  const int lp = w >> 1, side = w & 1;
  if (lp >= P.budget >> LOG2B) return;
  const int row = P.rows ? uniform(P.rows[j]) : j;
  if (row < 0 || row >= P.n_rows) return;
  const int64_t tbl = row * P.stride;
  const int e = (lp << LOG2B) + lane;
  const int s = lane < B ? P.src[((int64_t)j * P.H + h) * P.budget + e] : -1;
  const int block = uniform(P.table[tbl + lp]);
  const int len = (int)min((int64_t)max(uniform(P.kv_lens[j]), 0), P.cap);
  if (len <= P.budget) return;
  const bool comes = block >= 0 && block < P.n_blocks && s >= P.budget && s < len;
  int held = 0, gone = 0;
  const bool has_pos = P.pos && side == 0;
  if (has_pos) held = uniform(P.held[row]), gone = uniform(P.evicted[row]);
  int32_t* pos = P.pos + (row * P.sp_r + h * P.sp_h);
  if (!__any(comes)) {
    if (has_pos && lane < B && e >= held) pos[e] = e + gone;
    return;
  }
  int b = comes ? P.table[tbl + (s >> LOG2B)] : block;
  const bool moves = comes && b >= 0 && b < P.n_blocks;
  if (!moves) b = block;
  const int64_t from = ((((int64_t)b * P.H + h) << LOG2B) + ((moves ? s : e) & (B - 1))) * D;
  const int from_lo = (int)(uint32_t)from, from_hi = (int)(from >> 32);
  uint8_t* codes = side ? P.codes[1] : P.codes[0];
  float* scales = side ? P.scale[1] : P.scale[0];
  const float scale = scales[(int64_t)b * P.H + h];
  const uint64_t moved = __ballot(moves);
  const int64_t to = (((int64_t)block * P.H + h) << LOG2B) * D;
  auto row_of = [&](int i) { return (lane + 64 * i) / TPR; };
  u4v x[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const uint32_t lo = (uint32_t)__shfl(from_lo, row_of(i), 64), hi = (uint32_t)__shfl(from_hi, row_of(i), 64);
    x[i] = *reinterpret_cast<const u4v*>(codes + (int64_t)((uint64_t)hi << 32 | lo) + 16 * (lane % TPR));
  }
  if (lane < B) {
    if (P.weights && side == 0 && moves) {
      float* x = P.weights + (row * P.sw_r + h * P.sw_h);
      x[e] = x[s];
    }
    if (has_pos) {
      const int at = moves ? s : e;
      if (moves || e >= held) pos[e] = at < held ? pos[at] : at + gone;
    }
  }
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const float f = __shfl(scale, row_of(i), 64);
    // (infinity: a scale that is not finite)
    top = fmaxf(top, f - f == 0.0f ? fminf(magnitude<CODE>(x[i]) * f, 3.402823466e38f) : __builtin_inff());
  }
  top = group_max<64>(top);
  const bool finite = top < __builtin_inff();
  const float size = finite ? pow2_scale<CODE>(top) : __builtin_nanf(""), inv = 1.0f / size;
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int r = row_of(i);
    const float f = __shfl(scale, r, 64);
    const bool kept = f == size || !finite;                  // (not finite: the codes as they are)
    if (kept && !(moved >> r & 1)) continue;
    u4v o = x[i];
    if (!kept) {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float y[4];
        unpack4<CODE>(x[i][c], y);
        o[c] = pack4<CODE>(y[0] * f * inv, y[1] * f * inv, y[2] * f * inv, y[3] * f * inv);
      }
    }
    *reinterpret_cast<u4v*>(codes + to + (64 * i + lane) * 16) = o;
  }
  if (lane == 0) scales[(int64_t)block * P.H + h] = size;
}

template <int CODE, int D>
void evict_launch(const Evict& P, hipStream_t st) {
  const dim3 grid(((P.budget >> P.log2b) + 1) / 2, P.H, P.n);
  if (P.log2b == 4) evict_kernel<CODE, D, 16><<<grid, 256, 0, st>>>(P);
  else if (P.log2b == 5) evict_kernel<CODE, D, 32><<<grid, 256, 0, st>>>(P);
  else evict_kernel<CODE, D, 64><<<grid, 256, 0, st>>>(P);
}
template <int CODE>
void evict_launch_d(const Evict& P, int D, hipStream_t st) {
  if (D == 64) evict_launch<CODE, 64>(P, st);
  else if (D == 128) evict_launch<CODE, 128>(P, st);
  else evict_launch<CODE, 256>(P, st);
}

// ---------------------------------------------------------------------------------------------------------------- trim
constexpr int kMaxTrim = 1024, kStamps = 4096;
constexpr int kFewRounds = 4;         // of one workgroup's wavefronts
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

// One workgroup, where its 16 wavefronts have few rounds of a request and 64 blocks each: a thread per request finds its
// length and whether an earlier request has its row, a wavefront per request counts the blocks that it gives back, and
// after a scan writes them in request order.  us on the device, this / the two launches below: 64 requests of one block,
// or 64, 5.9 / 5.3, 16 of 256 5.0 / 5.2 (one launch less for the host, 2 - 3 us); 64 of 128 7.5 / 5.3, 256 of 16 14.8 /
// 5.5, one of 4,096 23.9 / 9.5, 200 of 400 40.4 / 6.0.
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

// Many entries behind the budget: a workgroup per request, in two launches.  The first one says of request j: its table
// row (-1: none, or one that an earlier request has), length and how many blocks it gives back.
struct Back { int row, len, count, pad; };

__global__ __launch_bounds__(256) void trim_count_kernel(const Trim P, Back* back) {
  __shared__ int total;
  const int j = blockIdx.x, t = threadIdx.x, lane = t & 63;
  const int row = uniform(P.seqs[j]);
  bool bad = row < 0 || row >= P.rows;
  for (int i = t; i < j; i += 256) bad |= P.seqs[i] == row;
  if (t == 0) total = 0;
  bad = __syncthreads_or(bad);
  const int len = bad ? 0 : max(uniform(P.seq_lens[row]), 0);
  const int last = (int)min(((int64_t)len + (1 << P.log2b) - 1) >> P.log2b, (int64_t)P.max_blocks);
  int c = 0;
#pragma unroll 4
  for (int lp = (P.budget >> P.log2b) + t; lp < last; lp += 256) {
    const int id = P.table[row * P.stride + lp];
    c += id >= 0 && id < P.n_free;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) c += __shfl_xor(c, o, 64);
  if (lane == 0) atomicAdd(&total, c);
  __syncthreads();
  if (t == 0) {
    back[j] = {bad ? -1 : row, len, total, 0};
    P.kv_lens[j] = min(len, P.budget);
    if (j == 0) back[P.n] = {min(max(*P.free_head, 0), P.n_free), 0, 0, 0};
    if (bad && P.status) atomicOr(P.status, kBadRow);
  }
}

__global__ __launch_bounds__(256) void trim_write_kernel(const Trim P, const Back* back) {
  __shared__ int sums[2][4];
  const int j = blockIdx.x, t = threadIdx.x, lane = t & 63, wave = t >> 6;
  const Back my = back[j];
  const int head = back[P.n].row;
  int earlier = 0, total = 0;
  for (int i = t; i < P.n; i += 256) {
    const int c = back[i].count;
    total += c, earlier += i < j ? c : 0;
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) total += __shfl_xor(total, o, 64), earlier += __shfl_xor(earlier, o, 64);
  if (lane == 0) sums[0][wave] = total, sums[1][wave] = earlier;
  __syncthreads();
  total = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
  int to = head - total + sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
  if (j == 0 && t == 0) {
    *P.next_head = max(head - total, 0);
    if (P.commit) *P.free_head = max(head - total, 0);
    if (total > head && P.status) atomicOr(P.status, kFreeOver);
  }
  if (my.row < 0 || my.len <= P.budget) return;
  const int first = P.budget >> P.log2b;
  const int last = (int)min(((int64_t)my.len + (1 << P.log2b) - 1) >> P.log2b, (int64_t)P.max_blocks);
  int32_t* table = P.table + my.row * P.stride;
  for (int base = first; base < last; base += 256) {
    const int lp = base + t;
    const int id = lp < last ? table[lp] : -1;
    const bool is = id >= 0 && id < P.n_free;
    const uint64_t b = __ballot(is);
    __syncthreads();                            // (the sums of the round before have been read)
    if (lane == 0) sums[0][wave] = __popcll(b);
    __syncthreads();
    int k = to + __popcll(b & (((uint64_t)1 << lane) - 1));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      k += i < wave ? sums[0][i] : 0;
      to += sums[0][i];
    }
    if (is && k >= 0) P.free_list[k] = id;
    if (lp < last && P.commit) table[lp] = -1;
  }
  if (P.commit && t == 0) {
    P.seq_lens[my.row] = P.budget;
    if (P.evicted) P.evicted[my.row] += my.len - P.budget, P.held[my.row] = P.budget;
  }
}

}  // namespace

extern "C" int kvt_block_keep(const void* weights, int64_t sw_r, int64_t sw_h, const void* kv_lens, int n, int H,
                              int n_rows, const void* rows, int64_t cap, int budget, int recent, int sinks, const void* pos,
                              int64_t sp_r, int64_t sp_h, const void* held, const void* evicted, void* src, void* work,
                              int64_t work_ints, void* stream) {
  if (n < 1 || H < 1 || n_rows < 1 || cap < 1 || budget < 1 || recent < 0 || sinks < 0 || (!rows && n_rows < n))
    return KVT_EINVAL;
  if ((int64_t)recent + sinks > budget || !pos != !held || !pos != !evicted) return KVT_EINVAL;
  const int64_t pairs = (int64_t)n * H;
  const int chunks = (int)max(min(min((cap + kChunk - 1) / kChunk, (int64_t)kMostChunks), kChunkBlocks / pairs), (int64_t)1);
  if (cap > ((int64_t)1 << 31) - 8192 || pairs >= 1 << 22) return KVT_ERANGE;
  Keep P;
  P.weights = (const float*)weights, P.kv_lens = (const int32_t*)kv_lens, P.rows = (const int32_t*)rows;
  P.pos = (const int32_t*)pos, P.held = (const int32_t*)held, P.evicted = (const int32_t*)evicted;
  P.src = (int32_t*)src, P.work = (int32_t*)work, P.sw_r = sw_r, P.sw_h = sw_h, P.sp_r = sp_r, P.sp_h = sp_h, P.cap = cap;
  P.n = n, P.n_rows = n_rows, P.H = H, P.budget = budget, P.recent = recent, P.sinks = sinks, P.chunks = chunks;
  const bool many = cap > kSmall && cap > budget;
  if (many && (((uintptr_t)work & 15) || work_ints < pairs * (3 * kBins + 4 * chunks + 12 + 2 * (((int64_t)budget + 1) & ~1))))
    return KVT_EINVAL;
  hipStream_t st = (hipStream_t)stream;
  keep_kernel<512, kFew / 512, 0><<<(int)pairs, 512, 0, st>>>(P);
  KVT_CHECK_LAUNCH();
  if (cap > kFew && cap > budget) {
    keep_kernel<1024, kSmall / 1024, kFew><<<(int)pairs, 1024, 0, st>>>(P);
    KVT_CHECK_LAUNCH();
  }
  if (!many) return KVT_OK;
  // (a launch has fewer than 2^32 threads; the workgroups of a pair take turns)
  const int grid = (int)pairs * chunks, blocks = max(min(min((budget + 255) / 256, 64), (int)(((1 << 24) - 1) / pairs)), 1);
  for (int pass = 0; pass < 3; ++pass) {
    keep_hist_kernel<<<grid, kKeepThreads, 0, st>>>(P, pass);
    KVT_CHECK_LAUNCH();
  }
  keep_count_kernel<<<grid, kKeepThreads, 0, st>>>(P);
  KVT_CHECK_LAUNCH();
  keep_list_kernel<<<grid, kKeepThreads, 0, st>>>(P);
  KVT_CHECK_LAUNCH();
  keep_place_kernel<<<(int)pairs * blocks, 256, 0, st>>>(P, blocks);
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
  if (n > 65535 || H > 65535 || (int64_t)n * H * (budget / block + 1) >= 1 << 25 ||   // (2^32 threads)
      (int64_t)max_blocks * block > ((int64_t)1 << 31) - 8192 ||
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
  if (code == kE4M3) evict_launch_d<kE4M3>(P, D, (hipStream_t)stream);
  else evict_launch_d<kI8>(P, D, (hipStream_t)stream);
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}

extern "C" int kvt_block_trim(int n, const void* seqs, void* seq_lens, int rows, void* block_table, int64_t bt_stride,
                              int max_blocks, void* free_list, int n_free, void* free_head, int block, int budget,
                              void* held, void* evicted, void* kv_lens, void* next_head, void* status, int commit,
                              void* work, void* stream) {
  if (n < 1 || n > kMaxTrim || rows < 1 || max_blocks < 1 || bt_stride < max_blocks || n_free < 0) return KVT_EINVAL;
  if ((block != 16 && block != 32 && block != 64) || budget < block || budget % block || !held != !evicted) return KVT_EINVAL;
  if (!work || (uintptr_t)work & 15) return KVT_EINVAL;
  Trim P;
  P.seqs = (const int32_t*)seqs, P.seq_lens = (int32_t*)seq_lens, P.table = (int32_t*)block_table;
  P.free_list = (int32_t*)free_list, P.free_head = (int32_t*)free_head, P.held = (int32_t*)held;
  P.evicted = (int32_t*)evicted, P.kv_lens = (int32_t*)kv_lens, P.next_head = (int32_t*)next_head;
  P.status = (int32_t*)status, P.stride = bt_stride, P.n = n, P.rows = rows, P.max_blocks = max_blocks;
  P.n_free = n_free, P.log2b = block == 16 ? 4 : block == 32 ? 5 : 6, P.budget = budget, P.commit = commit;
  const int64_t behind = max(max_blocks - budget / block, 0);
  if ((n + kWaves - 1) / kWaves * ((behind + 63) / 64) <= kFewRounds) {
    trim_kernel<<<1, 1024, 0, (hipStream_t)stream>>>(P);
  } else {
    trim_count_kernel<<<n, 256, 0, (hipStream_t)stream>>>(P, (Back*)work);
    KVT_CHECK_LAUNCH();
    trim_write_kernel<<<n, 256, 0, (hipStream_t)stream>>>(P, (const Back*)work);
  }
  KVT_CHECK_LAUNCH();
  return KVT_OK;
}
