// Block tables and slot maps of a step, from the requests' lengths on the device (kvt_block_plan).
//
// Request j (table row s = seqs[j], L0 = seq_lens[s] tokens held) appends c = counts[j] tokens at positions L0 .. L0 +
// c - 1.  It opens the blocks ceil(L0 / B) .. ceil((L0 + c) / B) - 1, which take the next entries of the free list in
// request order; position p goes to slot block * B + p % B.  With exclusive prefix sums C of the token counts and O of
// the opened blocks, token t of request j (C_j <= t < C_j+1) has p = L0 + t - C_j, and an opened block lp is
// free_list[head + O_j + lp - ceil(L0 / B)]: every token's slot follows from the sums alone.
//
// A block of 1,024 threads scans the (at most 1,024) requests by itself, keeps the sums in LDS and writes the slots of
// 4,096 tokens, four per thread (one 16-byte store): no second launch, no communication.  With `commit`, lengths and
// head advance in the same launch when it has one block, else in a launch behind it (other blocks may still be reading
// them).  Launch and load latency bound it: 64 requests of one token 6.0 us, 512 requests and 538,000 tokens with
// req_to_token 8.3 (4.6 MB written, 132 blocks that all scan).
#include "block_common.h"

using namespace kvt;

namespace {

constexpr int kThreads = 1024;
constexpr int kMaxPlan = 1024;                 // requests of one plan
constexpr int kTokens = 4 * kThreads;          // tokens per block
constexpr int kStamps = 4096;
enum { kPoolShort = 1, kRowFull = 2, kTokensOver = 4, kBadRow = 8 };

struct Plan {
  const int32_t* seqs;
  const int32_t* counts;
  int32_t* seq_lens;
  int32_t* table;
  const int32_t* free_list;
  int32_t* free_head;
  int32_t* cu;
  int32_t* slots;
  int32_t* kv_lens;
  int32_t* next_head;
  int32_t* status;
  int32_t* rtt;
  int64_t stride, rtt_stride;
  int n, rows, max_blocks, n_free, log2b, n_tokens, rtt_cols, commit;
};

struct Lds {
  int32_t cu[kMaxPlan + 1];
  int32_t row[kMaxPlan];        // -1: a row outside the tables, or a row that an earlier request of the plan has
  int32_t len[kMaxPlan];
  int32_t base[kMaxPlan];       // O_j - ceil(L0 / B): an opened block lp takes entry head + base + lp
  int32_t stamp[kStamps];
  int64_t sums[2][kThreads / 64];
  int32_t flags;
};

// Inclusive sum over the block's threads; sums: one partial per wavefront.
KVT_DEV int64_t block_scan(int64_t v, int64_t* sums) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  if (lane == 63) sums[w] = v;
  __syncthreads();
  int64_t before = 0;
  for (int i = 0; i < w; ++i) before += sums[i];
  return v + before;
}

__global__ __launch_bounds__(kThreads) void block_plan_kernel(const Plan P) {
  __shared__ Lds S;
  const int j = threadIdx.x;
  const int B = 1 << P.log2b;
  if (j == 0) S.flags = 0;
  for (int i = j; i < kStamps; i += kThreads) S.stamp[i] = kMaxPlan;
  int row = -1;
  if (j < P.n) {
    row = P.seqs[j];
    if (row < 0 || row >= P.rows) row = -1;
    S.row[j] = row;
  }
  __syncthreads();
  if (row >= 0) atomicMin(&S.stamp[row & (kStamps - 1)], j);
  __syncthreads();
  bool bad = j < P.n && row < 0;
  if (row >= 0) {   // a row that an earlier request has: the first one keeps it
    const int w = S.stamp[row & (kStamps - 1)];
    if (w != j) {
      bool twice = S.row[w] == row;
      if (!twice)   // (more than 4,096 table rows: another row has the stamp)
        for (int i = 0; i < j && !twice; ++i) twice = S.row[i] == row;
      bad = twice;
    }
  }
  __syncthreads();
  if (bad) S.row[j] = row = -1;
  int len = 0, count = 0;
  if (row >= 0) {
    len = max(P.seq_lens[row], 0);
    count = max(P.counts[j], 0);     // (the sums are 64 bits: not cut to n_tokens before kTokensOver is looked for)
  }
  const int64_t upto = block_scan(count, S.sums[0]);
  const int c1 = (int)min(upto, (int64_t)P.n_tokens), c0 = (int)min(upto - count, (int64_t)P.n_tokens);
  const int64_t end = (int64_t)len + (c1 - c0);
  const int first = (int)(((int64_t)len + B - 1) >> P.log2b);
  const int64_t last = (end + B - 1) >> P.log2b;
  const int opens = (int)max(min(last, (int64_t)P.max_blocks) - first, (int64_t)0);
  const int64_t taken = block_scan(opens, S.sums[1]);
  const int head = min(max(*P.free_head, 0), P.n_free);
  if (j < P.n) {
    if (j == 0) S.cu[0] = 0;
    S.cu[j + 1] = c1;
    S.len[j] = len;
    S.base[j] = (int)min(taken - opens, (int64_t)P.n_free) - first;
    int f = (bad ? kBadRow : 0) | (upto > P.n_tokens ? kTokensOver : 0) |
            (c1 > c0 && last > P.max_blocks ? kRowFull : 0) | (head + taken > P.n_free ? kPoolShort : 0);
    if (f) atomicOr(&S.flags, f);
  }
  __syncthreads();
  if (blockIdx.x == 0) {
    if (j < P.n) {
      if (j == 0) P.cu[0] = 0;
      P.cu[j + 1] = c1;
      P.kv_lens[j] = (int)min(end, (int64_t)0x7FFFFFFF);
    }
    if (j == P.n - 1) {
      const int next = (int)min(head + taken, (int64_t)P.n_free);
      *P.next_head = next;
      if (P.status && S.flags) atomicOr(P.status, S.flags);
      if (P.commit && gridDim.x == 1) *P.free_head = next;
    }
    if (P.commit && gridDim.x == 1 && c1 > c0) P.seq_lens[row] = (int)min(end, (int64_t)0x7FFFFFFF);
  }

  // the slots of this block's tokens
  const int t0 = blockIdx.x * kTokens + 4 * j;
  if (t0 >= P.n_tokens) return;
  const int total = S.cu[P.n];
  int r = 0;   // the last request with cu <= t0
  for (int lo = 0, hi = P.n; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (S.cu[mid] <= t0) lo = mid; else hi = mid;
    r = lo;
  }
  int slot[4], seen = -1, id = -1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + i;
    slot[i] = -1;
    if (t >= total) continue;
    int moved = 0;
    while (S.cu[r + 1] <= t) ++r, moved = 1;
    const int64_t p = (int64_t)S.len[r] + (t - S.cu[r]);
    const int64_t lp64 = p >> P.log2b;
    if (lp64 >= P.max_blocks) continue;
    const int lp = (int)lp64, s = S.row[r];
    if (moved || lp != seen) {
      seen = lp;
      const bool open = lp < ((S.len[r] + (int64_t)B - 1) >> P.log2b);   // the block that the request holds already
      const int at = head + S.base[r] + lp;
      id = open ? P.table[s * P.stride + lp] : at < P.n_free ? P.free_list[at] : -1;
    }
    if ((p & (B - 1)) == 0) P.table[s * P.stride + lp] = id;
    if (id >= 0) slot[i] = (id << P.log2b) + (int)(p & (B - 1));
    if (P.rtt && p < P.rtt_cols) P.rtt[s * P.rtt_stride + p] = slot[i];
  }
  if (t0 + 4 <= P.n_tokens && ((uintptr_t)P.slots & 15) == 0) {
    *reinterpret_cast<int4*>(P.slots + t0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
  } else {
    for (int i = 0; i < 4 && t0 + i < P.n_tokens; ++i) P.slots[t0 + i] = slot[i];
  }
}

// Lengths and head of a plan of several blocks (a request that appends nothing keeps its length: it may be one that the
// plan left out).
__global__ __launch_bounds__(kThreads) void block_commit_kernel(const Plan P) {
  const int j = threadIdx.x;
  if (j < P.n && P.cu[j + 1] > P.cu[j]) P.seq_lens[P.seqs[j]] = P.kv_lens[j];
  if (j == 0) *P.free_head = *P.next_head;
}

}  // namespace

extern "C" int kvt_block_plan(int n, const void* seqs, const void* counts, void* seq_lens, int rows, void* block_table,
                              int64_t bt_stride, int max_blocks, const void* free_list, int n_free, void* free_head,
                              int block, int n_tokens, void* cu, void* slots, void* kv_lens, void* next_head,
                              void* status, void* req_to_token, int64_t rtt_stride, int rtt_cols, int commit,
                              void* stream) {
  if (n < 1 || n > kMaxPlan || rows < 1 || max_blocks < 1 || bt_stride < max_blocks || n_free < 0 || n_tokens < 0)
    return KVT_EINVAL;
  if (block != 16 && block != 32 && block != 64) return KVT_EINVAL;
  if (req_to_token && (rtt_cols < 1 || rtt_stride < rtt_cols)) return KVT_EINVAL;
  if (n_tokens > (1 << 30) || (int64_t)n_free * block > ((int64_t)1 << 31)) return KVT_ERANGE;   // (int32 slots)
  Plan P;
  P.seqs = (const int32_t*)seqs, P.counts = (const int32_t*)counts, P.seq_lens = (int32_t*)seq_lens;
  P.table = (int32_t*)block_table, P.free_list = (const int32_t*)free_list, P.free_head = (int32_t*)free_head;
  P.cu = (int32_t*)cu, P.slots = (int32_t*)slots, P.kv_lens = (int32_t*)kv_lens, P.next_head = (int32_t*)next_head;
  P.status = (int32_t*)status, P.rtt = (int32_t*)req_to_token, P.stride = bt_stride, P.rtt_stride = rtt_stride;
  P.n = n, P.rows = rows, P.max_blocks = max_blocks, P.n_free = n_free, P.log2b = block == 16 ? 4 : block == 32 ? 5 : 6;
  P.n_tokens = n_tokens, P.rtt_cols = rtt_cols, P.commit = commit;
  const int grid = n_tokens > kTokens ? (n_tokens + kTokens - 1) / kTokens : 1;
  block_plan_kernel<<<grid, kThreads, 0, (hipStream_t)stream>>>(P);
  KVT_CHECK_LAUNCH();
  if (commit && grid > 1) {
    block_commit_kernel<<<1, kThreads, 0, (hipStream_t)stream>>>(P);
    KVT_CHECK_LAUNCH();
  }
  return KVT_OK;
}
