// Block tables and slot maps from request lengths, on the device, in one launch.
//
// Request b holds c_b tokens in its pages and gets n_b new ones.  With pages of
// `bs` slots it has ceil(c_b / bs) pages and needs ceil((c_b + n_b) / bs); the
// missing ones come from the free list in request order:
//   off_b = sum_{i<b} (need_i - have_i),  table[b, have_b + j] = free[off_b + j].
// The new tokens of all requests are packed: token t of request b (start_b =
// sum_{i<b} n_i) has position p = c_b + t - start_b and slot
//   page(b, p / bs) * bs + p % bs.
//
// Two prefix sums over the requests and then independent work per token and
// per new page.  No block waits for another: every block sums the lengths
// itself (8 bytes a request, from L2), keeps one partial sum per thread in
// shared memory, and takes an even share of the tokens, of the new pages and
// of the requests.  A token's page is read from the table only in columns the
// request had before, and from the free list otherwise, so no block depends on
// table entries written by another.  Bound by the launch for a decode batch and
// by the 20 bytes written per token for prompts.
#include <algorithm>

#include "common.cuh"
#include "serving_ops.h"

namespace lmc {
namespace {

constexpr int kSlotThreads = 512;
constexpr int kMostTokens = 4096;  // of a block, in whole turns of its threads

enum SlotWhere : int { kWhereLength = 1, kWhereTable = 2, kWhereFree = 3, kWhereTotal = 4 };

struct Need {
  unsigned tokens, pages;
};

// Positions stay below 2^32 (two lengths below 2^31); a power of two, as block
// sizes mostly are, takes a shift.
__device__ __forceinline__ unsigned page_of(const SlotArgs &a, unsigned position) {
  return a.block_shift >= 0 ? position >> a.block_shift
                            : position / static_cast<unsigned>(a.block_size);
}

// Pages of `tokens` slots.
__device__ __forceinline__ unsigned pages_of(const SlotArgs &a, unsigned tokens) {
  const unsigned whole = page_of(a, tokens);
  return whole + (tokens != whole * static_cast<unsigned>(a.block_size));
}

template <typename LT>
__device__ __forceinline__ unsigned length_of(const void *p, int b) {
  const long long v = static_cast<long long>(static_cast<const LT *>(p)[b]);
  // a length below zero counts as zero; one past 2^31 - 1 as that
  return static_cast<unsigned>(v < 0 ? 0 : (v > 0x7fffffffll ? 0x7fffffffll : v));
}

template <typename LT>
__device__ __forceinline__ Need need_of(const SlotArgs &a, int b) {
  const unsigned c = length_of<LT>(a.ctx, b), n = length_of<LT>(a.fresh, b);
  return {n, a.grow ? pages_of(a, c + n) - pages_of(a, c) : 0};
}

// Exclusive prefix of the request sums at each thread's segment of requests.
struct Sums {
  long long tokens[kSlotThreads + 1];
  long long pages[kSlotThreads + 1];
};

// Largest i with v[i] <= x (v ascending, v[0] = 0 <= x).
__device__ __forceinline__ int last_leq(const long long *v, int n, long long x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <typename LT, typename OT>
__global__ void __launch_bounds__(kSlotThreads) slot_mapping_kernel(SlotArgs a, int per_block) {
  __shared__ Sums s;
  __shared__ long long warp_tok[kSlotThreads / 32], warp_pg[kSlotThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seg = (a.batch + kSlotThreads - 1) / kSlotThreads;
  const int b0 = min(a.batch, tid * seg), b1 = min(a.batch, b0 + seg);
  struct {
    long long tokens, pages;
  } mine = {0, 0};
  for (int b = b0; b < b1; ++b) {
    const Need n = need_of<LT>(a, b);
    mine.tokens += n.tokens;
    mine.pages += n.pages;
  }
  long long ti = mine.tokens, pi = mine.pages;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, ti, o), y = __shfl_up_sync(0xffffffffu, pi, o);
    if (lane >= o) ti += x, pi += y;
  }
  if (lane == 31) warp_tok[warp] = ti, warp_pg[warp] = pi;
  __syncthreads();
  long long tb = 0, pb = 0;
  for (int w = 0; w < warp; ++w) tb += warp_tok[w], pb += warp_pg[w];
  s.tokens[tid] = tb + ti - mine.tokens;
  s.pages[tid] = pb + pi - mine.pages;
  if (tid == kSlotThreads - 1) s.tokens[kSlotThreads] = tb + ti, s.pages[kSlotThreads] = pb + pi;
  __syncthreads();
  const long long total_tokens = s.tokens[kSlotThreads], total_pages = s.pages[kSlotThreads];

  // --- per request: this block's share is written by the threads that summed it
  const int share = (a.batch + gridDim.x - 1) / gridDim.x;
  const int r0 = blockIdx.x * share, r1 = min(a.batch, r0 + share);
  if (b0 < r1 && b1 > r0) {
    long long t = s.tokens[tid], p = s.pages[tid];
    for (int b = b0; b < b1; ++b) {
      const Need n = need_of<LT>(a, b);
      if (b >= r0 && b < r1) {
        const unsigned c = length_of<LT>(a.ctx, b);
        a.start[b] = static_cast<int>(t);
        a.taken[b] = static_cast<int>(p);
        a.seq_lens[b] = static_cast<int>(min(c + n.tokens, 0x7fffffffu));
        if (static_cast<long long>(static_cast<const LT *>(a.ctx)[b]) != c ||
            static_cast<long long>(static_cast<const LT *>(a.fresh)[b]) != n.tokens)
          report_status(a.status, kStatusBadIndex, kWhereLength, b, 0);
        if (b == a.batch - 1) {
          a.start[a.batch] = static_cast<int>(t + n.tokens);
          a.taken[a.batch] = static_cast<int>(p + n.pages);
        }
      }
      t += n.tokens;
      p += n.pages;
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    if (a.batch == 0) a.start[0] = 0, a.taken[0] = 0;
    if (total_tokens > a.num_tokens)
      report_status(a.status, kStatusBadIndex, kWhereTotal, total_tokens, a.num_tokens);
    if (total_pages > a.num_free)
      report_status(a.status, kStatusBadIndex, kWhereFree, total_pages, a.num_free);
  }

  // --- new pages into the tables
  for (long long j = static_cast<long long>(blockIdx.x) * kSlotThreads + tid; j < total_pages;
       j += static_cast<long long>(gridDim.x) * kSlotThreads) {
    const int g = last_leq(s.pages, kSlotThreads, j);
    int b = g * seg;
    long long p = s.pages[g];
    long long n = need_of<LT>(a, b).pages;
    while (j >= p + n) {
      p += n;
      n = need_of<LT>(a, ++b).pages;
    }
    const long long col = pages_of(a, length_of<LT>(a.ctx, b)) + (j - p);
    if (col < a.width)
      a.tables[b * a.table_stride + col] = j < a.num_free ? a.free_blocks[j] : -1;
    else
      report_status(a.status, kStatusBadIndex, kWhereTable, b, col);
  }

  // --- tokens: a warp takes some hundred in a row, mostly of one request, which it
  // looks up once; where requests are short each lane looks up its own
  OT *slots = static_cast<OT *>(a.slots);
  OT *positions = static_cast<OT *>(a.positions);
  const int per_warp = per_block / (kSlotThreads / 32);
  const long long t0 = static_cast<long long>(blockIdx.x) * per_block + warp * per_warp;
  const long long t1 = min(a.num_tokens, t0 + per_warp);
  if (t0 >= t1) return;
  // (tokens and pages up to the last row of the outputs fit 32 bits)
  int b = 0;
  unsigned start = 0, pages = 0, c = 0, have = 0;
  Need n = {0, 0};
  auto look_up = [&](int request) {
    b = request;
    c = length_of<LT>(a.ctx, b);
    n = need_of<LT>(a, b);
    have = pages_of(a, c);
  };
  // the request of token t: the last segment of requests that starts at or before
  // it, then the few requests of the segment
  auto find = [&](unsigned t) {
    const int g = last_leq(s.tokens, kSlotThreads, t);
    start = static_cast<unsigned>(s.tokens[g]), pages = static_cast<unsigned>(s.pages[g]);
    look_up(g * seg);
    while (t - start >= n.tokens) {
      start += n.tokens;
      pages += n.pages;
      look_up(b + 1);
    }
  };
  const unsigned end = static_cast<unsigned>(min(t1, total_tokens));
  if (t0 < total_tokens) find(static_cast<unsigned>(t0));
  for (unsigned t = static_cast<unsigned>(t0) + lane; t < static_cast<unsigned>(t1); t += 32) {
    if (t >= end) {  // rows behind the last request
      slots[t] = -1;
      positions[t] = 0;
      a.request_ids[t] = -1;
      continue;
    }
    if (t - start >= n.tokens) {  // mostly the next request's
      start += n.tokens;
      pages += n.pages;
      look_up(b + 1);
      if (t - start >= n.tokens) find(t);
    }
    const unsigned pos = c + (t - start);
    const unsigned col = page_of(a, pos);
    int page = -1;
    if (col >= static_cast<unsigned>(a.width)) {
      report_status(a.status, kStatusBadIndex, kWhereTable, b, col);
    } else if (a.grow && col >= have) {
      const unsigned j = pages + (col - have);
      if (j < a.num_free) page = a.free_blocks[j];
    } else {
      page = a.tables[b * a.table_stride + col];
    }
    OT slot = -1;
    if (page >= 0 && page < a.num_blocks)
      slot = static_cast<OT>(page) * a.block_size + static_cast<OT>(pos - col * a.block_size);
    else if (col < static_cast<unsigned>(a.width))
      report_status(a.status, kStatusBadSlot, b, page, a.num_blocks);
    slots[t] = slot;
    positions[t] = static_cast<OT>(pos);
    a.request_ids[t] = b;
  }
}

}  // namespace

cudaError_t launch_slot_mapping(const SlotArgs &a, bool long_lens, bool long_slots,
                                cudaStream_t stream) {
  // few tokens on many blocks, but every block sums all lengths: 1000 requests of
  // one to eight new tokens 16.1 -> 6.1 us against blocks of kMostTokens, while 1M
  // tokens took 12.0 us instead of 9.1 on three blocks per SM
  const long long even = (a.num_tokens + 148 * 2 - 1) / (148 * 2);
  const long long turns = std::max(1ll, (even + kSlotThreads - 1) / kSlotThreads);
  const int per_block = static_cast<int>(std::min(1ll * kMostTokens, turns * kSlotThreads));
  const unsigned grid =
      static_cast<unsigned>(std::max(1ll, (a.num_tokens + per_block - 1) / per_block));
#define LMC_SLOTS(LT, OT) \
  slot_mapping_kernel<LT, OT><<<grid, kSlotThreads, 0, stream>>>(a, per_block)
  if (!long_lens) {
    if (long_slots) LMC_SLOTS(int, long long); else LMC_SLOTS(int, int);
  } else {
    if (long_slots) LMC_SLOTS(long long, long long); else LMC_SLOTS(long long, int);
  }
#undef LMC_SLOTS
  return cudaGetLastError();
}

}  // namespace lmc
