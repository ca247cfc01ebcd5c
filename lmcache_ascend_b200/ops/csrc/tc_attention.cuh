// Attention of many rows over a stream of keys on the tensor cores.
//
// A block owns 256 rows of one KV head, as two tiles of 128: rows are (token,
// query head of the group) pairs, token-major, so heads that share keys share
// their loads whatever the group's size.  Keys come in tiles of 128.  Per key
// tile and row tile
//   S = Q K^T            tcgen05, both operands in shared memory, S in TMEM
//   P = exp2(S c - m)    two threads per row, 64 keys each: S from TMEM to
//                        registers, running maximum m (common) and sum l (of
//                        each), P as 16-bit back over S in TMEM
//   O = O + P V          tcgen05, P from TMEM, V as it lies (MN-major); begun
//                        when half of P is there
// While one tile's scores are in the registers the tensor cores work on the
// other's.  m only moves when the maximum grows by more than 2^8, so O in TMEM
// is seldom rescaled (by the thread that owns the row; P stays below 2^8, or 2^15
// in float16, see kRaised, and sums are fp32).
//
// Roles: warps 0-7 and 8-15 one row tile each, warp 16 issues the mma, warp 17
// the TMA loads through a ring of two stages, each with the K of a tile and the V
// of the one before, which one turn of the mma loop uses (one wait for both); they
// give registers to the others (640 threads x 96 at launch = 512 x 112 + 128 x
// 32).  Eight warps a tile, because a tile's chain (scores, weights, product,
// next scores) is bound by the latency of the weights: with a thread per row
// (four warps) the tensor cores idled half the time.
// 256 rows a block because a K/V tile then feeds 256 flop a byte from L2.
//
// Measured: 16384 x 16384 rows of 64/8 heads of 128, causal, 3.9 ms (1.1 PFLOP/s,
// 0.68 of the measured product).  At D = 128 two row tiles take all of tensor memory
// (at 64 three quarters, and a third buffer for scores is not there yet), so a
// tile's next scores wait for its last weights: a turn is about 3250 cycles
// (weights 1270, maximum and meeting 480, products and waits the rest) against
// 2048 of mma.
#pragma once
#include "attention.cuh"
#include "tcgen05.cuh"

namespace lmc {

constexpr int kTileM = 128, kTileN = 128, kBlockRows = 256;
constexpr int kStages = 2;  // of a key tile's K and the V of the tile before it
constexpr int kTcThreads = 640, kMmaWarp = 16, kLoadWarp = 17;
constexpr int kTileThreads = 256;  // of one row tile: two per row
struct Yes { static constexpr bool value = true; };
struct No { static constexpr bool value = false; };
constexpr float kLazy = 8.f;  // log2 of how far P may pass 1 before O is rescaled
// log2 of a factor on the weights (the sum has it too, so only the row's log takes
// it off).  Below 2^-14 float16 rounds in steps of 2^-24, and 2^-25 of the maximum
// was lost: 100k keys of that size are 0.3% of a row.  2^7 times larger, weights of
// up to 2^8 stay below its 65504 and what is lost is 2^-32.
template <typename T>
constexpr float kRaised = __is_same(T, __half) ? 7.f : 0.f;

// Dense keys: positions and documents of a key tile.
struct TileStats {
  int pos_min, pos_max, doc_min, doc_max;
};

struct TcArgs {
  const void *q;
  void *out;      // [tokens, H, D] in the rows' type, when slices == 0
  float *lse;     // [tokens, H] or null
  float *part_o;  // [slices, tokens * H, D] normalised, when slices > 0
  float *part_lse;  // [slices, tokens * H], log2
  const float *slopes;
  long long q_batch, q_token, q_head;
  int tokens, q_len, heads, group;
  int k_tiles, tiles_per_slice, slices;
  // x = s scale_log2, or cap_out tanh(u) with u = s cap_u and cap_in = 2 cap_u log2 e;
  // for |s| up to cap_small x = s P(u^2)
  float scale_log2, cap_u, cap_in, cap_out, cap_small;
  float2 cap_poly[5];
  // dense keys (prepared arrays, padded to whole tiles)
  PositionArgs pos;
  const int *k_pos32, *k_doc32;
  const float *k_rel;  // position minus the tile's smallest, for the distance bias
  const int *k_run;    // the tile's positions go up by one
  const TileStats *stats;
  // paged prefix
  const int *pages, *own_lens;
  int block_size, num_blocks;
  long long prefix_len;
  DeviceStatus *status;
};

template <int D>
struct TcSmem {
  static constexpr int kTile = kTileN * D * 2;
  static constexpr int kQ = 0;  // two row tiles; at the end their results pass through
  static constexpr int kQTile = kTileM * 256;
  static constexpr int kKV = 2 * kQTile;             // kStages times K, V
  static constexpr int kBars = kKV + kStages * 2 * kTile;
  static constexpr int kXch = kBars + 256;    // two floats per row
  static constexpr int kQAt = kXch + 2048;    // where each row's query lies
  static constexpr int kRowAt = kQAt + 2048;  // and its result, -1 behind the last row
  static constexpr int kBytes = kRowAt + 1024 + 1024;  // + alignment to the swizzle's 1 KB
};

// True in all of `kThreads` threads that meet at a barrier if it is in any of them.
template <int kThreads>
__device__ __forceinline__ bool any_of(int barrier, bool v) {
  uint32_t r;
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\n"
      "barrier.cta.red.or.pred q, %2, %3, p;\nselp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(v ? 1u : 0u), "r"(barrier), "n"(kThreads)
      : "memory");
  return r != 0;
}
// The threads of a row tile, and the two warps that share 32 of its rows.
__device__ __forceinline__ bool tile_any(int tile, bool v) {
  return any_of<kTileThreads>(1 + tile, v);
}
__device__ __forceinline__ bool pair_any(int tile, int rows, bool v) {
  return any_of<64>(3 + tile * 4 + rows, v);
}

struct RowRef {
  int token, head;
  bool valid;
};

// (tokens * heads < 2^31, so a row index fits 32 bits)
__device__ __forceinline__ RowRef row_ref(const TcArgs &a, int kv_head, unsigned rho) {
  RowRef r;
  const unsigned t = rho / static_cast<unsigned>(a.group);
  r.valid = t < static_cast<unsigned>(a.tokens);
  r.token = r.valid ? static_cast<int>(t) : 0;
  r.head = kv_head * a.group + static_cast<int>(rho - t * a.group);
  return r;
}

constexpr int kSeesNothing = -2147483647 - 1;

// What a dense row may see: key positions below `limit` in document `doc`.
struct RowMask {
  int limit, doc, pos;
};

__device__ __forceinline__ int clamp_pos(long long p) {
  return static_cast<int>(min(max(p, -2147483646ll), 2147483645ll));
}

// What a row's mask is made of, as it is loaded: several loads can be under way
// before the first is used.
struct RawMask {
  long long at;
  int prefix, doc;
};

__device__ __forceinline__ RawMask load_mask(const PositionArgs &p, int token) {
  RawMask r;
  r.at = position_at(p.q_pos, p.long_q_pos, token);
  r.prefix = p.q_prefix ? p.q_prefix[token] : 0;
  r.doc = p.q_doc ? p.q_doc[token] : 0;
  return r;
}

__device__ __forceinline__ RowMask row_mask(const PositionArgs &p, const RawMask &r) {
  RowMask m;
  m.pos = clamp_pos(r.at);
  m.limit = p.causal ? m.pos + 1 : 2147483647;
  if (p.q_prefix) m.limit = max(m.limit, r.prefix);
  m.doc = r.doc;
  if (m.doc < 0) m.limit = kSeesNothing;  // a padding row
  return m;
}

// Which of 64 keys each row of the warp sees, as bits: lane i holds positions and
// documents of keys i and 32 + i.  Rows of one document (mostly all 32) share
// the keys below their least limit and above their greatest; only keys between
// are compared row by row.
__device__ __forceinline__ void visible_keys(const RowMask &row, int kp0, int kp1, int kd0, int kd1,
                                             bool docs, uint32_t &vis0, uint32_t &vis1) {
  constexpr uint32_t kAll = 0xffffffffu;
  vis0 = vis1 = 0;
  uint32_t todo = __ballot_sync(kAll, row.limit != kSeesNothing);
  while (todo) {
    const int doc = __shfl_sync(kAll, row.doc, __ffs(todo) - 1);
    const bool mine = row.limit != kSeesNothing && row.doc == doc;
    todo &= ~__ballot_sync(kAll, mine);
    const int lo = __reduce_min_sync(kAll, mine ? row.limit : 2147483647);
    const int hi = __reduce_max_sync(kAll, mine ? row.limit : kSeesNothing);
    const bool in0 = !docs || kd0 == doc, in1 = !docs || kd1 == doc;
    uint32_t v0 = __ballot_sync(kAll, in0 && kp0 < lo), v1 = __ballot_sync(kAll, in1 && kp1 < lo);
    uint32_t s0 = __ballot_sync(kAll, in0 && kp0 >= lo && kp0 < hi);
    uint32_t s1 = __ballot_sync(kAll, in1 && kp1 >= lo && kp1 < hi);
    while (s0) {
      const int b = __ffs(s0) - 1;
      s0 &= s0 - 1;
      v0 |= static_cast<uint32_t>(__shfl_sync(kAll, kp0, b) < row.limit) << b;
    }
    while (s1) {
      const int b = __ffs(s1) - 1;
      s1 &= s1 - 1;
      v1 |= static_cast<uint32_t>(__shfl_sync(kAll, kp1, b) < row.limit) << b;
    }
    if (mine) vis0 = v0, vis1 = v1;
  }
}

// A row whose tensor-core result holds an infinity or NaN is computed again by
// the definition, by one warp: a masked key's weight is 0, and 0 times an
// infinity in its value is not, so only keys that the row sees may take part.
template <typename T, int D>
__device__ __forceinline__ void strict_position_row(const PositionArgs &a, int token, int h) {
  const RowMask m = row_mask(a, load_mask(a, token));
  const int kv = h / (a.heads / a.kv_heads);
  WarpRow<T, D> row;
  row.start(static_cast<const T *>(a.q) + token * a.q_token + h * a.q_head);
  const float slope = a.slopes ? a.slopes[h] : 0.f;
#pragma unroll 1
  for (int j0 = 0; j0 < a.k_tokens && !row.lost(); j0 += 32) {
    const int j = min(j0 + static_cast<int>(threadIdx.x & 31), a.k_tokens - 1);
    const int kp = a.k_pos ? clamp_pos(position_at(a.k_pos, a.long_k_pos, j)) : j;
    const bool sees = j0 + static_cast<int>(threadIdx.x & 31) < a.k_tokens && kp < m.limit &&
                      (!a.k_doc || a.k_doc[j] == m.doc);
    row.add(sees, static_cast<const T *>(a.k) + j * a.k_token + kv * a.k_head,
            static_cast<const T *>(a.v) + j * a.v_token + kv * a.v_head, a.scale, a.softcap,
            slope * fabsf(static_cast<float>(static_cast<long long>(m.pos) - kp)));
  }
  const long long r = static_cast<long long>(token) * a.heads + h;
  row.finish(static_cast<T *>(a.out) + r * D, a.lse ? a.lse + r : nullptr);
}

// The same as a call of its own, for the join (inlined, its registers and code cost a
// join of 27 parts 0.3 of 16.7 us).
template <typename T, int D>
__device__ __noinline__ void strict_position_row_again(const PositionArgs &a, int token, int h) {
  strict_position_row<T, D>(a, token, h);
}

// The key tiles of a block, in order; every role walks them alike.
template <bool kDense>
struct TileScan {
  const TcArgs &a;
  int end, base;
  uint32_t live, full;
  int lim_min, lim_max, doc_min, doc_max;

  __device__ TileScan(const TcArgs &args, int begin, int stop, const int *group)
      : a(args), end(stop), base(begin - 32), live(0), full(0) {
    if (kDense) lim_min = group[0], lim_max = group[1], doc_min = group[2], doc_max = group[3];
    else base = begin - 1;
  }

  // How many tiles there are; the scan is used up.
  __device__ __forceinline__ int count() {
    if constexpr (!kDense) return max(0, end - base - 1);
    int n = 0, tile;
    bool whole;
    while (next(tile, whole)) {
      n += 1 + __popc(live);
      live = 0;
    }
    return n;
  }

  __device__ __forceinline__ bool next(int &tile, bool &whole) {
    if constexpr (!kDense) {
      tile = ++base;
      whole = true;
      return base < end;
    } else {
      return next_dense(tile, whole);
    }
  }

  __device__ __forceinline__ bool next_dense(int &tile, bool &whole) {
    while (live == 0) {
      base += 32;
      if (base >= end) return false;
      const int t = base + (threadIdx.x & 31);
      bool some = false, all = false;
      if (t < end) {
        const TileStats s = a.stats[t];
        some = s.pos_min < lim_max && s.doc_min <= doc_max && s.doc_max >= doc_min;
        all = s.pos_max < lim_min && s.doc_min == s.doc_max && doc_min == doc_max &&
              s.doc_min == doc_min;
      }
      live = __ballot_sync(0xffffffffu, some);
      full = __ballot_sync(0xffffffffu, some && all);
    }
    const int bit = __ffs(live) - 1;
    live &= live - 1;
    tile = base + bit;
    whole = (full >> bit) & 1;
    return true;
  }
};

template <typename T, int D, bool kDense, bool kDocs, bool kCap, bool kBias>
__global__ void __launch_bounds__(kTcThreads, 1)
    tc_attention_kernel(const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map,
                        const __grid_constant__ TcArgs a) {
  using L = TcSmem<D>;
  constexpr int kHalves = D / 64;            // 128-byte column blocks of a row
  constexpr int kHalfBytes = kTileN * 128;   // of one tile
  constexpr bool kBf16 = __is_same(T, __nv_bfloat16);
  // of 8 pairs of weights, how many the FMA pipe computes: ex2 and the mma are
  // equally long at D = 128, ex2 is the longer at D = 64, and a cap or a bias
  // keeps the FMA pipe busy
  constexpr int kFmaOf8 = kCap || kBias ? 0 : D == 128 ? 2 : 3;
  extern __shared__ uint8_t raw_smem[];
  uint8_t *smem = reinterpret_cast<uint8_t *>(
      (reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kBars);
  uint64_t *kv_full = bars, *kv_empty = bars + kStages, *s_full = bars + 2 * kStages,
           *p_full = s_full + 2, *o_done = p_full + 2, *p_half = o_done + 2, *q_full = p_half + 2,
           *drain = q_full + 1;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(drain + 1);
  int *stopped = reinterpret_cast<int *>(tmem_slot + 1);
  int *seen = stopped + 1;  // limits and documents of the block's rows

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform, for the compiler too
  const int kv_heads = a.heads / a.group;
  // the last rows see the most keys: they start first
  const int per_row_group = kv_heads * max(1, a.slices);
  const long long rows = static_cast<long long>(a.tokens) * a.group;
  const int n_groups = static_cast<int>((rows + kBlockRows - 1) / kBlockRows);
  const int row_group = n_groups - 1 - static_cast<int>(blockIdx.x / per_row_group);
  const int rest = static_cast<int>(blockIdx.x % per_row_group);
  const int kv_head = rest % kv_heads, slice = rest / kv_heads;
  const unsigned rho0 = static_cast<unsigned>(row_group) * kBlockRows;
  const int tiles = rho0 + kTileM < rows ? 2 : 1;
  const int t_begin = slice * a.tiles_per_slice;
  const int t_end = min(a.k_tiles, t_begin + a.tiles_per_slice);

  if (a.slices) let_next_start();
  if (warp == kMmaWarp) tmem_alloc(tmem_slot, 512);
  if (warp == kLoadWarp && lane == 0) {
    prefetch_map(&k_map), prefetch_map(&v_map);
    for (int i = 0; i < kStages; ++i) mbar_init(&kv_full[i], 1), mbar_init(&kv_empty[i], 1);
    for (int i = 0; i < 2; ++i)
      mbar_init(&s_full[i], 1), mbar_init(&p_half[i], kTileThreads),
          mbar_init(&p_full[i], kTileThreads), mbar_init(&o_done[i], 1);
    mbar_init(q_full, kTileThreads * tiles);
    mbar_init(drain, 1);
    *stopped = 0;
    seen[0] = 2147483647, seen[1] = -2147483647 - 1;
    seen[2] = 2147483647, seen[3] = -2147483647 - 1;
    fence_mbar_init();
  }
  // Rows, while that happens: Q on its way to shared memory (128-byte swizzled
  // rows), then the masks.
  RowRef ref = {0, 0, false};
  RowMask mask = {0, 0, 0};
  const int x = warp >> 3, half = (warp >> 2) & 1;  // row tile, and which 64 keys
  const int row_in_tile = tid & 127;
  int lim_lo = 2147483647, lim_hi = kSeesNothing, doc_lo = lim_lo, doc_hi = lim_hi;
  long long *q_at = reinterpret_cast<long long *>(smem + L::kQAt) + x * kTileM;
  int *row_at = reinterpret_cast<int *>(smem + L::kRowAt) + x * kTileM;
  if (warp < kMmaWarp && x < tiles) {
    ref = row_ref(a, kv_head, rho0 + x * kTileM + row_in_tile);
    RawMask raw = {0, 0, 0};
    if (kDense && ref.valid) raw = load_mask(a.pos, ref.token);
    if (half == 0) {
      const int b = ref.token / a.q_len;
      q_at[row_in_tile] = b * a.q_batch + (ref.token - b * a.q_len) * a.q_token +
                          (ref.valid ? ref.head : 0) * a.q_head;
      row_at[row_in_tile] = ref.valid ? ref.token * a.heads + ref.head : -1;
    }
    tile_any(x, false);
    constexpr int kVecs = D / 8, kAtOnce = kTileThreads / kVecs;
    const int c = tid % kVecs, r0 = (tid & (kTileThreads - 1)) / kVecs;
    const uint32_t dst = smem_u32(smem + L::kQ + x * L::kQTile) + (c >> 3) * kHalfBytes;
    const T *q = static_cast<const T *>(a.q) + c * 8;
#pragma unroll
    for (int i = 0; i < kTileM / kAtOnce; ++i) {
      const int r = r0 + i * kAtOnce;
      cp_async16(dst + r * 128 + (((c & 7) ^ (r & 7)) << 4), q + q_at[r], row_at[r] >= 0);
    }
    if (kDense) {
      mask.limit = lim_hi;
      if (ref.valid) mask = row_mask(a.pos, raw);
      const bool in_doc = ref.valid && mask.doc >= 0;
      lim_lo = __reduce_min_sync(0xffffffffu, ref.valid ? mask.limit : lim_lo);
      lim_hi = __reduce_max_sync(0xffffffffu, in_doc ? mask.limit : lim_hi);
      doc_lo = __reduce_min_sync(0xffffffffu, in_doc ? mask.doc : doc_lo);
      doc_hi = __reduce_max_sync(0xffffffffu, in_doc ? mask.doc : doc_hi);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // the whole of tensor memory starts at column 0: a constant address
  constexpr uint32_t tmem = 0;
  if (kDense) {
    wait_for_previous();  // the key tiles' ranges
    if (warp < kMmaWarp && x < tiles && lane == 0 && half == 0) {
      atomicMin(&seen[0], lim_lo), atomicMax(&seen[1], lim_hi);
      atomicMin(&seen[2], doc_lo), atomicMax(&seen[3], doc_hi);
    }
    __syncthreads();  // `seen` is whole
  }
  TileScan<kDense> scan(a, t_begin, t_end, seen);

  // (each role sets its registers in its own branch: the compiler then allots
  // them per branch)
  if (warp == kLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    // ------------------------------------------------------------- loader
    int tile = 0, before = -1, it = 0;
    bool whole, ok = true, more = true;
    const int boxes = kDense ? 1 : max(1, kTileN / a.block_size);
    auto fetch = [&](uint8_t *dst, const CUtensorMap *map, int of, uint64_t *bar) {
      if (kDense) {
        if (lane < kHalves)
          tma_load_3d(dst + lane * kHalfBytes, map, lane * 64, kv_head, of * kTileN, bar);
      } else if (lane < boxes) {
        // a page, or 128 slots of a larger one; an id outside the cache reads zeros
        const int box_rows = min(kTileN, a.block_size);
        const int j = of * kTileN + lane * box_rows;
        const int col = j / a.block_size;
        int page = a.pages[col];
        if (page < 0 || page >= a.num_blocks) page = a.num_blocks;
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
          tma_load_4d(dst + h * kHalfBytes + lane * box_rows * 128, map, h * 64, kv_head,
                      j - col * a.block_size, page, bar);
      }
    };
    while (more) {
      more = scan.next(tile, whole);
      if (!more && before < 0) break;  // no tiles
      const int st = it % kStages;
      if (it >= kStages) ok = wait_or_stop(&kv_empty[st], (it / kStages - 1) & 1, stopped);
      if (!ok) break;
      uint8_t *dst = smem + L::kKV + st * 2 * L::kTile;
      if (lane == 0)
        mbar_arrive_expect_tx(&kv_full[st], (more ? L::kTile : 0) + (before >= 0 ? L::kTile : 0));
      __syncwarp();
      if (more) fetch(dst, &k_map, tile, &kv_full[st]);
      if (before >= 0) fetch(dst + L::kTile, &v_map, before, &kv_full[st]);
      before = tile;
      ++it;
    }
    // loads in flight land before the block's memory is given back
    for (int i = max(0, it - kStages); i < it; ++i)
      mbar_wait_bounded(&kv_full[i % kStages], (i / kStages) & 1, 2000000000ull);
  } else if (warp == kMmaWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
    // ------------------------------------------------------------- mma
    constexpr uint32_t kQK = mma_desc(kBf16, false, kTileM, kTileN);
    constexpr uint32_t kPV = mma_desc(kBf16, true, kTileM, D);
    const uint32_t q_addr = smem_u32(smem + L::kQ), kv_addr = smem_u32(smem + L::kKV);
    auto score = [&](int t, int st) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        const uint32_t off = (k >> 2) * kHalfBytes + (k & 3) * 32;
        mma_ss(tmem + t * kTileN, smem_desc(q_addr + t * L::kQTile + off, 16, 1024),
               smem_desc(kv_addr + st * 2 * L::kTile + off, 16, 1024), kQK, k > 0);
      }
      mma_commit(&s_full[t]);
    };
    // keys 0-31 and 64-95 of a tile (part 0), or the others (part 1)
    auto weigh = [&](int t, int st, int part, bool accumulate) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = (i >> 1) * 4 + part * 2 + (i & 1);
        mma_ts(tmem + 2 * kTileN + t * D, tmem + t * kTileN + k * 8,
               smem_desc(kv_addr + (st * 2 + 1) * L::kTile + k * 2048, kHalfBytes, 1024), kPV,
               accumulate || i > 0);
      }
    };
    // One thread waits and issues: a vote per wait would cost as much as an mma.
    const int n = scan.count();
    if (elect_one()) {
      bool ok = lane_wait(q_full, 0, stopped);
      if (n > 0) {
        ok = ok && lane_wait(&kv_full[0], 0, stopped);
        tc_fence_after();
        if (ok) {
          score(0, 0);
          if (tiles > 1) score(1, 0);
          mma_commit(&kv_empty[0]);
        }
      }
      int st = 1, phase = 0;  // of V_j and K_{j + 1}
#pragma unroll 1
      for (int j = 0; ok && j < n; ++j) {
        const bool more = j + 1 < n;
        ok = lane_wait(&kv_full[st], phase, stopped);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (t >= tiles) break;
          ok = ok && lane_wait(&p_half[t], j & 1, stopped);
          if (!ok) break;
          tc_fence_after();
          weigh(t, st, 0, j > 0);
          ok = lane_wait(&p_full[t], j & 1, stopped);
          if (!ok) break;
          tc_fence_after();
          weigh(t, st, 1, true);
          if (more) score(t, st);
          if (t == tiles - 1) mma_commit(&kv_empty[st]);
          if (!more) mma_commit(&o_done[t]);
        }
        if (++st == kStages) st = 0, phase ^= 1;
      }
      if (!ok) {  // only after a wait that ran out: let the mma in flight end
        mma_commit(drain);
        mbar_wait_bounded(drain, 0, 2000000000ull);
      }
    }
    __syncwarp();
  } else if (warp > kLoadWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 112;");
    if (x < tiles) {
      // ------------------------------------------------------------- softmax
      const uint32_t lane_base = static_cast<uint32_t>(warp & 3) << 21;
      constexpr int kKeys = kTileN / 2;  // of this thread
      const uint32_t s_addr = tmem + lane_base + x * kTileN;
      const uint32_t o_addr = tmem + lane_base + 2 * kTileN + x * D + half * (D / 2);
      float *xch = reinterpret_cast<float *>(smem + L::kXch) + x * 2 * kTileM;
      float *mine = xch + half * kTileM + row_in_tile;
      const float *other = xch + (1 - half) * kTileM + row_in_tile;
      float m = -INFINITY, l = 0.f;
      const float slope = kBias && ref.valid ? a.slopes[ref.head] * kLog2e : 0.f;
      long long q_place = 0;  // position behind the prefix, for the distance bias
      if (!kDense && kBias && ref.valid) {
        const int b = ref.token / a.q_len;
        q_place = a.prefix_len + max(0, a.own_lens[b]) - a.q_len + (ref.token - b * a.q_len);
      }
      cp_async_commit();
      cp_async_wait<0>();
      fence_proxy_async_smem();
      mbar_arrive(q_full);
      int tile, j = 0;
      bool whole, ok = true;
      while (scan.next(tile, whole)) {
        const int key0 = tile * kTileN + half * kKeys;
        // masks while the scores are computed
        uint32_t vis0 = 0xffffffffu, vis1 = 0xffffffffu;
        if (kDense && !whole) {
          const int kp0 = a.k_pos32[key0 + lane], kp1 = a.k_pos32[key0 + 32 + lane];
          const int kd0 = kDocs ? a.k_doc32[key0 + lane] : 0;
          const int kd1 = kDocs ? a.k_doc32[key0 + 32 + lane] : 0;
          visible_keys(mask, kp0, kp1, kd0, kd1, kDocs, vis0, vis1);
        }
        uint32_t bad = 0;  // pages of this tile that lie outside the cache
        bool some_page = true;
        if (!kDense) {
          const int boxes = max(1, kTileN / a.block_size);
          bool out_of_cache = false;
          if (lane < boxes) {
            const int page =
                a.pages[(tile * kTileN + lane * min(kTileN, a.block_size)) / a.block_size];
            out_of_cache = page < 0 || page >= a.num_blocks;
            if (out_of_cache) report_status(a.status, kStatusBadSlot, -1, tile, page);
          }
          bad = __ballot_sync(0xffffffffu, out_of_cache);
          some_page = __popc(bad) < boxes;
        }
        ok = wait_or_stop(&s_full[x], j & 1, stopped);
        tc_fence_after();
        // Between documents most warps' rows see none of their half of a tile that
        // another row of the block sees: they hand in zeros only (8k rows in
        // 24 documents 197 -> 166 us).  Under positions alone that is a warp or
        // two at the diagonal, and the branch around everything costs 8%.
        const bool none = kDocs && !whole && !__any_sync(0xffffffffu, (vis0 | vis1) != 0);
        const float c = kCap || kBias ? 1.f : a.scale_log2;
        float s[kKeys], top = -INFINITY;
        float lift = 0.f;  // what all scores of this row and tile still lack
        if (!none) {
#pragma unroll
          for (int part = 0; part < kKeys / 32; ++part)
            tmem_ld32(s_addr + half * kKeys + part * 32,
                      reinterpret_cast<uint32_t(&)[32]>(s[part * 32]));
          tmem_wait_ld();
          // x = s c in log2 units, unless it is only scaled (then c goes into exp2)
          if (kCap) {
            // tanh by an odd polynomial while every score of the warp's rows is small
            // against the cap, as they mostly are: four FMA slots a score instead of
            // the exponential and reciprocal of tanh(u) = 1 - 2 / (1 + e^2u)
            float big = 0.f;
#pragma unroll
            for (int i = 0; i < kKeys; i += 2)
              big = fmaxf(fmaxf(big, fabsf(s[i])), fabsf(s[i + 1]));
            if (__all_sync(0xffffffffu, big <= a.cap_small)) {
              f32x2 k[5];
              const f32x2 cap_u = pack2(a.cap_u, a.cap_u);
#pragma unroll
              for (int i = 0; i < 5; ++i) k[i] = pack2(a.cap_poly[i].x, a.cap_poly[i].y);
#pragma unroll
              for (int i = 0; i < kKeys; i += 2) {
                const f32x2 v = pack2(s[i], s[i + 1]), u = mul2(v, cap_u), w = mul2(u, u);
                unpack2(mul2(v, fma2(fma2(fma2(fma2(k[4], w, k[3]), w, k[2]), w, k[1]), w, k[0])),
                        s[i], s[i + 1]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < kKeys; ++i)
                s[i] = fmaf(rcp(1.f + ex2(s[i] * a.cap_in)), -2.f * a.cap_out, a.cap_out);
            }
          } else if (kBias) {
#pragma unroll
            for (int i = 0; i < kKeys; ++i) s[i] *= a.scale_log2;
          }
          if (kBias) {
            // -slope |p - p_j|; for keys one apart at or before the row, slope j plus
            // a constant (what else is in the tile is masked)
            bool run = true;
            float at;  // the row's place counted from this thread's first key
            if (kDense) {
              run = a.k_run[tile] != 0;
              at = static_cast<float>(static_cast<long long>(mask.pos) - a.stats[tile].pos_min) -
                   (run ? static_cast<float>(half * kKeys) : 0.f);
            } else {
              at = static_cast<float>(q_place - key0);
            }
            const bool before =
                kDense ? mask.limit <= mask.pos + 1 || at >= kKeys : at >= kKeys - 1;
            if (run && __all_sync(0xffffffffu, before || !ref.valid)) {
              lift = -slope * at;
              const f32x2 sl = pack2(slope, slope), two = pack2(2.f, 2.f);
              f32x2 n = pack2(0.f, 1.f);
#pragma unroll
              for (int i = 0; i < kKeys; i += 2) {
                unpack2(fma2(sl, n, pack2(s[i], s[i + 1])), s[i], s[i + 1]);
                n = add2(n, two);
              }
            } else if (run) {
#pragma unroll
              for (int i = 0; i < kKeys; ++i)
                s[i] = fmaf(-slope, fabsf(at - static_cast<float>(i)), s[i]);
            } else {
              const float4 *rel = reinterpret_cast<const float4 *>(a.k_rel + key0);
#pragma unroll
              for (int i = 0; i < kKeys / 4; ++i) {
                const float4 p = rel[i];
                s[4 * i] = fmaf(-slope, fabsf(at - p.x), s[4 * i]);
                s[4 * i + 1] = fmaf(-slope, fabsf(at - p.y), s[4 * i + 1]);
                s[4 * i + 2] = fmaf(-slope, fabsf(at - p.z), s[4 * i + 2]);
                s[4 * i + 3] = fmaf(-slope, fabsf(at - p.w), s[4 * i + 3]);
              }
            }
          }
          if (kDense && !whole) {
            if (__any_sync(0xffffffffu, vis0 != 0xffffffffu)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((vis0 >> i) & 1)) s[i] = -INFINITY;
            }
            if (__any_sync(0xffffffffu, vis1 != 0xffffffffu)) {
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (!((vis1 >> i) & 1)) s[32 + i] = -INFINITY;
            }
          }
          if (!kDense && bad) {
            const int rows_of = min(kTileN, a.block_size);
#pragma unroll
            for (int i = 0; i < kKeys; ++i)
              if ((bad >> ((half * kKeys + i) / rows_of)) & 1) s[i] = -INFINITY;
          }
          float t0 = s[0], t1 = s[1], t2 = s[2], t3 = s[3];
#pragma unroll
          for (int i = 4; i + 7 < kKeys; i += 8) {
            t0 = fmaxf(fmaxf(t0, s[i]), s[i + 1]);
            t1 = fmaxf(fmaxf(t1, s[i + 2]), s[i + 3]);
            t2 = fmaxf(fmaxf(t2, s[i + 4]), s[i + 5]);
            t3 = fmaxf(fmaxf(t3, s[i + 6]), s[i + 7]);
          }
          t0 = fmaxf(fmaxf(t0, s[kKeys - 4]), s[kKeys - 3]);
          t1 = fmaxf(fmaxf(t1, s[kKeys - 2]), s[kKeys - 1]);
          top = fmaf(fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)), c, lift);
        }
        // O is rescaled when a row's maximum has grown (also at its first finite
        // score), by both of its threads alike.  The meeting also keeps a warp from
        // writing weights over scores that the other has not read.
        if (pair_any(x, warp & 3, top > m + kLazy || !ok)) {
          *mine = top;
          if (pair_any(x, warp & 3, !ok)) {
            ok = false;
            break;
          }
          const float both = fmaxf(top, *other);
          const bool grow = both > m + kLazy;
          const float to = grow ? both : m;
          const float keep = grow ? ex2(m - to) : 1.f;
          m = to;
          l *= keep;
          if (j > 0) {  // the score barrier also covers the last product into O
#pragma unroll 1
            for (int k = 0; k < D / 64; ++k) {
              uint32_t o[32];
              tmem_ld32(o_addr + k * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * keep);
              tmem_st32(o_addr + k * 32, o);
            }
          }
        }
        // Without a finite score yet: zero weights for a row that sees no key of its
        // half of this tile; one that does has only scores of -inf there, and NaN
        // weights (-inf less -inf) lead it to the definition.
        const bool sees = kDense ? whole || (vis0 | vis1) != 0 : some_page;
        const float off = (m == -INFINITY && !sees ? 0.f : m) - lift - kRaised<T>;
        const f32x2 c2 = pack2(c, c), off2 = pack2(-off, -off);
        f32x2 l0 = pack2(0.f, 0.f), l1 = l0;
        // the weights of 32 keys, some of them by the polynomial; the product may
        // start with the first 32
        auto weights = [&](int part, auto some_fma) {
          uint32_t p[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int k = part * 32 + 2 * i;
            const f32x2 v = fma2(pack2(s[k], s[k + 1]), c2, off2);
            float e, f;
            if (decltype(some_fma)::value && i % 8 >= 8 - kFmaOf8) {
              exp2_fma(v, e, f);
            } else {
              unpack2(v, e, f);
              e = ex2(e), f = ex2(f);
            }
            if (i & 1)
              l1 = add2(l1, pack2(e, f));
            else
              l0 = add2(l0, pack2(e, f));
            p[i] = pair_from_float<T>(e, f);
          }
          tmem_st16(s_addr + half * (kKeys / 2) + part * 16, p);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(part == 0 ? &p_half[x] : &p_full[x]);
        };
        if (none) {
          const uint32_t zeros[16] = {};
          tmem_st16(s_addr + half * (kKeys / 2), zeros);
          tmem_st16(s_addr + half * (kKeys / 2) + 16, zeros);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&p_half[x]);
          mbar_arrive(&p_full[x]);
        } else if (whole) {
          weights(0, Yes{}), weights(1, Yes{});
        } else {
          weights(0, No{}), weights(1, No{});
        }
        float u0, u1;
        unpack2(add2(l0, l1), u0, u1);
        l += u0 + u1;
        ++j;
      }
      // ------------------------------------------------------------- result
      if (ok && j > 0) ok = wait_or_stop(&o_done[x], 0, stopped);
      tc_fence_after();
      if (ok || j == 0) *mine = l;  // (after a break nobody reads it)
      ok = !tile_any(x, !ok);
      if (ok) l += *other;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : NAN);
      const long long row = row_at[row_in_tile];
      bool finite = true;
      // 64 columns at a time (32 of each half) through the tile's share of Q's
      // memory, so that stores to the rows run along them
      uint8_t *stage = smem + L::kQ + x * L::kQTile;
#pragma unroll 1
      for (int k = 0; k < D / 64; ++k) {
        float o[32];
        if (ok && j > 0) {
          tmem_ld32(o_addr + k * 32, reinterpret_cast<uint32_t(&)[32]>(o));
          tmem_wait_ld();
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          o[i] = ok ? (j > 0 ? o[i] * inv : 0.f) : NAN;
          finite = finite && fabsf(o[i]) <= 3.4028235e38f;
        }
        const int swz = row_in_tile & 7;
        if (a.slices == 0) {
          uint8_t *w = stage + row_in_tile * 128;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            int4 v;
            v.x = pair_from_float<T>(o[8 * i], o[8 * i + 1]);
            v.y = pair_from_float<T>(o[8 * i + 2], o[8 * i + 3]);
            v.z = pair_from_float<T>(o[8 * i + 4], o[8 * i + 5]);
            v.w = pair_from_float<T>(o[8 * i + 6], o[8 * i + 7]);
            *reinterpret_cast<int4 *>(w + (((half * 4 + i) ^ swz) << 4)) = v;
          }
        } else {
          uint8_t *w = stage + half * kHalfBytes + row_in_tile * 128;
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4 *>(w + ((i ^ swz) << 4)) =
                make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
        }
        tile_any(x, false);
        const int in_tile = tid & (kTileThreads - 1);
        if (a.slices == 0) {
#pragma unroll
          for (int i = 0; i < kTileM * 8 / kTileThreads; ++i) {
            const int r = (in_tile >> 3) + i * (kTileThreads / 8), v = in_tile & 7;
            if (row_at[r] < 0) continue;
            st_v4(static_cast<T *>(a.out) + static_cast<long long>(row_at[r]) * D +
                      (v >> 2) * (D / 2) + k * 32 + (v & 3) * 8,
                  *reinterpret_cast<const int4 *>(stage + r * 128 + ((v ^ (r & 7)) << 4)));
          }
        } else {
          float *part = a.part_o + static_cast<long long>(slice) * a.tokens * a.heads * D;
#pragma unroll
          for (int i = 0; i < kTileM * 16 / kTileThreads; ++i) {
            const int r = (in_tile >> 4) + i * (kTileThreads / 16), v = in_tile & 15;
            if (row_at[r] < 0) continue;
            st_v4(part + static_cast<long long>(row_at[r]) * D + (v >> 3) * (D / 2) + k * 32 +
                      (v & 7) * 4,
                  *reinterpret_cast<const int4 *>(stage + (v >> 3) * kHalfBytes + r * 128 +
                                                  (((v & 7) ^ (r & 7)) << 4)));
          }
        }
        if (k + 1 < D / 64) tile_any(x, false);
      }
      if (ref.valid && half == 0) {
        if (a.slices == 0) {
          if (a.lse) a.lse[row] = log2_of_sum(ok, m - kRaised<T>, l) * kLn2;
        } else {
          a.part_lse[static_cast<long long>(slice) * a.tokens * a.heads + row] =
              log2_of_sum(ok, m - kRaised<T>, l);
        }
      }
      if (!ok && row_in_tile == 0 && half == 0)
        report_status(a.status, kStatusMbarTimeout, kv_head, row_group, slice);
      if (kDense && a.slices == 0) {
        const bool wrong = ref.valid && !finite;
        if (tile_any(x, wrong)) {  // what was written above is written again below
          *mine = wrong ? 1.f : 0.f;
          tile_any(x, false);
          // (the two warps of 32 rows take every other one)
          uint32_t again = __ballot_sync(0xffffffffu, *mine + *other > 0.f) &
                           (half == 0 ? 0x55555555u : 0xaaaaaaaau);
          while (again) {
            const int src = __ffs(again) - 1;
            again &= again - 1;
            strict_position_row<T, D>(a.pos, __shfl_sync(0xffffffffu, ref.token, src),
                                      __shfl_sync(0xffffffffu, ref.head, src));
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kMmaWarp) tmem_free(tmem, 512);
}

}  // namespace lmc
