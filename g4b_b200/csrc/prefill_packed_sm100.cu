// Attention of packed rows -- prompts, chunks and single tokens of several slots behind one another,
// without padding -- over a paged KV cache, on the 5th-generation tensor cores: causal (or full),
// grouped query heads, optional per-query sliding window, head dims 256 and 128, f16 / bf16.
//
//   o[n, h] = sum_j p_j v[j, g] / sum_j p_j,   p_j = exp(scale q[n, h] . k[j, g]),   g = h / (H / G)
//
// over the keys j that row n (position pos of slot b) sees: j < time[b], j <= pos (causal), j > pos - W.
// A row that sees none is zero.  One pass over the keys with a running maximum and sum.
//
// The padded form of the same attention is prefill_sm100.cu; the tensor-core pipeline here is
// that kernel's (its comments say why it is built that way): a cluster of two CTAs shares every K / V
// tile through cta_group::2 MMAs, a producer warp feeds a ring of shared memory by TMA, one warp
// issues every MMA, eight warps turn scores into probabilities in tensor memory.  What differs:
//
// Rows.  A tile's 128 rows are (token, query head of one kv head) pairs: 128 / (H/G) tokens x H/G heads, one TMA
//   box of the packed q.  All heads of a group share the tile, so one token is one row per head
//   instead of a tile per head, and the ragged end of a causal block is 2 x 128 / (H/G) tokens wide.
// Items.  A work item is a block of tokens of one slot and one kv head.  How many there are is known
//   on the device only; a small launch before this one (plan_kernel) lists them.  With enough of them they
//   are dealt whole, those with most keys first.  Where a few long ones would keep some workers busy
//   long after the others (chunks behind long contexts, single tokens), every worker gets the same share of
//   the tiles instead: an item that lies across a boundary leaves its un-normalised parts in the
//   workspace, and a third launch joins them.
// Pages.  A box is one page's rows (up to what a CTA stages); groups of rows past the context, and
//   groups whose table entry is bad, are boxes outside the pool, which TMA fills with zeros.  Where the
//   context ends inside a group the producer zeroes the rest of V itself (it may hold anything, and
//   0 x NaN would poison the accumulator); K needs no such care, its scores are replaced.
//
// Output rows are turned through shared memory, so that they leave as TMA boxes or as 128-byte row pieces.
//
// Measured (8 / 2 heads, 16-row pages, bf16; 300 to 340 us by box and clock): prompts of 8192, 5000, 2500 and 701 rows at head
// dim 256, 0.405 TFLOP: 1.2 to 1.35 PFLOP/s, tensor pipe 75 % active; bound by the tensor pipe and the power it draws.  4 x
// 8192 rows with 64-row pages 741 us = 1484 TFLOP/s.  A window of 512 keys: 68 to 80 us for 0.052 TFLOP, bound by an item's end
// (6500 cycles for five tiles of 2450).  Head dim 128: 87 to 99 us for 0.067 TFLOP, bound by the softmax warps' latency (2070
// cycles a tile for 1024 of tensor work).  Three prompts of 62 rows in all: 12 us, of which the list 1.7, the first loads 3.
#include "common.cuh"
#include "sm100_ptx.cuh"

#include <cudaTypedefs.h>

namespace g4b {

namespace {

constexpr int kBM = 128;           // rows per CTA: (token, head) pairs
constexpr int kBN = 128;           // keys per S tile
constexpr int kThreads = 384;      // 2 softmax warpgroups; producer warps 8 (Q and K) and 10 (V), MMA warp 9, one idle
// Registers a thread: launched with 168, of which the softmax warps take from the others (2 x 128 x 200 + 128 x 104 =
// 384 x 168)
constexpr int kRegsSoftmax = 200, kRegsOther = 104;
constexpr int kStageBytes = 8 * 4096;         // output: 4 KB per softmax warp
constexpr int kXchgBytes = 2 * 2 * kBM * 4;   // row maxima: [tile parity][column half][row]

template <int kD> struct Geo {
  static constexpr int kSlabs = kD / 64;
  static constexpr int kQBytes = kBM * kD * 2;
  static constexpr int kChunkBytes = 64 * kD * 2;     // K: 64 keys x kD; V: 128 keys x kD / 2
  static constexpr int kStages = kD == 256 ? 4 : 8;
  static constexpr int kSmemBytes = kQBytes + kStages * kChunkBytes + kStageBytes + 512 + kXchgBytes;
};

constexpr uint32_t kColO = 0, kColS0 = 256, kColS1 = 384;

enum : int32_t {
  kErrStarts = 0x107,
  kErrQFull = 0x301, kErrKvEmpty = 0x302, kErrKvFull = 0x303, kErrSFull = 0x304, kErrPFull = 0x305, kErrPvDone = 0x306,
  kErrSmemAlign = 0x307, kErrPair = 0x308, kErrBadPage = 0x309, kErrQEmpty = 0x30a, kErrOFree = 0x30b, kErrTail = 0x30d,
};

// One block of tokens of one slot and kv head, or a piece of its keys.
struct __align__(16) PackedItem {
  int row0, n_tok;        // its rows of q and o (n_tok 0: an entry without work)
  int qpos0;              // position of the first
  int window;             // keys [0, window) exist
  int tile_lo, n_tiles;   // its 128-key tiles
  int slot;
  int g_part;             // kv head; upper 16 bits: 0, or 1 + the part of the workspace that this piece leaves
};

// The pieces of one split item.
struct JoinEntry {
  int row0, n_tok, g;
  int w_lo, w_hi;         // workers that hold a piece
  int part_lo;            // the first one's part; worker w > w_lo left part 2 w
  int pad[2];
};

constexpr int kMaxWorkers = 74;          // CTA pairs of a 148-SM GPU
constexpr int kMaxSplitItems = 2048;     // items (per kv head) up to which shares are dealt
constexpr int kPartRows = 2 * kBM;

// Workspace, in this order: counts, what each worker walks, split items, (l, m) of the parts, the parts,
// the list (the only piece whose size depends on the call).
struct PackedHeader {
  int n_entries;          // whole items, dealt in turns (walks absent)
  int shares;             // 1: worker w walks entries [begin[w], end[w])
  int n_joins;
  int pad[13];
  int begin[kMaxWorkers], end[kMaxWorkers];
  JoinEntry joins[kMaxWorkers];
  float part_lm[2 * kMaxWorkers][kPartRows][2];
};
constexpr int64_t kPartsAt = (sizeof(PackedHeader) + 255) / 256 * 256;
constexpr int64_t kPartBytes = (int64_t)kPartRows * 256 * 4;       // head dim 256; 128 uses half
constexpr int64_t kItemsAt = kPartsAt + 2 * kMaxWorkers * kPartBytes;

struct PackedParams {
  void* o;
  const int32_t* q_starts; const int32_t* times; const int32_t* block_tables;
  PackedHeader* header; float* parts; PackedItem* items;
  int64_t o_row, o_head, starts_s, time_s, bt_s0, bt_s1;
  int N, B, H, G;
  int group, tpt;                 // query heads per kv head; tokens per CTA (kBM / group)
  int group_mul;                  // r / group = r * group_mul >> 16 for r < kBM
  int max_items, workers;
  int may_split;                  // few enough blocks that shares can pay; then a join launch follows
  int page_shift, num_pages, max_pages;
  int k_rows, v_rows;             // rows of a K / V box
  int o_boxes;                    // the output goes out by TMA: 32 (token, head) rows are a box
  int sliding_window, causal, o_dtype;
  float scale_log2;
  int32_t* status;
};

__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther)); }
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax)); }
__device__ __forceinline__ void record(int32_t* status, int32_t code) { atomicCAS(status, 0, code); }
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_launch_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---------------------------------------------------------------------------------------
// the list of items
// ---------------------------------------------------------------------------------------
struct SlotRows {
  int first, n, time;     // rows of q, tokens of the slot
  int keys;               // of those tokens, the ones that its table reaches
  bool bad;
};
__device__ __forceinline__ SlotRows slot_rows(const PackedParams& p, int b) {
  SlotRows s{0, 0, 0, 0, false};
  if (b >= p.B) return s;
  const int lo = p.q_starts[b * p.starts_s], hi = p.q_starts[(int64_t)(b + 1) * p.starts_s];
  s.bad = lo < 0 || hi < lo || hi > p.N;
  if (s.bad) return s;
  s.first = lo;
  s.n = hi - lo;
  s.time = min(max(p.times[b * p.time_s], 0), 0x7fffff00);
  s.keys = (int)min((int64_t)s.time, (int64_t)p.max_pages << p.page_shift);
  return s;
}

// Which 128-key tiles a block of tokens at positions [qpos0, qpos0 + n_tok) needs.
__device__ __forceinline__ void tiles_of(const PackedParams& p, int qpos0, int n_tok, int window, int& lo, int& n) {
  const int key_hi = p.causal ? min(window, qpos0 + n_tok) : window;
  const int key_lo = p.sliding_window > 0 ? max(0, qpos0 - p.sliding_window + 1) : 0;
  lo = key_lo / kBN;
  n = key_hi > key_lo ? (key_hi + kBN - 1) / kBN - lo : 0;
}

__device__ __forceinline__ PackedItem block_of(const PackedParams& p, const SlotRows& s, int slot, int index, int block) {
  PackedItem it;
  const int tok0 = index * block;
  it.row0 = s.first + tok0;
  it.n_tok = min(block, s.n - tok0);
  it.qpos0 = s.time - s.n + tok0;
  it.window = s.keys;
  tiles_of(p, it.qpos0, it.n_tok, it.window, it.tile_lo, it.n_tiles);
  it.slot = slot;
  it.g_part = 0;
  return it;
}

// Over the block's 256 threads: the sum of the values before this thread's (kMax: the maximum up to and with
// this thread's), and of all.
template <bool kMax, typename V>
__device__ __forceinline__ V block_scan(V x, V* warp_sums, V& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V sum = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum = kMax ? max(sum, y) : sum + y;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  V before = kMax ? sum : 0;
  total = kMax ? sum : 0;
  for (int w = 0; w < 8; ++w) {
    const V y = warp_sums[w];
    if (w < warp) before = kMax ? max(before, y) : before + y;
    total = kMax ? max(total, y) : total + y;
  }
  return kMax ? before : before + sum - x;
}

constexpr int kEntryCost = 2;      // an item's start and epilogue, in tiles

// Every worker the same share of the cost (tiles + kEntryCost an item) along the line of all items, slot by
// slot and head by head; one block.  The entry of unit u (item, kv head) for worker w is u + w: along
// the line either the unit or the worker goes up by one.
__device__ __noinline__ void deal_shares(const PackedParams& p, int n_items) {
  __shared__ int slot_of[kMaxSplitItems], start_of[kMaxSplitItems];      // an item's slot, and the slot's first item
  __shared__ long long cost_before[kMaxSplitItems + 1];
  __shared__ long long sums[8];
  __shared__ int sums32[8], n_joins;
  const int tid = threadIdx.x, block = 2 * p.tpt;
  for (int i = tid; i < n_items; i += 256) slot_of[i] = -1;
  if (tid == 0) n_joins = 0;
  int at = 0;
  for (int b0 = 0; b0 < p.B; b0 += 256) {                 // (the scan's barriers order the -1 before the marks)
    const SlotRows s = slot_rows(p, b0 + tid);
    const int n = (s.n + block - 1) / block;
    int all_here;
    const int before = block_scan<false>(n, sums32, all_here);
    if (n > 0) slot_of[at + before] = b0 + tid;
    at += all_here;
  }
  __syncthreads();
  long long total = 0;
  int last_start = 0;
  for (int i0 = 0; i0 < n_items; i0 += 256) {
    const int i = i0 + tid;
    int start, unused;
    {
      const int marked = i < n_items && slot_of[i] >= 0 ? i : last_start;
      start = block_scan<true>(marked, sums32, unused);
    }
    long long c = 0, here;
    if (i < n_items) {
      const int slot = slot_of[start];
      start_of[i] = start;
      c = block_of(p, slot_rows(p, slot), slot, i - start, block).n_tiles + kEntryCost;
    }
    const long long before = block_scan<false>(c, sums, here);
    if (i < n_items) cost_before[i] = total + before;
    total += here;
    last_start = unused;
  }
  if (tid == 0) cost_before[n_items] = total;
  __syncthreads();
  const long long all = total * p.G;
  const long long share = max((all + p.workers - 1) / p.workers, (long long)(4 + kEntryCost));
  // unit that holds the point x of the line
  auto unit_at = [&](long long x) -> int {
    int lo = 0, n = n_items;
    while (n > 1) {
      const int h = n / 2;
      if (cost_before[lo + h] * p.G <= x) { lo += h; n -= h; } else { n = h; }
    }
    const long long c = cost_before[lo + 1] - cost_before[lo];
    return lo * p.G + (int)((x - cost_before[lo] * p.G) / c);
  };
  for (int w = tid; w < p.workers; w += 256) {
    const long long a = w * share, e = min(a + share, all);
    p.header->begin[w] = a < all ? unit_at(a) + w : 0;
    p.header->end[w] = a < all ? unit_at(e - 1) + w + 1 : 0;
  }
  for (int u = tid; u < n_items * p.G; u += 256) {
    const int item = u / p.G, g = u - item * p.G;
    const long long c = cost_before[item + 1] - cost_before[item];
    const long long from = cost_before[item] * p.G + g * c;
    const int st = start_of[item], slot = slot_of[st];
    const PackedItem it = block_of(p, slot_rows(p, slot), slot, item - st, block);
    const int n = it.n_tiles, lo_all = it.tile_lo;
    // tiles in front of the point `x` of the item; pieces of one tile are not worth their epilogue
    auto tiles_before = [&](long long x) -> int {
      const long long t = x - kEntryCost / 2;
      return t < 2 ? 0 : t > n - 2 ? n : (int)t;
    };
    const int w1 = (int)(from / share), w2 = (int)((from + c - 1) / share);
    auto cut = [&](int w) { return tiles_before(min(max((long long)w * share - from, 0ll), c)); };
    int w_lo = -1, w_hi = -1;
    for (int w = w1; w <= w2; ++w)
      if (cut(w) < cut(w + 1)) { if (w_lo < 0) w_lo = w; w_hi = w; }
    for (int w = w1; w <= w2; ++w) {
      const int lo = cut(w), hi = cut(w + 1);
      PackedItem piece = it;
      int part = 0;
      if (lo < hi) {
        piece.tile_lo = lo_all + lo;
        piece.n_tiles = hi - lo;
        if (w_lo < w_hi) part = 1 + (w == w1 && from > w1 * share ? 2 * w + 1 : 2 * w);
      } else if (n > 0 || w > w1) {
        piece.n_tok = piece.n_tiles = 0;
      }
      piece.g_part = g | (part << 16);
      p.items[u + w] = piece;
    }
    if (w_lo < w_hi) {
      JoinEntry j;
      j.row0 = it.row0; j.n_tok = it.n_tok; j.g = g;
      j.w_lo = w_lo; j.w_hi = w_hi;
      j.part_lo = w_lo == w1 && from > w1 * share ? 2 * w_lo + 1 : 2 * w_lo;
      j.pad[0] = j.pad[1] = 0;
      p.header->joins[atomicAdd(&n_joins, 1)] = j;       // (every split item lies on a boundary of its own: fewer than workers)
    }
  }
  __syncthreads();
  if (tid == 0) {
    p.header->n_entries = 0;
    p.header->shares = 1;
    p.header->n_joins = n_joins;
  }
}

// Lists the items.  Whole ones are sorted by the position they end at (heaviest first; under a sliding
// window everything past the window weighs the same).  Within a slot that position grows by `block` from
// item to item, so how many items of another slot come before a given one is a closed form, and one
// warp ranks an item with one look at every slot: no sort, no pass in between, any number of warps.
__global__ void __launch_bounds__(256) plan_kernel(const __grid_constant__ PackedParams p) {
  wait_for_launch_before();
  let_next_launch_start();
  const int lane = threadIdx.x & 31;
  const int warp = blockIdx.x * 8 + (threadIdx.x >> 5);
  const int block = 2 * p.tpt;
  const int cap = p.sliding_window > 0 ? min(p.sliding_window, 0x40000000) + 2 * kBN : 0x7fffffff;
  // which slot and which of its items: a scan over the slots' item counts.  On the way: the longest item and
  // (nearly) the cost of all, both in tiles
  int at = 0, mine = -1, slot = 0, longest = 0;
  float cost = 0.f;
  bool bad = false;
  for (int b0 = 0; b0 < p.B; b0 += 32) {
    const SlotRows s = slot_rows(p, b0 + lane);
    bad |= s.bad;
    const int n = (s.n + block - 1) / block;
    if (n > 0) {
      const int last = min(s.keys, cap), first = p.causal ? min(max(s.time - s.n + block, 0), last) : last;
      longest = max(longest, (last + kBN - 1) / kBN);
      cost += (float)n * ((float)(first + last) / (2 * kBN) + 0.5f + kEntryCost);
    }
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += y;
    }
    const int local = warp - at - (sum - n);
    const unsigned here = __ballot_sync(0xffffffffu, local >= 0 && local < n);
    if (here != 0) {
      slot = b0 + __ffs(here) - 1;
      mine = __shfl_sync(0xffffffffu, local, __ffs(here) - 1);
    }
    at += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (__any_sync(0xffffffffu, bad)) {          // starts that contradict themselves: nothing is computed
    if (warp == 0 && lane == 0) {
      record(p.status, kErrStarts);
      p.header->n_entries = p.header->shares = p.header->n_joins = 0;
    }
    return;
  }
  if (p.may_split) {
    // Shares pay where the longest item alone takes longer than its worker's fair part of everything (and is
    // worth cutting at all).  Both sides: chunks of 1 to 512 rows behind contexts of 777 to 30000 tokens, 8 / 2 heads,
    // longest item 4 times the fair part: 573 us whole, 175 in shares (123 to 146 now), in kernels alike but for that; sixteen prompts
    // of 1 to 2000 rows, longest item half the fair part: 52 us whole, 64 in shares.  Every warp comes to the same answer.
    longest = __reduce_max_sync(0xffffffffu, longest);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) cost += __shfl_xor_sync(0xffffffffu, cost, o);
    if (longest > 8 && at <= kMaxSplitItems && (float)(longest + kEntryCost) * p.workers > 1.1f * cost * p.G) {
      if (blockIdx.x == 0) deal_shares(p, at);
      return;
    }
  }
  if (warp == 0 && lane == 0) {
    p.header->n_entries = at * p.G;            // (at <= N / block + B: the starts do not decrease)
    p.header->shares = p.header->n_joins = 0;
  }
  if (mine < 0) return;
  const SlotRows s = slot_rows(p, slot);
  auto ends_at = [&](int time, int n, int i) { return p.causal ? time - n + min((i + 1) * block, n) : time; };
  const int x = min(ends_at(s.time, s.n, mine), cap);
  int rank = 0;
  for (int b = lane; b < p.B; b += 32) {
    const SlotRows t = slot_rows(p, b);
    const int n = (t.n + block - 1) / block;
    // how many of slot b's items end at or before position y
    auto up_to = [&](int y) { return y >= t.time ? n : (!p.causal || y < t.time - t.n) ? 0 : (y - (t.time - t.n)) / block; };
    const int below = up_to(x - 1), same = x == cap ? n - below : up_to(x) - below;
    rank += n - below - same;
    if (b < slot) rank += same;
    if (b == slot) rank += min(max(mine - below, 0), same);
  }
  rank = __reduce_add_sync(0xffffffffu, rank);
  PackedItem it = block_of(p, s, slot, mine, block);
  if (rank < p.max_items)
    for (int g = lane; g < p.G; g += 32) {
      it.g_part = g;
      p.items[(int64_t)rank * p.G + g] = it;
    }
}

// ---------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------
struct Barriers {
  uint64_t q_full;
  uint64_t kv_full[8];
  uint64_t kv_empty[8];
  uint64_t s_full[2];
  uint64_t p_a[2];          // first quarter-pairs of P(j) written (keys 0..31 and 64..95)
  uint64_t p_b[2];          // the rest of P(j) written
  uint64_t pv_done;
  uint64_t q_empty;         // last Q.K^T of a work item done: the Q buffer may be refilled
  uint64_t o_free;          // the softmax warps have read O out of tensor memory
  uint64_t tail;            // a V chunk whose context ends inside has landed: its rest is zeroed next
  uint64_t pair[4];         // one per softmax warp pair: shared-memory exchanges
  uint32_t tmem_base;
  int32_t abort_flag;
};

template <typename T> struct PackT;
template <> struct PackT<__nv_bfloat16> {
  static constexpr uint32_t kFmt = 1;
  // 8 significant bits: rows that see only a few keys get their probabilities as a
  // (rounded + residue) pair, multiplied by two MMAs
  static constexpr bool kSplitP = true;
  __device__ static __forceinline__ float lo_val(uint32_t v) { return __uint_as_float(v << 16); }
  __device__ static __forceinline__ float hi_val(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
  __device__ static __forceinline__ float sum2(uint32_t v) { return lo_val(v) + hi_val(v); }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};
template <> struct PackT<__half> {
  static constexpr uint32_t kFmt = 0;
  static constexpr bool kSplitP = false;
  __device__ static __forceinline__ float lo_val(uint32_t v) { return __low2float(*reinterpret_cast<const __half2*>(&v)); }
  __device__ static __forceinline__ float hi_val(uint32_t v) { return __high2float(*reinterpret_cast<const __half2*>(&v)); }
  __device__ static __forceinline__ float sum2(uint32_t v) { return lo_val(v) + hi_val(v); }
  __device__ static __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};

// A worker's walk: its share of the line of items or, of whole items, item r * workers + w in round r,
// alternating the direction so that heavy and light ones pair up.  The entry is read one item ahead: fetched at
// the switch itself, the load would hold up the MMA issuer and the softmax warps.
#define G4B_PACKED_LOOP_PROLOGUE()                                                                   \
  PackedItem it_nx_;                                                                                 \
  fetch_item(item_of_round(0), it_nx_)
#define G4B_PACKED_LOOP_HEAD(round)                                                                  \
  const int item = item_of_round(round);                                                             \
  const PackedItem it = it_nx_;                                                                      \
  fetch_item(item_of_round((round) + 1), it_nx_)

template <typename T, int kD>
__global__ void __launch_bounds__(kThreads, 1)
packed_prefill_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                      const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap o_map,
                      const __grid_constant__ PackedParams p) {
  using Gm = Geo<kD>;
  constexpr int kSt = Gm::kStages / 2, kChunk = Gm::kChunkBytes, kSlabs = Gm::kSlabs;
  constexpr int kHalfCols = kD / 2;             // output columns of a softmax warpgroup
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = ptx::cluster_ctarank();   // 0 = the CTA that issues the MMAs
  const bool leader = rank == 0;

  uint8_t* sQ = smem;
  uint8_t* sRing = smem + Gm::kQBytes;
  uint8_t* sStage = sRing + 2 * kSt * kChunk;            // (ring: kSt chunks of K, then kSt of V)
  Barriers* bars = reinterpret_cast<Barriers*>(sStage + kStageBytes);
  float* xchg = reinterpret_cast<float*>(sStage + kStageBytes + 512);
  const uint32_t bar_q = ptx::smem_u32(&bars->q_full);
  const uint32_t bar_pv = ptx::smem_u32(&bars->pv_done);
  if (threadIdx.x == 0) {
    // The barriers the MMA issuer waits on live in CTA 0 and count both CTAs.
    ptx::mbar_init(bar_q, 2);
    for (int s = 0; s < 2 * kSt; ++s) {
      ptx::mbar_init(ptx::smem_u32(&bars->kv_full[s]), 2);
      ptx::mbar_init(ptx::smem_u32(&bars->kv_empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      ptx::mbar_init(ptx::smem_u32(&bars->s_full[s]), 1);
      ptx::mbar_init(ptx::smem_u32(&bars->p_a[s]), 16);   // one arrival per softmax warp
      ptx::mbar_init(ptx::smem_u32(&bars->p_b[s]), 16);
    }
    ptx::mbar_init(bar_pv, 1);
    ptx::mbar_init(ptx::smem_u32(&bars->q_empty), 1);
    ptx::mbar_init(ptx::smem_u32(&bars->o_free), 16);
    ptx::mbar_init(ptx::smem_u32(&bars->tail), 1);
    for (int s = 0; s < 4; ++s) ptx::mbar_init(ptx::smem_u32(&bars->pair[s]), 2);
    ptx::fence_barrier_init();
    ptx::prefetch_tensormap(&q_map);
    ptx::prefetch_tensormap(&k_map);
    ptx::prefetch_tensormap(&v_map);
    // An earlier CTA gave up on a wait (0x3xx; a bad table entry is not one): drain the grid.  One
    // thread reads so that all agree.  The swizzled tiles need the buffer on a 1024-byte boundary.
    if (leader) {
      int32_t a = *reinterpret_cast<volatile int32_t*>(p.status);
      if ((a & 0xf00) != 0x300 || a == kErrBadPage) a = 0;
      if (a == 0 && (ptx::smem_u32(smem) & 1023u) != 0) { record(p.status, kErrSmemAlign); a = kErrSmemAlign; }
      bars->abort_flag = a;
      ptx::st_cluster_u32(ptx::map_to_cta(ptx::smem_u32(&bars->abort_flag), 1), (uint32_t)a);
    }
  }
  // rows of the tile that no (token, head) pair fills (group sizes that do not divide 128) are never
  // loaded: zero, once
  if (p.tpt * p.group < kBM) {
    for (int i = threadIdx.x; i < Gm::kQBytes / 16; i += kThreads) reinterpret_cast<uint4*>(sQ)[i] = make_uint4(0u, 0u, 0u, 0u);
    ptx::fence_proxy_async_smem();
  }
  ptx::cluster_sync_all();
  if (*reinterpret_cast<volatile int32_t*>(&bars->abort_flag) != 0) {
    wait_for_launch_before();           // (what follows this launch may rely on the one before it being done)
    return;
  }

  if (warp == 9) {
    ptx::tmem_alloc_pair(ptx::smem_u32(&bars->tmem_base), 512);
    ptx::tmem_relinquish_pair();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(&bars->tmem_base);

  wait_for_launch_before();             // the list of items is complete
  let_next_launch_start();
  const int n_workers = (int)gridDim.x / 2, worker = (int)blockIdx.x / 2;
  const bool shares = __ldcg(&p.header->shares) != 0;
  const int first_entry = shares ? __ldcg(&p.header->begin[worker]) : 0;
  const int last_entry = shares ? __ldcg(&p.header->end[worker]) : __ldcg(&p.header->n_entries);
  const int n_rounds = shares ? last_entry - first_entry : (last_entry + n_workers - 1) / n_workers;
  auto item_of_round = [&](int round) -> int {
    if (round >= n_rounds) return -1;
    const int item = shares ? first_entry + round : round * n_workers + ((round & 1) ? n_workers - 1 - worker : worker);
    return item < last_entry ? item : -1;
  };
  auto fetch_item = [&](int item, PackedItem& out) {
    if (item < 0) { out.n_tok = 0; out.n_tiles = 0; return; }
    const int4* src = reinterpret_cast<const int4*>(p.items + item);
    const int4 a = __ldcg(src), c = __ldcg(src + 1);
    out = PackedItem{a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
  };
  // rows of the block that see fewer than 64 keys: the precise path (for the whole block, both CTAs)
  auto sees_few = [&](const PackedItem& x) {
    return (p.causal ? x.qpos0 : x.window - 1) < 64 || (p.sliding_window > 0 && p.sliding_window < 64);
  };
  // where this CTA's arrivals for the MMA issuer go (CTA 0's copy of the barrier)
  auto issuer_bar = [&](uint64_t* local) -> uint32_t { return ptx::map_to_cta(ptx::smem_u32(local), 0); };
  // one arrival per warp: every lane has finished (and fenced) its own tensor-memory stores.  P lives in
  // tensor memory (ordered by tcgen05.wait::st + tcgen05.fence), so the arrival needs no ordering of its own
  auto arrive_issuer = [&](uint32_t bar) {
    __syncwarp();
    if (lane == 0) ptx::mbar_arrive_cluster_relaxed(bar);
  };

  if (warp >= 8) {
  give_registers();       // (all four warps of the group, the idle one too)
  if (warp == 8 || warp == 10) {
    // =============================== producers ===============================
    // Warp 8 fetches Q and K, warp 10 V: a page of 16 rows is a box of 2 KB (V: 4), two dozen of them a tile, and one
    // warp does not issue them as fast as the tensor pipe consumes them (with 2 KB boxes of V too: 4 prompts of 8192 rows, 8 / 2 heads,
    // pages of 16: 1153 us with one producer warp, 846 us with two).
    // Each has its own half of the ring: with one ring the V warp, which nothing holds up at an item switch, came to a
    // slot whose use before (a K chunk) was not even issued, and the slot's one-bit phase cannot tell that apart.
    const bool for_k = warp == 8, for_v = warp == 10;
    const uint64_t pol_kv = ptx::policy_evict_last();    // K/V tiles are re-read by every block of the slot
    const uint64_t pol_q = ptx::policy_evict_first();
    const uint32_t q_bytes = (uint32_t)(kSlabs * p.tpt * p.group * 128);
    const uint32_t bar_tail = ptx::smem_u32(&bars->tail);
    uint32_t cc = 0;   // chunks of this warp so far (runs on across work items)
    uint32_t tails = 0;
    int n_done = 0;
    bool ok = true;
    G4B_PACKED_LOOP_PROLOGUE();
    for (int round = 0; round < n_rounds && ok; ++round) {
      G4B_PACKED_LOOP_HEAD(round);
      if (item < 0 || it.n_tiles <= 0) continue;
      const int g = it.g_part & 0xffff;
      const int32_t* bt = p.block_tables + it.slot * p.bt_s0;
      const int page_mask = (1 << p.page_shift) - 1;
      auto wait_lane0 = [&](uint32_t bar, uint32_t parity, int32_t code) -> bool {
        int w = 1;
        if (lane == 0) w = ptx::mbar_wait(bar, parity) ? 1 : 0;
        w = __shfl_sync(0xffffffffu, w, 0);
        if (!w) { if (lane == 0) record(p.status, code); ok = false; }
        return w != 0;
      };
      // the Q buffer is free once the last Q.K^T of the previous item has run
      if (for_k && n_done > 0 && !wait_lane0(ptx::smem_u32(&bars->q_empty), (n_done - 1) & 1, kErrQEmpty)) break;
      if (for_k && lane == 0) {
        const uint32_t qb = issuer_bar(&bars->q_full);
        ptx::mbar_arrive_expect_tx_cluster(qb, q_bytes);
        for (int s = 0; s < kSlabs; ++s)
          ptx::tma_load_3d_pair(ptx::smem_u32(sQ + s * 16384), &q_map, qb, s * 64, g * p.group, it.row0 + (int)rank * p.tpt, pol_q);
      }
      // page of the group of `rows` keys that starts at `key`; num_pages (outside the pool: zero fill) for groups past
      // the context, in front of every row's window (their pages may be gone) and for bad entries
      const int first_key = p.sliding_window > 0 ? it.qpos0 - p.sliding_window + 1 : 0;
      auto page_of = [&](int key, int rows) -> int {
        if (key >= it.window || key + rows <= first_key) return p.num_pages;
        const int pg = key >> p.page_shift;          // (< max_pages: the window is bounded by the table)
        const int id = bt[pg * p.bt_s1];
        if (id < 0 || id >= p.num_pages) { record(p.status, kErrBadPage); return p.num_pages; }
        return id;
      };
      // slot of this warp's next chunk
      const int st_base = for_v ? kSt : 0;
      auto wait_empty = [&](int st) { return wait_lane0(ptx::smem_u32(&bars->kv_empty[st]), ((cc / kSt) & 1) ^ 1, kErrKvEmpty); };
      // K chunk = this CTA's 64 keys of the tile x kD (slabs of [64 rows x 64 d]); V chunk = all 128 keys x
      // this CTA's half of the head dim, group by group of rows (a group: slabs of [v_rows x 64 d]), since a step of
      // the product takes 16 keys and does not care where the next 16 lie: one box a group, where K needs one a group and
      // slab (sixteen prompts over pages of 16: 56.3 -> 55.2 us).  Lane i fetches the i-th group of rows.  Every CTA accounts for its own bytes on CTA 0's barrier.
      auto load_k = [&](int j) {
        const int key0 = (it.tile_lo + j) * kBN + 64 * (int)rank + lane * p.k_rows;
        const int boxes = 64 / p.k_rows;
        const int page = lane < boxes ? page_of(key0, p.k_rows) : 0;
        const int st = st_base + cc % kSt;
        if (!wait_empty(st)) return;
        const uint32_t full = issuer_bar(&bars->kv_full[st]);
        if (lane == 0) ptx::mbar_arrive_expect_tx_cluster(full, kChunk);
        __syncwarp();
        if (lane < boxes) {
          const uint32_t dst = ptx::smem_u32(sRing + st * kChunk + lane * p.k_rows * 128);
#pragma unroll
          for (int s = 0; s < kSlabs; ++s)
            ptx::tma_load_4d_pair(dst + s * 8192, &k_map, full, s * 64, key0 & page_mask, g, page, pol_kv);
        }
        __syncwarp();
        ++cc;
      };
      auto load_v = [&](int j) {
        const int tile0 = (it.tile_lo + j) * kBN;
        const int key0 = tile0 + lane * p.v_rows;
        const int boxes = kBN / p.v_rows;
        const int page = lane < boxes ? page_of(key0, p.v_rows) : 0;
        const int live = min(it.window - tile0, kBN);           // rows of this tile that exist
        const int dirty = live % p.v_rows;                      // the context ends inside a group
        const int st = st_base + cc % kSt;
        if (!wait_empty(st)) return;
        const uint32_t full = issuer_bar(&bars->kv_full[st]);
        const uint32_t bar = dirty != 0 ? bar_tail : full;
        if (lane == 0) {
          if (dirty != 0) ptx::mbar_arrive_expect_tx(bar, kChunk);
          else ptx::mbar_arrive_expect_tx_cluster(bar, kChunk);
        }
        __syncwarp();
        uint8_t* chunk = sRing + st * kChunk;
        if (lane < boxes) {
          const uint32_t dst = ptx::smem_u32(chunk + lane * p.v_rows * (128 * kSlabs / 2));
          const int slab = (int)rank * (kSlabs / 2);
          if (dirty != 0) ptx::tma_load_5d_hint(dst, &v_map, bar, 0, key0 & page_mask, slab, g, page, pol_kv);
          else ptx::tma_load_5d_pair(dst, &v_map, bar, 0, key0 & page_mask, slab, g, page, pol_kv);
        }
        __syncwarp();
        if (dirty != 0) {
          // rows [live, end of the group) hold whatever the page held: zero them before the MMAs may read
          if (!wait_lane0(bar_tail, tails & 1, kErrTail)) return;
          ++tails;
          const int rows = p.v_rows - dirty;
          for (int i = lane; i < rows * 8 * (kSlabs / 2); i += 32) {
            const int s = i / (rows * 8), at = i - s * rows * 8;
            *reinterpret_cast<uint4*>(chunk + (live - dirty) * (128 * kSlabs / 2) + s * p.v_rows * 128 + dirty * 128 + at * 16) =
                make_uint4(0u, 0u, 0u, 0u);
          }
          ptx::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive_cluster(full);
        }
        ++cc;
      };
      for (int j = 0; j < it.n_tiles && ok; ++j) {
        if (for_k) load_k(j);
        else load_v(j);
      }
      ++n_done;
    }
  } else if (warp == 9) {
    // =============================== MMA issuer ===============================
    // Only CTA 0 issues.  One MMA spans both CTAs: rows 0..127 of the 256-row tile (A operand,
    // accumulator, P) are CTA 0's, rows 128..255 CTA 1's; the B operand is split between the two
    // shared memories (K: keys 0..63 | 64..127, V: the halves of the head dim) at the same offsets.
    if (leader) {
      constexpr uint32_t idesc_qk = ptx::make_idesc_f16(PackT<T>::kFmt, 256, 128, 0, 0);
      constexpr uint32_t idesc_pv = ptx::make_idesc_f16(PackT<T>::kFmt, 256, kD, 0, 1);
      constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);   // SBO 1024 B, version 1, SWIZZLE_128B
      constexpr uint32_t kLoKMajor = 1u << 16;
      const uint32_t v_slab = (uint32_t)p.v_rows * 128;       // LBO: 64-wide slabs of a group of rows lie behind one another
      const uint32_t lo_v_major = (v_slab >> 4) << 16;
      uint32_t v_step[8];                                     // where the 16 keys of a step lie (one slab: behind one another)
#pragma unroll
      for (int k16 = 0; k16 < 8; ++k16)
        v_step[k16] = (k16 * 16 / p.v_rows * p.v_rows * (128 * kSlabs / 2) + k16 * 16 % p.v_rows * 128) >> 4;
      const uint32_t q_lo = (ptx::smem_u32(sQ) >> 4) | kLoKMajor;
      const uint32_t ring_lo = ptx::smem_u32(sRing) >> 4;
      auto wait_all = [&](uint32_t bar, uint32_t parity) -> bool { return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity)); };
      auto commit_both = [&](uint64_t* local) {   // same barrier in CTA 0 and CTA 1
        const uint32_t a = ptx::smem_u32(local);
        ptx::tc_commit_pair(ptx::map_to_cta(a, 0));
        ptx::tc_commit_pair(ptx::map_to_cta(a, 1));
      };
      bool ok = true;
      uint32_t kc = 0, vc = 0;     // chunks of K and V so far
      int tg = 0;       // tiles issued so far: S buffer and barrier phases run on across items
      int n_done = 0;
      G4B_PACKED_LOOP_PROLOGUE();
      for (int round = 0; round < n_rounds && ok; ++round) {
        G4B_PACKED_LOOP_HEAD(round);
        if (item < 0 || it.n_tiles <= 0) continue;
        const int n_tiles = it.n_tiles;
        const bool precise = PackT<T>::kSplitP && sees_few(it);
        ok = wait_all(bar_q, n_done & 1);
        if (!ok) { if (lane == 0) record(p.status, kErrQFull); break; }
        ptx::tc_fence_after();
        auto issue_qk = [&](int j) {
          const int t = tg + j;
          const uint32_t d_tmem = tmem + ((t & 1) ? kColS1 : kColS0);
          const int st = kc % kSt;
          if (!wait_all(ptx::smem_u32(&bars->kv_full[st]), (kc / kSt) & 1)) {
            if (lane == 0) record(p.status, kErrKvFull);
            ok = false; return;
          }
          ptx::tc_fence_after();
          const uint32_t k_lo = (ring_lo + st * (kChunk >> 4)) | kLoKMajor;
          if (ptx::elect_one()) {
#pragma unroll
            for (int k16 = 0; k16 < kD / 16; ++k16) {
              const uint32_t aoff = ((k16 >> 2) * 16384 + (k16 & 3) * 32) >> 4;   // Q: slabs of 128 rows
              const uint32_t boff = ((k16 >> 2) * 8192 + (k16 & 3) * 32) >> 4;    // K: slabs of 64 rows
              ptx::mma_ss_pair(d_tmem, ptx::desc64(q_lo + aoff, kDescHi), ptx::desc64(k_lo + boff, kDescHi), idesc_qk, k16 != 0);
            }
            commit_both(&bars->kv_empty[st]);
            commit_both(&bars->s_full[t & 1]);
            if (j == n_tiles - 1) commit_both(&bars->q_empty);   // last use of this item's Q
          }
          __syncwarp();
          ++kc;
        };
        auto issue_pv = [&](int j) {
          const int st = kSt + vc % kSt;
          if (!wait_all(ptx::smem_u32(&bars->kv_full[st]), (vc / kSt) & 1)) {
            if (lane == 0) record(p.status, kErrKvFull);
            ok = false; return;
          }
          const int t = tg + j;
          const uint32_t v_lo = (ring_lo + st * (kChunk >> 4)) | lo_v_major;
          const uint32_t p_tmem = tmem + ((t & 1) ? kColS1 : kColS0);
          if (j == 0 && n_done > 0) {
            // the first product of an item overwrites O: the previous item's O must have been read
            if (!wait_all(ptx::smem_u32(&bars->o_free), (n_done - 1) & 1)) {
              if (lane == 0) record(p.status, kErrOFree);
              ok = false; return;
            }
            ptx::tc_fence_after();
          }
          for (int part = 0; part < 2 && ok; ++part) {
            const uint32_t bar = ptx::smem_u32(part == 0 ? &bars->p_a[t & 1] : &bars->p_b[t & 1]);
            if (!wait_all(bar, (t >> 1) & 1)) {
              if (lane == 0) record(p.status, kErrPFull);
              ok = false; return;
            }
            ptx::tc_fence_after();
            if (ptx::elect_one()) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                // part 0: keys 0..31 and 64..95 (k16 = 0,1,4,5); part 1: the rest
                const int k16 = (i >> 1) * 4 + part * 2 + (i & 1);
                const uint64_t vdesc = ptx::desc64(v_lo + (kSlabs == 2 ? k16 * 2048 >> 4 : v_step[k16]), kDescHi);
                ptx::mma_ts_pair(tmem + kColO, p_tmem + k16 * 8, vdesc, idesc_pv, (j | part | i) != 0);
                if (precise) ptx::mma_ts_pair(tmem + kColO, p_tmem + 64 + k16 * 8, vdesc, idesc_pv, 1u);
              }
              if (part == 1) {
                commit_both(&bars->kv_empty[st]);
                commit_both(&bars->pv_done);
              }
            }
            __syncwarp();
          }
          ++vc;
        };
        issue_qk(0);
        if (ok && n_tiles > 1) issue_qk(1);
        for (int j = 0; j < n_tiles && ok; ++j) {
          issue_pv(j);
          if (ok && j + 2 < n_tiles) issue_qk(j + 2);
        }
        tg += n_tiles;
        ++n_done;
      }
    }
    __syncwarp();
  }
  } else {
    // =============================== softmax / epilogue ===============================
    // Two warpgroups share every row: warps 0..3 own the first 64 keys of a tile (and the first half of
    // O's columns), warps 4..7 the other 64.  A warp and its partner (warp + 4, same TMEM lanes) trade
    // row maxima through shared memory.
    take_registers();
    const int half = warp >> 2;
    const int lane_base = (warp & 3) * 32;
    const int r = lane_base + lane;                       // row of the tile = TMEM lane
    const uint32_t trow = tmem + ((uint32_t)lane_base << 16);
    const uint32_t pair_bar = ptx::smem_u32(&bars->pair[warp & 3]);
    uint8_t* stage = sStage + warp * 4096;
    const int tok_r = (int)rank * p.tpt + (r * p.group_mul >> 16);    // this row's token of the block ...
    const bool in_tile = r < p.tpt * p.group;
    uint32_t pair_phase = 0;
    // bounded rendezvous of the two warps that share these rows; false when the partner never arrived
    auto pair_sync = [&]() -> bool {
      __syncwarp();
      if (lane == 0) ptx::mbar_arrive(pair_bar);
      const bool w = __all_sync(0xffffffffu, ptx::mbar_wait(pair_bar, pair_phase & 1));
      ++pair_phase;
      return w;
    };
    // Stores 32 rows x 128 bytes out of this warp's stage.  `bytes0`: offset of the piece inside an output row.
    // Rows that all exist leave as one TMA box, which the copy engine reads while the warp moves on (64 KB
    // an item, stored by the warps themselves, cost them 3500 cycles of an item's 20000 under a window of 512 keys);
    // otherwise eight lanes store a row, so that a row piece is one whole line.
    const uint64_t pol_o = ptx::policy_evict_first();    // the output is not read again here
    auto stage_free = [&]() {
      if (lane == 0) ptx::bulk_wait_read_all();
      __syncwarp();
    };
    const int osz = p.o_dtype == G4B_F32 ? 4 : 2;
    auto store_stage = [&](const PackedItem& it, int g, int part, int bytes0) {
      // rows are (token, head) pairs in this order, so those that exist are the first
      const int rows_valid = min(it.n_tok - (int)rank * p.tpt, p.tpt) * p.group - lane_base;
      if (p.o_boxes && part == 0 && rows_valid >= 32) {
        ptx::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          const int tok = lane_base * p.group_mul >> 16;
          ptx::tma_store_3d_hint(&o_map, ptx::smem_u32(stage), bytes0 >> 1, g * p.group + lane_base - tok * p.group,
                                 it.row0 + (int)rank * p.tpt + tok, pol_o);
          ptx::bulk_commit();
        }
        return;
      }
      __syncwarp();
      const int c = lane & 7;
      char* base = part > 0 ? (char*)p.parts + (int64_t)(part - 1) * kPartBytes + ((int)rank * kBM + lane_base) * (kD * 4)
                            : (char*)p.o + ((int64_t)(it.row0 + (int)rank * p.tpt) * p.o_row + (int64_t)(g * p.group) * p.o_head) * osz;
      base += bytes0 + c * 16;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = i * 4 + (lane >> 3);
        if (row < rows_valid) {
          const uint4 val = *reinterpret_cast<const uint4*>(stage + row * 128 + ((c ^ (row & 7)) << 4));
          const int tok = (lane_base + row) * p.group_mul >> 16, head = lane_base + row - tok * p.group;
          const int64_t off = part > 0 ? (int64_t)row * (kD * 4) : (tok * p.o_row + head * p.o_head) * osz;
          *reinterpret_cast<uint4*>(base + off) = val;
        }
      }
      __syncwarp();
    };
    bool ok = true;
    int tg = 0;
    int n_done = 0;
    // The reference maximum a row ended the last item with is the first guess for the same row of the
    // next one.  A guess at most 2^8 below or 2^4 above the first maximum the row really sees is kept --
    // any reference in that range is as good as the maximum itself -- so the first tile of an item
    // can take the optimistic path too.
    float m_carry = -INFINITY;
    // (the next entry is fetched behind the tile loop, where registers are free, and arrives during the epilogue)
    G4B_PACKED_LOOP_PROLOGUE();
    for (int round = 0; round < n_rounds && ok; ++round) {
      const int item = item_of_round(round);
      const PackedItem it = it_nx_;
      auto fetch_next = [&]() { fetch_item(item_of_round(round + 1), it_nx_); };
      if (item < 0) continue;
      const int n_tiles = it.n_tiles;
      if (n_tiles <= 0) {
        const int g = it.g_part & 0xffff;
        fetch_next();
        // no visible key for any row of the block: the output rows are zero
        stage_free();
        for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(stage + lane * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
        for (int c = 0; c < kHalfCols * osz / 128; ++c) store_stage(it, g, 0, half * kHalfCols * osz + c * 128);
        continue;
      }
      const int window = it.window;
      const bool few_keys = sees_few(it);
      const int qpos = it.qpos0 + tok_r;
      const int qpos_min = it.qpos0 + (int)rank * p.tpt;       // of this CTA's rows
      const int qpos_max = qpos_min + p.tpt - 1;
      const int key_lo = p.sliding_window > 0 ? max(0, qpos_min - p.sliding_window + 1) : 0;
      int hi_r = p.causal ? min(window, qpos + 1) : window;
      if (!in_tile) hi_r = 0;
      const int lo_r = p.sliding_window > 0 ? max(0, qpos - p.sliding_window + 1) : 0;
      float m_used = !few_keys ? m_carry : -INFINITY;   // reference maximum the accumulated O and l are scaled by
      bool anchored = false;      // m_used has been checked against a key this row sees
      float l_run = 0.f;          // this thread's half of the row sum

      for (int j = 0; j < n_tiles && ok; ++j) {
        const int t = tg + j;
        const uint32_t s_col = (t & 1) ? kColS1 : kColS0;
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(ptx::smem_u32(&bars->s_full[t & 1]), (t >> 1) & 1))) {
          record(p.status, kErrSFull); ok = false; break;
        }
        ptx::tc_fence_after();
        uint32_t sraw[2][32];       // this thread's half of a row of scores
        ptx::tmem_ld32(trow + s_col + half * 64, sraw[0]);
        ptx::tmem_ld32(trow + s_col + half * 64 + 32, sraw[1]);
        ptx::tc_wait_ld32x2(sraw[0], sraw[1]);
        const int kbase = (it.tile_lo + j) * kBN;
        // warp-uniform: does any row of this CTA need element masks in this tile?
        const bool need_mask = (p.causal && kbase + kBN - 1 > qpos_min) || (kbase + kBN > window) || (kbase < key_lo) ||
                               (p.sliding_window > 0 && kbase < qpos_max - p.sliding_window + 1);
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (need_mask) {
          // the keys this row sees are one range [nlo, nhi) of the thread's 64: one bit per key
          const int nlo = lo_r - kbase - half * 64, nhi = hi_r - kbase - half * 64;
#pragma unroll
          for (int q2 = 0; q2 < 2; ++q2) {
            const int lo = min(max(nlo - 32 * q2, 0), 32), hi = min(max(nhi - 32 * q2, 0), 32);
            const uint32_t below_hi = hi >= 32 ? 0xffffffffu : ((1u << hi) - 1u);
            const uint32_t below_lo = lo >= 32 ? 0xffffffffu : ((1u << lo) - 1u);
            const uint32_t bits = below_hi & ~below_lo;
#pragma unroll
            for (int i = 0; i < 32; ++i) sraw[q2][i] = (bits & (1u << i)) ? sraw[q2][i] : 0xff800000u;
          }
        }
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            mx4[(i >> 1) & 3] = ptx::max3(mx4[(i >> 1) & 3], __uint_as_float(sraw[q2][i]), __uint_as_float(sraw[q2][i + 1]));
        float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        // publish the half-row maximum for the partner warp; collect the partner's later.  The buffers
        // alternate with every rendezvous of the pair, so a write cannot overtake the partner's read
        float* xm = xchg + (pair_phase & 1) * (2 * kBM);
        xm[half * kBM + r] = mx;
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(pair_bar);

        const uint32_t bar_pa = issuer_bar(&bars->p_a[t & 1]);
        const uint32_t bar_pb = issuer_bar(&bars->p_b[t & 1]);
        uint32_t pk[32];
        // Optimistic path: the reference maximum rarely moves (it only has to stay within 2^8 of the
        // true one), so start exponentiating against the current one while the maxima are traded.
        bool fast = !few_keys && __all_sync(0xffffffffu, m_used != -INFINITY);
        float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        auto weights = [&](const uint32_t (&x)[32], float neg_m, uint32_t* out) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 e = ptx::fma2(make_float2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])),
                                       make_float2(p.scale_log2, p.scale_log2), make_float2(neg_m, neg_m));
            const float2 w = make_float2(ptx::ex2_approx(e.x), ptx::ex2_approx(e.y));
            sum2[(i >> 1) & 1] = ptx::add2(sum2[(i >> 1) & 1], w);
            out[i >> 1] = PackT<T>::pack(w.x, w.y);
          }
        };
        if (fast) {
          const float neg_m = -m_used;
          weights(sraw[0], neg_m, pk);
        }
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(pair_bar, pair_phase & 1))) {
          record(p.status, kErrPair); ok = false; break;
        }
        ++pair_phase;
        mx = fmaxf(mx, xm[(half ^ 1) * kBM + r]);
        const float m_blk = mx * p.scale_log2;
        bool exceed = m_blk > m_used + 8.f;
        bool first_seen = false;
        if (!few_keys && !anchored && m_blk != -INFINITY) {
          // the row's first visible key: a guess that lies too far ABOVE is replaced as well (nothing has
          // been accumulated against it yet, so nothing is rescaled)
          first_seen = anchored = true;
          exceed = exceed || m_blk < m_used - 4.f;   // (f16 probabilities: keep them well above the subnormals)
        }
        if (fast && __any_sync(0xffffffffu, exceed)) fast = false;   // same outcome in the partner warp

        if (fast) {
          // first 32 keys of this half are final: let the P.V product start on them
          ptx::tmem_st16(trow + s_col + half * 32, pk);
          ptx::tc_wait_st();
          ptx::tc_fence_before();
          arrive_issuer(bar_pa);
          const float neg_m = -m_used;
          weights(sraw[1], neg_m, pk + 16);
          ptx::tmem_st16(trow + s_col + half * 32 + 16, pk + 16);
          l_run += (sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y);
          // keep the PV-done phase bookkeeping in step (no stall: PV(j-1) ended long ago); before P(j) is handed over,
          // since a warp held up behind that could find PV(j) done too and its one-bit phase as it was
          if (j > 0 && !__all_sync(0xffffffffu, ptx::mbar_wait(bar_pv, (t - 1) & 1))) {
            record(p.status, kErrPvDone); ok = false; break;
          }
          ptx::tc_wait_st();
          ptx::tc_fence_before();
          arrive_issuer(bar_pb);
          continue;
        }

        // The reference maximum moves (first tile of an item, or a jump of more than 2^8: lazy rescale -- p
        // stays <= 256, exact enough in f32 sums and representable in f16/bf16), or some row of the
        // block sees fewer than 64 keys.
        float alpha = 1.f;
        bool rescale = false;
        if (exceed) {
          rescale = (m_used != -INFINITY) && !first_seen;
          alpha = rescale ? ptx::ex2_approx(m_used - m_blk) : 1.f;
          m_used = m_blk;
        }
        l_run *= alpha;
        const float neg_m = (m_used == -INFINITY) ? 0.f : -m_used;
        float sum4[4] = {0.f, 0.f, 0.f, 0.f};
        // O may only be touched once PV(j-1) has drained, and must be rescaled before any part of P(j) is
        // published
        if (j > 0) {
          if (!__all_sync(0xffffffffu, ptx::mbar_wait(bar_pv, (t - 1) & 1))) { record(p.status, kErrPvDone); ok = false; break; }
          ptx::tc_fence_after();
          if (__any_sync(0xffffffffu, rescale)) {
#pragma unroll 1
            for (int c = 0; c < kHalfCols / 32; ++c) {
              uint32_t ov[32];
              ptx::tmem_ld32(trow + kColO + half * kHalfCols + c * 32, ov);
              ptx::tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
              ptx::tmem_st32(trow + kColO + half * kHalfCols + c * 32, ov);
            }
          }
        }
#pragma unroll
        for (int q2 = 0; q2 < 2; ++q2) {
          uint32_t plo[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float p0 = ptx::ex2_approx(fmaf(__uint_as_float(sraw[q2][i]), p.scale_log2, neg_m));
            const float p1 = ptx::ex2_approx(fmaf(__uint_as_float(sraw[q2][i + 1]), p.scale_log2, neg_m));
            const uint32_t packed = PackT<T>::pack(p0, p1);
            pk[i >> 1] = packed;
            if (few_keys) {
              // rows that see only a few keys: sum the ROUNDED probabilities the tensor core multiplies, so
              // numerator and denominator agree (exact for one visible key) ...
              sum4[(i >> 1) & 3] += PackT<T>::sum2(packed);
              if constexpr (PackT<T>::kSplitP) {
                // ... and give bf16 its rounding residue back through a second product
                const uint32_t lo = PackT<T>::pack(p0 - PackT<T>::lo_val(packed), p1 - PackT<T>::hi_val(packed));
                sum4[(i >> 1) & 3] += PackT<T>::sum2(lo);
                plo[i >> 1] = lo;
              }
            } else {
              sum4[(i >> 1) & 3] += p0 + p1;
            }
          }
          ptx::tmem_st16(trow + s_col + half * 32 + q2 * 16, pk);
          if constexpr (PackT<T>::kSplitP) {
            if (few_keys) ptx::tmem_st16(trow + s_col + 64 + half * 32 + q2 * 16, plo);
          }
          ptx::tc_wait_st();
          ptx::tc_fence_before();
          arrive_issuer(q2 == 0 ? bar_pa : bar_pb);
        }
        l_run += (sum4[0] + sum4[1]) + (sum4[2] + sum4[3]);
      }

      if (!few_keys && m_used != -INFINITY) m_carry = m_used;
      // (what the epilogue needs of the entry is read again: kept through the tile loop it costs registers there)
      PackedItem me;
      fetch_item(item, me);
      fetch_next();
      const int g = me.g_part & 0xffff;
      // ---- epilogue: O / l -> global ----
      if (ok) {
        if (!__all_sync(0xffffffffu, ptx::mbar_wait(bar_pv, (tg + n_tiles - 1) & 1))) { record(p.status, kErrPvDone); ok = false; }
        ptx::tc_fence_after();
      }
      // the row sum is the sum of both halves (both scaled by the same m_used)
      if (ok) {
        float* xl = xchg + (pair_phase & 1) * (2 * kBM);
        xl[half * kBM + r] = l_run;
        if (!pair_sync()) { record(p.status, kErrPair); ok = false; }
        l_run += xl[(half ^ 1) * kBM + r];
      }
      if (ok) {
        const float inv_l = l_run > 0.f ? 1.f / l_run : 0.f;
        const uint32_t o_col = trow + kColO + half * kHalfCols;
        auto put = [&](int c, uint32_t a, uint32_t b2, uint32_t c2, uint32_t d) {
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((c ^ (lane & 7)) << 4)) = make_uint4(a, b2, c2, d);
        };
        const int part = me.g_part >> 16;
        if (part > 0 || p.o_dtype == G4B_F32) {
          // f32 rows: an output of that type, or a part (un-normalised, with its sum and reference maximum in
          // log2 units; a row that saw no key here has neither)
          const float factor = part > 0 ? 1.f : inv_l;
          if (part > 0 && half == 0 && in_tile && tok_r < me.n_tok)
            *reinterpret_cast<float2*>(p.header->part_lm[part - 1][(int)rank * kBM + r]) = make_float2(l_run, l_run == 0.f ? -INFINITY : m_used);
#pragma unroll 1
          for (int c = 0; c < kHalfCols / 32; ++c) {
            uint32_t ov[32];
            ptx::tmem_ld32(o_col + c * 32, ov);
            ptx::tc_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * factor);
            stage_free();
#pragma unroll
            for (int i = 0; i < 8; ++i) put(i, ov[4 * i], ov[4 * i + 1], ov[4 * i + 2], ov[4 * i + 3]);
            store_stage(me, g, part, (half * kHalfCols + c * 32) * 4);
          }
          ptx::tc_fence_before();
          arrive_issuer(issuer_bar(&bars->o_free));
        } else {
#pragma unroll
          for (int c = 0; c < kHalfCols / 64; ++c) {
            uint32_t pk[2][16];
#pragma unroll
            for (int c2 = 0; c2 < 2; ++c2) {
              uint32_t ov[32];
              ptx::tmem_ld32(o_col + (2 * c + c2) * 32, ov);
              ptx::tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                pk[c2][i] = PackT<T>::pack(__uint_as_float(ov[2 * i]) * inv_l, __uint_as_float(ov[2 * i + 1]) * inv_l);
            }
            if (c == kHalfCols / 64 - 1) {
              // O is out of tensor memory: the next item's first P.V may overwrite it
              ptx::tc_fence_before();
              arrive_issuer(issuer_bar(&bars->o_free));
            }
            stage_free();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint32_t* x = &pk[i >> 2][(i & 3) * 4];
              put(i, x[0], x[1], x[2], x[3]);
            }
            store_stage(me, g, 0, (half * kHalfCols + c * 64) * 2);
          }
        }
      }
      tg += n_tiles;
      ++n_done;
    }
  }

  // ---- teardown: every thread arrives here, on success and after a failed wait ----
  if (warp < 8 && lane == 0) ptx::bulk_wait_all();   // the output boxes handed to the copy engine are stored
  ptx::tc_fence_before();
  __syncthreads();
  // CTA 0's MMAs read this CTA's shared and tensor memory: leave together
  ptx::cluster_sync_all();
  if (warp == 9) {
    ptx::tc_fence_after();
    ptx::tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------
// the parts of split items joined:  o = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i
// ---------------------------------------------------------------------------------------
// A warp takes one (item, row): few CTAs, so that a call that split nothing pays little for this launch, and every
// warp with the loads of several parts in flight.
constexpr int kJoinWarps = 16, kJoinBlocks = 296;

template <typename O, int kD>
__global__ void __launch_bounds__(kJoinWarps * 32) join_kernel(const __grid_constant__ PackedParams p) {
  wait_for_launch_before();
  const int32_t status = __ldcg(p.status);
  if ((status & 0xf00) == 0x300 && status != kErrBadPage) return;      // the parts are not complete
  const int n_rows = __ldcg(&p.header->n_joins) * kPartRows;
  const int lane = threadIdx.x & 31;
  constexpr int kVecs = kD / 128;                // float4 of a lane
  for (int u = blockIdx.x * kJoinWarps + (threadIdx.x >> 5); u < n_rows; u += kJoinBlocks * kJoinWarps) {
    const JoinEntry e = p.header->joins[u / kPartRows];
    const int row = u % kPartRows, rr = row % kBM, tok_c = rr * p.group_mul >> 16, tok = row / kBM * p.tpt + tok_c;
    if (rr >= p.tpt * p.group || tok >= e.n_tok) continue;
    auto part_of = [&](int w) { return w == e.w_lo ? e.part_lo : 2 * w; };
    float top = -INFINITY;
    for (int w = e.w_lo + lane; w <= e.w_hi; w += 32) top = fmaxf(top, p.header->part_lm[part_of(w)][row][1]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float l = 0.f;
    float4 acc[kVecs];
#pragma unroll
    for (int v = 0; v < kVecs; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int w = e.w_lo; w <= e.w_hi; ++w) {
      const int part = part_of(w);
      const float2 lm = *reinterpret_cast<const float2*>(p.header->part_lm[part][row]);
      const float f = lm.y == -INFINITY ? 0.f : ptx::ex2_approx(lm.y - top);
      l += f * lm.x;
#pragma unroll
      for (int v = 0; v < kVecs; ++v) {
        const float4 x = __ldcs(reinterpret_cast<const float4*>((const char*)p.parts + (int64_t)part * kPartBytes + (row * kD + v * 128 + lane * 4) * 4));
        acc[v].x += f * x.x; acc[v].y += f * x.y; acc[v].z += f * x.z; acc[v].w += f * x.w;
      }
    }
    const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
    for (int v = 0; v < kVecs; ++v) {
      O* dst = (O*)p.o + (int64_t)(e.row0 + tok) * p.o_row + (int64_t)(e.g * p.group + rr - tok_c * p.group) * p.o_head + v * 128 + lane * 4;
      O y[4] = {ElemTraits<O>::from_float(acc[v].x * inv), ElemTraits<O>::from_float(acc[v].y * inv), ElemTraits<O>::from_float(acc[v].z * inv),
                ElemTraits<O>::from_float(acc[v].w * inv)};
      if constexpr (sizeof(O) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(y);
      else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(y);
    }
  }
}

// ---------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------
template <typename T, int kD>
int launch_typed(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, const CUtensorMap& om, const PackedParams& p, int workers, cudaStream_t st) {
  static bool attr_set[64] = {false};
  int dev = 0;
  G4B_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64 && !attr_set[dev]) {
    // (the registers that the softmax warps take must be there, or they wait for ever)
    cudaFuncAttributes fa;
    G4B_CUDA_CHECK(cudaFuncGetAttributes(&fa, packed_prefill_kernel<T, kD>));
    if (fa.numRegs * kThreads < 256 * kRegsSoftmax + 128 * kRegsOther) return fail(G4B_ERR_CUDA, "packed attention was built with %d registers a thread", fa.numRegs);
    G4B_CUDA_CHECK(cudaFuncSetAttribute(packed_prefill_kernel<T, kD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<kD>::kSmemBytes));
    attr_set[dev] = true;
  }
  // Each launch is set up while the one before it drains (and waits for it before it reads anything).
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)((p.max_items + 7) / 8), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  G4B_CUDA_CHECK(cudaLaunchKernelEx(&cfg, plan_kernel, p));
  cfg.gridDim = dim3((unsigned)(2 * workers), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = Geo<kD>::kSmemBytes;
  cfg.numAttrs = 2;
  G4B_CUDA_CHECK(cudaLaunchKernelEx(&cfg, packed_prefill_kernel<T, kD>, qm, km, vm, om, p));
  if (!p.may_split) return G4B_OK;
  cfg.gridDim = dim3(kJoinBlocks, 1, 1);
  cfg.blockDim = dim3(kJoinWarps * 32, 1, 1);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  if (p.o_dtype == G4B_F32) G4B_CUDA_CHECK(cudaLaunchKernelEx(&cfg, join_kernel<float, kD>, p));
  else G4B_CUDA_CHECK(cudaLaunchKernelEx(&cfg, join_kernel<T, kD>, p));
  return G4B_OK;
}

int check_rank(const G4bTensor& t, const char* name, int ndim) {
  if (t.ndim != ndim) return fail(G4B_ERR_BAD_ARG, "%s: expected rank %d, got %d", name, ndim, t.ndim);
  bool empty = false;
  for (int i = 0; i < ndim; ++i) {
    if (t.shape[i] < 0) return fail(G4B_ERR_BAD_ARG, "%s: negative extent", name);
    empty |= t.shape[i] == 0;
  }
  if (t.ptr == nullptr && !empty) return fail(G4B_ERR_BAD_ARG, "%s: null pointer", name);
  return G4B_OK;
}

int64_t items_bound(int64_t rows, int64_t slots, int64_t group) {
  const int64_t block = 2 * (kBM / group);
  return rows / block + slots;       // every slot adds at most one partly filled block
}

}  // namespace

int launch_prefill_packed(const G4bPackedAttnArgs& a, cudaStream_t st) {
  int rc;
  if ((rc = check_rank(a.q, "q", 3)) || (rc = check_rank(a.o, "o", 3)) || (rc = check_rank(a.k_pool, "k_pool", 4)) ||
      (rc = check_rank(a.v_pool, "v_pool", 4)) || (rc = check_rank(a.q_starts, "q_starts", 1)) ||
      (rc = check_rank(a.time_dim_sizes, "time_dim_sizes", 1)) || (rc = check_rank(a.block_tables, "block_tables", 2)) ||
      (rc = check_rank(a.workspace, "workspace", 1))) return rc;
  const int64_t N = a.q.shape[0], H = a.q.shape[1], D = a.q.shape[2], B = a.time_dim_sizes.shape[0], G = a.k_pool.shape[1];
  for (int i = 0; i < 3; ++i)
    if (a.o.shape[i] != a.q.shape[i]) return fail(G4B_ERR_BAD_ARG, "o shape must equal q shape");
  if (a.k_pool.dtype != G4B_F16 && a.k_pool.dtype != G4B_BF16) return fail(G4B_ERR_BAD_DTYPE, "k_pool/v_pool must both be f16 or both bf16");
  if (a.v_pool.dtype != a.k_pool.dtype) return fail(G4B_ERR_BAD_DTYPE, "k_pool/v_pool must both be f16 or both bf16");
  if (a.q.dtype != a.k_pool.dtype) return fail(G4B_ERR_BAD_DTYPE, "q must have the pools' dtype");
  if (a.o.dtype != a.k_pool.dtype && a.o.dtype != G4B_F32) return fail(G4B_ERR_BAD_DTYPE, "o must have the pools' dtype or be f32");
  for (int i = 0; i < 4; ++i)
    if (a.k_pool.shape[i] != a.v_pool.shape[i]) return fail(G4B_ERR_BAD_ARG, "k_pool/v_pool shapes differ");
  if (!contiguous_from(a.k_pool, 0) || !contiguous_from(a.v_pool, 0)) return fail(G4B_ERR_BAD_STRIDE, "k_pool/v_pool must be contiguous");
  if (a.k_pool.shape[3] != D) return fail(G4B_ERR_BAD_ARG, "head dim of q and pools differ");
  if (D != 256 && D != 128) return fail(G4B_ERR_UNSUPPORTED, "head dim %lld not supported (128, 256)", (long long)D);
  if (G <= 0 || H <= 0 || H % G != 0) return fail(G4B_ERR_BAD_ARG, "query heads must be a multiple of kv heads");
  if (G > 0x7fff) return fail(G4B_ERR_UNSUPPORTED, "at most 32767 kv heads");
  if (H / G > kBM) return fail(G4B_ERR_UNSUPPORTED, "at most %d query heads per kv head", kBM);
  if (a.page_size < 16 || (a.page_size & (a.page_size - 1)) != 0) return fail(G4B_ERR_BAD_ARG, "page_size must be a power of two >= 16");
  if (a.k_pool.shape[2] != a.page_size) return fail(G4B_ERR_BAD_ARG, "pool dim 2 must equal page_size");
  if (a.q_starts.dtype != G4B_I32 || a.time_dim_sizes.dtype != G4B_I32 || a.block_tables.dtype != G4B_I32)
    return fail(G4B_ERR_BAD_DTYPE, "q_starts, time_dim_sizes and block_tables must be int32");
  if (a.q_starts.shape[0] != B + 1 || a.block_tables.shape[0] != B)
    return fail(G4B_ERR_BAD_ARG, "q_starts must have B + 1 entries and block_tables B rows");
  if (a.stage != G4B_STAGE_CAUSAL && a.stage != G4B_STAGE_FULL) return fail(G4B_ERR_BAD_ARG, "stage must be STAGE_FULL (1) or STAGE_CAUSAL (3)");
  if (a.sliding_window < 0) return fail(G4B_ERR_BAD_ARG, "sliding_window must be >= 0");
  if (!(a.scale > 0.f) || !(a.scale < 1e30f)) return fail(G4B_ERR_BAD_ARG, "scale must be positive and finite");
  const G4bTensor* rows[2] = {&a.q, &a.o};
  for (int k = 0; k < 2; ++k) {
    const G4bTensor& t = *rows[k];
    const char* nm = k == 0 ? "q" : "o";
    if (t.stride[2] != 1) return fail(G4B_ERR_BAD_STRIDE, "%s: innermost stride must be 1", nm);
    for (int i = 0; i < 2; ++i)
      if (t.shape[i] > 1 && (t.stride[i] <= 0 || (t.stride[i] * dtype_size(t.dtype)) % 16 != 0))
        return fail(G4B_ERR_BAD_STRIDE, "%s: strides must be positive multiples of 16 bytes", nm);
  }
  if (rows_overlap(a.o)) return fail(G4B_ERR_BAD_STRIDE, "o: rows that are written must not overlap");
  if ((((uintptr_t)a.q.ptr) | ((uintptr_t)a.o.ptr) | ((uintptr_t)a.k_pool.ptr) | ((uintptr_t)a.v_pool.ptr)) & 15)
    return fail(G4B_ERR_BAD_STRIDE, "q, o and the pools must be 16-byte aligned");
  if (a.workspace.stride[0] != 1 && a.workspace.shape[0] > 1) return fail(G4B_ERR_BAD_STRIDE, "workspace must be contiguous");
  const int64_t need = g4b_packed_workspace_bytes(N, B, (int)H, (int)G);
  if (a.workspace.shape[0] * dtype_size(a.workspace.dtype) < need)
    return fail(G4B_ERR_BAD_ARG, "workspace: %lld bytes needed (g4b_packed_workspace_bytes)", (long long)need);
  if (((uintptr_t)a.workspace.ptr) & 15) return fail(G4B_ERR_BAD_STRIDE, "workspace must be 16-byte aligned");
  const int64_t max_items = items_bound(N, B, H / G);
  if (N > 0x3fffffffLL || max_items * G > 0x3fffffffLL || a.k_pool.shape[0] >= 0x7fffffffLL || a.block_tables.shape[1] > 0x7fffffffLL)
    return fail(G4B_ERR_TOO_LARGE, "rows, items and pages are counted in 30 bits");
  G4B_STOP_IF_VALIDATE_ONLY();
  if (N == 0 || B == 0) return G4B_OK;
  if (a.k_pool.shape[0] == 0) return fail(G4B_ERR_BAD_ARG, "the pools hold no page");

  PackedParams p{};
  p.o = a.o.ptr;
  p.q_starts = (const int32_t*)a.q_starts.ptr; p.starts_s = a.q_starts.stride[0];
  p.times = (const int32_t*)a.time_dim_sizes.ptr; p.time_s = a.time_dim_sizes.stride[0];
  p.block_tables = (const int32_t*)a.block_tables.ptr;
  p.bt_s0 = a.block_tables.stride[0]; p.bt_s1 = a.block_tables.stride[1];
  p.header = (PackedHeader*)a.workspace.ptr;
  p.parts = (float*)((char*)a.workspace.ptr + kPartsAt);
  p.items = (PackedItem*)((char*)a.workspace.ptr + kItemsAt);
  p.o_row = a.o.stride[0]; p.o_head = a.o.stride[1];
  p.N = (int)N; p.B = (int)B; p.H = (int)H; p.G = (int)G;
  p.group = (int)(H / G); p.tpt = kBM / p.group;
  p.group_mul = (65536 + p.group - 1) / p.group;
  p.max_items = (int)max_items;
  while ((1 << p.page_shift) < a.page_size) ++p.page_shift;
  p.num_pages = (int)a.k_pool.shape[0]; p.max_pages = (int)a.block_tables.shape[1];
  p.k_rows = a.page_size < 64 ? a.page_size : 64;
  p.v_rows = a.page_size < kBN ? a.page_size : kBN;
  p.sliding_window = a.sliding_window < (1 << 30) ? a.sliding_window : 1 << 30;    // (no context is longer; sums stay in 32 bits)
  p.causal = a.stage == G4B_STAGE_CAUSAL; p.o_dtype = a.o.dtype;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.status = device_status_ptr();
  if (p.status == nullptr) return G4B_ERR_CUDA;

  const uint64_t esz = 2;
  CUtensorMap qm, km, vm;
  {
    // (extents of 1 may come with any stride; the descriptor wants a valid one)
    const uint64_t head = H > 1 ? (uint64_t)a.q.stride[1] * esz : (uint64_t)D * esz;
    const uint64_t row = N > 1 ? (uint64_t)a.q.stride[0] * esz : (uint64_t)(H * D) * esz;
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)H, (uint64_t)N};
    const uint64_t strides[2] = {head, row};
    const uint32_t box[3] = {64, (uint32_t)p.group, (uint32_t)p.tpt};
    if ((rc = encode_map(&qm, a.q.dtype, 3, a.q.ptr, dims, strides, box, "q"))) return rc;
    const uint64_t P = (uint64_t)a.page_size;
    const uint64_t pdims[4] = {(uint64_t)D, P, (uint64_t)G, (uint64_t)p.num_pages};
    const uint64_t pstr[3] = {(uint64_t)D * esz, P * D * esz, (uint64_t)G * P * D * esz};
    const uint32_t kbox[4] = {64, (uint32_t)p.k_rows, 1, 1};
    // V with the head dim as slabs of 64: a box is the rows of a group and a CTA's slabs
    const uint64_t vdims[5] = {64, P, (uint64_t)D / 64, (uint64_t)G, (uint64_t)p.num_pages};
    const uint64_t vstr[4] = {(uint64_t)D * esz, 128, P * D * esz, (uint64_t)G * P * D * esz};
    const uint32_t vbox[5] = {64, (uint32_t)p.v_rows, (uint32_t)(D / 128), 1, 1};
    if ((rc = encode_map(&km, a.k_pool.dtype, 4, a.k_pool.ptr, pdims, pstr, kbox, "k_pool"))) return rc;
    if ((rc = encode_map(&vm, a.v_pool.dtype, 5, a.v_pool.ptr, vdims, vstr, vbox, "v_pool"))) return rc;
  }
  // The output as boxes of the 32 rows that a warp holds: 32 / (heads of a group) tokens, or 32 heads of one.  Other
  // group sizes, f32, and layouts that a descriptor cannot express (the driver refuses it) are stored by the warps.
  CUtensorMap om = qm;
  if ((p.group & (p.group - 1)) == 0 && a.o.dtype != G4B_F32) {
    const uint64_t head = H > 1 ? (uint64_t)a.o.stride[1] * esz : (uint64_t)D * esz;
    const uint64_t row = N > 1 ? (uint64_t)a.o.stride[0] * esz : (uint64_t)(H * D) * esz;
    const uint64_t dims[3] = {(uint64_t)D, (uint64_t)H, (uint64_t)N};
    const uint64_t strides[2] = {head, row};
    const uint32_t gw = p.group < 32 ? (uint32_t)p.group : 32u;
    const uint32_t box[3] = {64, gw, 32 / gw};
    p.o_boxes = encode_map(&om, a.o.dtype, 3, a.o.ptr, dims, strides, box, "o") == G4B_OK;
    if (!p.o_boxes) om = qm;
  }
  static int sm_count[64] = {0};
  int dev = 0;
  G4B_CUDA_CHECK(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64) return fail(G4B_ERR_CUDA, "device index out of range");
  if (sm_count[dev] == 0) G4B_CUDA_CHECK(cudaDeviceGetAttribute(&sm_count[dev], cudaDevAttrMultiProcessorCount, dev));
  int64_t workers = sm_count[dev] / 2;
  if (workers > kMaxWorkers) workers = kMaxWorkers;
  if (workers < 1) workers = 1;
  // Shares pay only where items are few (with six a worker the list of whole ones is balanced) and contexts
  // can be long; what the contexts really are is looked at on the device.  Nor without any of that a third launch.  The bound
  // is loose: a small step over a manager's wide table has the third launch too, which then finds nothing to join (three
  // prompts of 62 rows: 13.2 us with a table of three pages, 15.7 us with one of 2048 columns).
  p.may_split = (N / (2 * p.tpt)) * G < 6 * workers && (int64_t)p.max_pages * a.page_size > 8 * kBN;
  if (!p.may_split && workers > max_items * G) workers = max_items * G;
  p.workers = (int)workers;
  if (a.k_pool.dtype == G4B_BF16)
    return D == 256 ? launch_typed<__nv_bfloat16, 256>(qm, km, vm, om, p, (int)workers, st) : launch_typed<__nv_bfloat16, 128>(qm, km, vm, om, p, (int)workers, st);
  return D == 256 ? launch_typed<__half, 256>(qm, km, vm, om, p, (int)workers, st) : launch_typed<__half, 128>(qm, km, vm, om, p, (int)workers, st);
}

}  // namespace g4b

extern "C" int64_t g4b_packed_workspace_bytes(int64_t rows, int64_t slots, int q_heads, int kv_heads) {
  if (rows < 0 || slots < 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > g4b::kBM) return 0;
  // (every worker's boundary may add an entry)
  return g4b::kItemsAt + (int64_t)sizeof(g4b::PackedItem) * (g4b::items_bound(rows, slots, q_heads / kv_heads) * kv_heads + 2 * g4b::kMaxWorkers);
}

extern "C" int g4b_flash_attention_packed(const G4bPackedAttnArgs* args, void* cuda_stream) {
  if (args == nullptr) return g4b::fail(G4B_ERR_BAD_ARG, "args is null");
  return g4b::launch_prefill_packed(*args, (cudaStream_t)cuda_stream);
}
