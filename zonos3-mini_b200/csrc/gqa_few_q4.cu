// Attention of few rows over a paged KV cache in 4 bits (kv_q4.cuh): the single tokens, and short drafts of them, of a decode
// batch. The mathematics is that of gqa_chunk.cu; requests of more rows are its kernel's.
//
// The rows of a request's score matrix for one KV head are its (token, head of the group) pairs, up to 8 (NT = 1) or 16. A row
// reads every code once, so the work is the codes' way from HBM and their unpacking; the products are few. So they are
// formed from registers (m16n8k16: 16 keys or dims by 8 rows), where a code goes from the loaded word into a matrix fragment
// with two instructions for two codes, and nothing is written out in between as a tensor-memory product would need it:
//   scores^T [16 keys, 8 rows] = sum over groups g of  s_g ((128 + c) . q)_g + (m_g - 128 s_g) (sum q)_g:  the codes themselves are
//     the operand, as 128 + c in bf16 (exact), s goes onto the products' sums in fp32; the second term is a product of its own, the
//     pairs as they lie in the cache times the queries' sums, split into three bf16 each: the scores have the precision of fp32;
//   out^T [16 dims, 8 rows] += V^T p^T with V = m + s c and the weights in fp16, 2^-12 of each: bf16's 2^-9 would be the largest
//     error here. fp16 has less range, so a block whose pairs are not all within it (magnitudes of 2^-10 to 2^14, or 0) takes bf16.
// A weight is 2^(score - m + 15) with m a row's reference, its largest score or up to 8 (log2) above it when it is set; it is set
// anew by a score above it, hardly ever after the first block. So weights lie in fp16's range: up to 2^15, the largest not below 2^7
// when m is set, and those below 2^-39 of m count as 0. m and the sum cancel in the end.
// The keys of a 16-key block stand in the scores' rows in the order 0 1 3 2 4 5 7 6 and 8 on: the two rows of a quarter of the lanes then
// read other banks, and the four rows that a lane's values come from too, as far as 64-byte rows allow.
//
// Every warp works for itself. All units' keys are one long run of items (two blocks of 16 keys, at hd 128 2560 bytes
// each), of which a warp takes an equal share (the split is as in gqa_chunk.cu, to warps instead of CTAs): it looks up the places of
// its blocks, has the copies of the next item under way while it computes one, and keeps m, the sum and the accumulator of a unit in
// its registers, where a lane has 8 consecutive elements of up to four rows' outputs. A unit that spans warps leaves a part of each
// in the workspace; the warp that finishes the last of up to 16 neighbouring parts joins them in the order of their keys, and so on
// for the joined ones. No warp waits for another, and results do not depend on timing.
//
// Measured ways that were slower (256 tokens of 16 / 4 heads of 128 over 1628 keys): seven warps a CTA that share a unit's items, an eighth
// that starts the copies, the accumulators joined in shared memory: 105-112 us. Each warp waited for copies and at every
// unit's end for the slowest; half of the cycles issued nothing.
#include <algorithm>

#include "few_q4.cuh"

namespace {

namespace q4 = zb::q4;

constexpr int kItem = 2;      // blocks of an item
constexpr int kUnitCost = 1;  // of a unit, in items
constexpr int kMinShare = 3;  // items of a warp, its units' cost among them
constexpr int kJoin = 16;     // parts that are joined at once
constexpr float kAbove = 8.f, kShift = 15.f;
constexpr float kNone = -3.0e38f;  // m of a row that has seen no key

struct FewParams {
  q4::FewCall c;
  int G, workers;
  unsigned page_mul, page_shift;  // division by the page size
  // [warp][2]: the call's tag and, below it, the parts that have arrived of those that are joined with one of the warp's (the first
  // of them; [0]: of the unit that began there, [1]: of one that had begun before); 0 again when all have. What a call whose waits
  // gave up has left has another tag.
  unsigned* counters;
  unsigned tag;
  float* acc;  // [warp][2][rows][hd]: parts
  float* ml;   // [warp][2][2][rows]: m, sum
  unsigned* status;
};

// What a warp does with one unit.
struct Desc {
  int token0, pos0, keys;  // first token row, its key position, keys of the request
  int rows, kvh;
  int items;
  int index, parts, first;  // of the unit's parts this one, their number, and the warp that has the first
  int from;                 // keys from the sinks' end to here are hidden from every row
  int all_lo, all_hi;       // keys of [all_lo, all_hi), and those below min(sinks, all_hi), are seen by every row
};
// Where a block lies; its first key, and how many of its keys there are.
struct Place {
  const unsigned char* at;
  int key0, exist;
};
// A warp's own shared memory, behind its stages and queries.
struct Own {
  alignas(16) int2 info[2][kItem];  // of the stages' blocks: first key, and how many there are
  alignas(16) Place places[32];
  Desc desc[2];
  // the unit after those opened: how far its request and the share have got
  int64_t at;
  int b, kvh, off;
  int row0, tokens, keys;
  // of the unit opened last: blocks whose places are not looked up yet, and what that takes
  int next, end, n, sink_blocks, gap, of_b, of_kvh, held;
};

template <int GROUPS, int NT>
struct Shape {
  static constexpr int kHd = GROUPS * q4::kGroup, kBlockBytes = q4::block_bytes(kHd), kRows = 8 * NT;
  static constexpr int kStage = kItem * kBlockBytes;
  static constexpr int kOffQ = 2 * kStage;
  static constexpr int kOffPairs = kOffQ + kRows * kHd * 2;  // pairs of values, as the lanes need them
  static constexpr int kOffOwn = kOffPairs + kItem * GROUPS * 64;
  static constexpr int kPerWarp = (kOffOwn + (int)sizeof(Own) + 127) / 128 * 128;
  // 16 warps an SM have 128 registers a thread; with 16 rows the accumulators alone are 64, so 12 have 168
  static constexpr int kWarps = NT == 1 ? 8 : 6, kCtas = 2, kThreads = 32 * kWarps;
  // The queries' fragments stay in registers, or are read again for every block where the accumulators take those.
  static constexpr bool kKeep = NT == 1;
};
struct Tail {
  int sums[2][8];
  int before[256], cost[256];
  int idle[2];
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// D += A B
template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// D = A B of bf16
__device__ __forceinline__ void mma_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <bool HALF>
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  if constexpr (HALF) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float low_of(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float high_of(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// Whether fp16 keeps m + s c of a pair to near its 11 bits: |m| is below 2^14 and s below 2^10, and either |m| is 2^-10 or more or
// s 2^-14, or the pair is 0.
__device__ __forceinline__ bool half_holds(uint32_t pair) {
  const uint32_t a = pair & 0x7fff7fffu;
  const uint32_t over = a + (((0x8000u - 0x4680u) << 16) | (0x8000u - 0x4480u));
  const uint32_t under = a + (((0x8000u - 0x3a80u) << 16) | (0x8000u - 0x3880u));
  return (over & 0x80008000u) == 0 && ((under & 0x80008000u) != 0 || a == 0);
}

// (x & mask) | bits, in one instruction.
__device__ __forceinline__ uint32_t masked_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(mask), "r"(bits));
  return d;
}
// 16 bytes into shared memory, asynchronously and for this thread's next commit.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() {  // all but the last N groups of this thread
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// A request's new rows (none where they are another kernel's) and its blocks of keys, which are taken two at a time. Blocks from sink_blocks on are counted
// without the `gap` blocks between the first keys and the windows.
struct Request {
  int row0, tokens, keys;
};
__device__ __forceinline__ Request request(const FewParams& p, int b, bool& more) {
  Request r;
  r.row0 = min(max(p.c.kv.cu[b], 0), p.c.kv.N);
  r.tokens = min(max(p.c.kv.cu[b + 1], r.row0), p.c.kv.N) - r.row0;
  r.keys = max(p.c.kv.keys[b], 0);
  if ((int64_t)r.tokens * p.G > p.c.rows) {
    more = true;
    r.tokens = 0;
  }
  return r;
}
struct Blocks {
  int n, sink_blocks, gap;
  int lo_first, lo_last, hi_first;
};
__device__ __forceinline__ int held_keys(const FewParams& p, int keys) { return min(keys, p.c.kv.max_pages * p.c.kv.page_size); }
__device__ __forceinline__ int first_seen(const FewParams& p, int pos) {  // of a token's window
  const int lo = p.c.window > 0 ? (int)max((int64_t)0, (int64_t)pos + 1 - p.c.window) : 0;
  return lo <= p.c.sinks ? 0 : lo;
}
__device__ __forceinline__ int behind_seen(const FewParams& p, int held, int pos) {
  return max(p.c.causal ? min(held, pos + 1) : held, 0);
}
__device__ __forceinline__ Blocks blocks_of(const FewParams& p, const Request& r) {
  const int held = held_keys(p, r.keys), pos0 = r.keys - r.tokens;
  const int lo = first_seen(p, pos0), hi = behind_seen(p, held, pos0 + r.tokens - 1);
  Blocks x;
  x.lo_first = lo;
  x.lo_last = first_seen(p, pos0 + r.tokens - 1);
  x.hi_first = behind_seen(p, held, pos0);
  const int begin = lo / q4::kBlock;
  x.n = hi > lo ? (hi + q4::kBlock - 1) / q4::kBlock - begin : 0;
  x.sink_blocks = 0;
  x.gap = begin;
  const int sinks = min(p.c.sinks, hi);
  if (lo > 0 && sinks > 0) {
    x.sink_blocks = min((sinks + q4::kBlock - 1) / q4::kBlock, begin);
    x.gap = begin - x.sink_blocks;
    x.n += x.sink_blocks;
  }
  return x;
}

__device__ __forceinline__ int cost_of(const FewParams& p, const Request& r) {
  return r.tokens > 0 ? kUnitCost + (blocks_of(p, r).n + kItem - 1) / kItem : 0;
}

// Exclusive prefix of v over the block's threads; `total` the sum. `buffer` alternates from call to call.
template <int WARPS>
__device__ __forceinline__ int block_scan(int v, Tail& tl, int buffer, int& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int in = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int u = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += u;
  }
  if (lane == 31) tl.sums[buffer][warp] = in;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int s = tl.sums[buffer][w];
    if (w < warp) before += s;
    total += s;
  }
  return before + in - v;
}

__device__ __forceinline__ float sigmoid(__nv_bfloat16 x) { return 1.f / (1.f + ex2(-1.4426950408889634f * __bfloat162float(x))); }

// Part `index` of a unit whose first part is warp `first`'s: the slots are its own second one, then the first ones of those after it.
__device__ __forceinline__ int64_t part_slot(int first, int index) { return (int64_t)(first + index) * 2 + (index == 0); }

template <int GROUPS, int NT>
__global__ void __launch_bounds__(Shape<GROUPS, NT>::kThreads, Shape<GROUPS, NT>::kCtas)
    gqa_few_q4_kernel(const __grid_constant__ FewParams p) {
  using L = Shape<GROUPS, NT>;
  constexpr int hd = L::kHd, kWarps = L::kWarps, kThreads = L::kThreads;
  extern __shared__ __align__(128) unsigned char gbase[];
  Tail& tl = *reinterpret_cast<Tail*>(gbase + kWarps * L::kPerWarp);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid % 32;
  unsigned char* own = gbase + warp * L::kPerWarp;
  Own& my = *reinterpret_cast<Own*>(own + L::kOffOwn);
  const int B = p.c.kv.B, Hkv = p.c.kv.Hkv;
  const int worker = warp * gridDim.x + blockIdx.x;  // few of them are spread over the SMs
  zb::pdl_enter();

  // ---- the plan: the work of all units, and where this warp's begins
  bool more = false, out_of_order = false;
  const Request mine = tid < B ? request(p, tid, more) : Request{0, 0, 0};
  const int mine_cost = cost_of(p, mine);
  if (tid == 0) {
    tl.idle[0] = min(max(p.c.kv.cu[0], 0), p.c.kv.N);
    tl.idle[1] = min(max(p.c.kv.cu[B], tl.idle[0]), p.c.kv.N);
  }
  int64_t work = 0;
  int buffer = 0, mine_before = 0, mine_total = 0;
#pragma unroll 1
  for (int b0 = 0; b0 < B; b0 += kThreads, buffer ^= 1) {
    const int b = b0 + tid;
    if (b < B) out_of_order |= p.c.kv.cu[b + 1] < p.c.kv.cu[b] || p.c.kv.cu[b] < 0 || p.c.kv.cu[b + 1] > p.c.kv.N;
    const int cost = b0 == 0 ? mine_cost : b < B ? cost_of(p, request(p, b, more)) : 0;
    int total;
    const int before = block_scan<kWarps>(cost, tl, buffer, total);
    if (b0 == 0) {
      mine_before = before;
      mine_total = total;
    }
    work += total;
  }
  const bool refused = __syncthreads_or(out_of_order);
  const bool left_out = __syncthreads_or(more) && p.c.only;
  if (worker == 0 && lane == 0 && p.status && (refused || left_out))
    atomicOr(p.status, refused ? zb::kStatusAttnChunkBatch : zb::kStatusAttnFewRows);
  work = refused ? 0 : work * Hkv;
  const int64_t share = max((int64_t)kMinShare, (work + p.workers - 1) / p.workers);
  const int64_t begin = share * worker, end = min(work, begin + share);
  {
    int64_t seen = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < B; b0 += kThreads) {
      int cost = mine_cost, before = mine_before, total = mine_total;
      if (b0 > 0) {
        cost = b0 + tid < B ? cost_of(p, request(p, b0 + tid, more)) : 0;
        buffer ^= 1;
        before = block_scan<kWarps>(cost, tl, buffer, total);
      }
      if (work > 0) {
        tl.before[tid] = before;
        tl.cost[tid] = cost;
      }
      __syncthreads();
      if (begin < end && begin >= seen * Hkv && begin < (seen + total) * Hkv) {
#pragma unroll 1
        for (int i = lane; i < kThreads; i += 32) {
          const int64_t at = (seen + tl.before[i]) * Hkv;
          if (tl.cost[i] > 0 && begin >= at && begin < at + (int64_t)tl.cost[i] * Hkv) {
            bool ignored = false;
            const Request r = request(p, b0 + i, ignored);
            my.at = begin;
            my.b = b0 + i;
            my.kvh = (int)((begin - at) / tl.cost[i]);
            my.off = (int)((begin - at) % tl.cost[i]);
            my.row0 = r.row0;
            my.tokens = r.tokens;
            my.keys = r.keys;
          }
        }
      }
      seen += total;
      __syncthreads();
    }
  }
  if (begin < end) {
    const int gid = lane / 4, t4 = lane % 4;
    const int key_row = gid ^ ((gid >> 1) & 1);             // the key of scores' row gid; 8 more for row gid + 8
    const int va = 2 * t4 + (t4 & 1), vb = va ^ 1;  // the keys of rows 2 t4 and 2 t4 + 1
    int opened = 0, done = 0;      // units
    int fetched = 0, computed = 0;  // items
    int place = 0, places = 0;      // the next of the places looked up, and their number
    bool loaded = false, more_units = true;  // the queries of unit `done` have been taken from shared memory

    // Opens the next unit of which items lie in the share: its description, and its queries' copy.
    auto open_unit = [&]() {
      __syncwarp();
      int64_t at = my.at;
      int b = my.b, kvh = my.kvh, off = my.off;
      Request req{my.row0, my.tokens, my.keys};
      bool found = false;
      __syncwarp();
#pragma unroll 1
      while (!found && at < end) {
        const Blocks x = blocks_of(p, req);
        const int unit_items = (x.n + kItem - 1) / kItem, cost = kUnitCost + unit_items;
        const int to_cost = (int)min((int64_t)cost, off + (end - at));
        const int from = max(off - kUnitCost, 0), to = max(to_cost - kUnitCost, 0);
        if (to > from || (x.n == 0 && off == 0)) {
          found = true;
          const int64_t first = at - off + kUnitCost;  // of the unit's items
          if (lane == 0) {
            Desc d;
            d.token0 = req.row0;
            d.pos0 = req.keys - req.tokens;
            d.keys = req.keys;
            d.rows = req.tokens * p.G;
            d.kvh = kvh;
            d.items = to - from;
            d.first = x.n > 0 ? (int)(first / share) : worker;
            d.index = worker - d.first;
            d.parts = x.n > 0 ? (int)((first + unit_items - 1) / share) - d.first + 1 : 1;
            d.from = x.lo_first;
            d.all_lo = x.lo_last;
            d.all_hi = x.hi_first;
            my.desc[opened % 2] = d;
            my.next = from * kItem;
            my.end = to * kItem;
            my.n = x.n;
            my.sink_blocks = x.sink_blocks;
            my.gap = x.gap;
            my.of_b = b;
            my.of_kvh = kvh;
            my.held = held_keys(p, req.keys);
          }
          // the queries, with the copies of the unit's first item: a token's heads of the group lie side by side
          const int pieces = p.G * (hd / 8);
#pragma unroll 1
          for (int i = lane; i < (to > from ? req.tokens * pieces : 0); i += 32)
            copy16(zb::smem_addr(own + L::kOffQ) + i * 16,
                   p.c.q + (int64_t)(req.row0 + i / pieces) * p.c.q_stride + (int64_t)kvh * p.G * hd + i % pieces * 8);
        }
        // the next unit: KV head, then request
        at += to_cost - off;
        off = 0;
        if (at < end && ++kvh == Hkv) {
          kvh = 0;
          req.tokens = 0;
#pragma unroll 1
          for (++b; b < B; b += 32) {  // 32 requests at a time
            bool ignored = false;
            const Request r = b + lane < B ? request(p, b + lane, ignored) : Request{0, 0, 0};
            const unsigned have = __ballot_sync(0xffffffffu, r.tokens > 0);
            if (have == 0) continue;
            const int k = __ffs(have) - 1;
            b += k;
            req.row0 = __shfl_sync(0xffffffffu, r.row0, k);
            req.tokens = __shfl_sync(0xffffffffu, r.tokens, k);
            req.keys = __shfl_sync(0xffffffffu, r.keys, k);
            break;
          }
          if (req.tokens == 0) at = end;  // not while the lengths stay as they were when the work was added up
        }
      }
      if (lane == 0) {
        my.at = at;
        my.b = b;
        my.kvh = kvh;
        my.off = off;
        my.row0 = req.row0;
        my.tokens = req.tokens;
        my.keys = req.keys;
      }
      __syncwarp();
      place = places = 0;
      opened += found;
      more_units = found;
    };
    // Starts the copies of the next item. Those of a unit after the one that is computed wait until its queries are in registers,
    // which makes room for theirs.
    auto fetch = [&]() {
#pragma unroll 1
      while (place == places) {
        const int next = my.next, stop = my.end;
        if (opened > done && next < stop) {  // a lane's block
          const int j = next + lane, block = j < my.sink_blocks ? j : j + my.gap, key0 = block * q4::kBlock;
          const int column = (int)(((uint64_t)(unsigned)key0 * p.page_mul) >> p.page_shift);
          const int page = j < min(stop, my.n) && key0 < my.held ? p.c.kv.table[(int64_t)my.of_b * p.c.kv.table_stride + column] : -1;
          const bool there = page >= 0 && page < p.c.kv.num_pages;
          Place found;
          found.at = reinterpret_cast<const unsigned char*>(p.c.kv.k) + (there ? (int64_t)page * p.c.kv.page_stride : 0) +
                     (int64_t)my.of_kvh * p.c.kv.head_stride + (int64_t)(key0 - column * p.c.kv.page_size) / q4::kBlock * L::kBlockBytes;
          found.key0 = key0;
          found.exist = there ? min(q4::kBlock, my.held - key0) : 0;
          __syncwarp();
          my.places[lane] = found;
          place = 0;
          places = min(32, stop - next);
          if (lane == 0) my.next = next + places;
          __syncwarp();
        } else {
          if (!more_units || opened - done > 1 || (opened - done == 1 && !(L::kKeep && loaded))) return;
          open_unit();
        }
      }
      const int stage = fetched % 2;
#pragma unroll
      for (int x = 0; x < kItem; ++x) {
        const Place found = my.places[place + x];
        const uint32_t to = zb::smem_addr(own + stage * L::kStage + x * L::kBlockBytes) + lane * 16;
        if (lane == 0) my.info[stage][x] = make_int2(found.key0, found.exist);
        if (found.exist > 0)
#pragma unroll
          for (int i = 0; i < L::kBlockBytes; i += 512)
            if (i + 512 <= L::kBlockBytes || lane * 16 < L::kBlockBytes - i) copy16(to + i, found.at + i + lane * 16);
      }
      commit_copies();
      place += kItem;
      ++fetched;
    };
    // Masks that the compiler does not see through stay in registers, and a code takes one instruction with the constant it is
    // joined to; with both as immediates it takes two.
    uint32_t low4 = 0x000f000fu, high4 = 0x00f000f0u;
    asm("" : "+r"(low4), "+r"(high4));

    fetch();
    fetch();
#pragma unroll 1
    while (true) {
      if (opened == done) open_unit();
      if (opened == done) break;
      const Desc d = my.desc[done % 2];
      // The copies of the item to be computed, and with them those of its unit's queries.
      auto arrived = [&]() {
        if (fetched - computed > 1) wait_copies<1>();
        else wait_copies<0>();
        __syncwarp();
      };
      if (fetched == computed) fetch();
      arrived();
      // ---- queries: B fragments; and of what a group's pair multiplies, -128 and 1 times the sum of its elements of the query, as
      // three bf16 each: (c . q) comes with 128 instead of 0 for every code's zero
      const unsigned char* q_rows = own + L::kOffQ;
      auto fragment = [&](int nt, int g) {
        return 8 * nt + gid < d.rows ? *reinterpret_cast<const uint4*>(q_rows + (8 * nt + gid) * hd * 2 + (32 * g + 8 * t4) * 2)
                                     : make_uint4(0, 0, 0, 0);
      };
      uint4 q[L::kKeep ? GROUPS : 1];
      uint32_t qs[NT][3];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float of_group = 0.f;  // t4
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const uint4 w = fragment(nt, g);
          float sum = low_of(w.x) + high_of(w.x) + (low_of(w.y) + high_of(w.y)) + (low_of(w.z) + high_of(w.z)) + (low_of(w.w) + high_of(w.w));
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if (g == t4) of_group = sum;
          if (L::kKeep) q[g] = w;
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const float kept = zb::bf16_round(of_group);
          qs[nt][i] = pack<false>(-128.f * kept, kept);
          of_group -= kept;
        }
      }
      __syncwarp();
      loaded = true;
      float m[NT][2], l[NT][2], o[NT][2 * GROUPS][4];  // of rows 2 t4 and 2 t4 + 1 (and 8 on)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = kNone;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * GROUPS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      }
      uint32_t* pairs_out = reinterpret_cast<uint32_t*>(own + L::kOffPairs);
#pragma unroll 1
      for (int item = 0; item < d.items; ++item) {
        while (fetched - computed < 2) {
          const int before = fetched;
          fetch();
          if (fetched == before) break;
        }
        const int stage = computed % 2;
        arrived();
        const int4 info = *reinterpret_cast<const int4*>(my.info[stage]);
        unsigned char* blocks = own + stage * L::kStage;
        auto k_pairs = [&](int x) { return reinterpret_cast<uint32_t*>(blocks + x * L::kBlockBytes + 16 * hd); };
        auto v_pairs = [&](int x) { return reinterpret_cast<uint32_t*>(blocks + x * L::kBlockBytes + 18 * hd); };
        // keys that some rows do not see
        bool partly = false;
#pragma unroll
        for (int x = 0; x < kItem; ++x) {
          const int key0 = x ? info.z : info.x, exist = x ? info.w : info.y;
          partly |= exist < q4::kBlock || key0 + q4::kBlock > d.all_hi || (key0 < d.all_lo && key0 + q4::kBlock > p.c.sinks);
        }
        if (partly) {  // rows that are no keys hold anything, and what no row sees shall not choose the values' type either
          for (int i = lane; i < kItem * 16 * GROUPS; i += 32) {
            const int x = i / (16 * GROUPS), j = i / GROUPS % 16, key = (x ? info.z : info.x) + j;
            if (j >= (x ? info.w : info.y) || (key >= p.c.sinks && key < d.from))
              k_pairs(x)[i % (16 * GROUPS)] = v_pairs(x)[i % (16 * GROUPS)] = 0;
          }
          __syncwarp();
        }
        // Pairs: none of the keys' may count as one that is not finite; the values' go to where the lanes that need them read
        // them, two keys' s and m beside each other.
        bool half = true;
        {
          const int g = lane / 8 % GROUPS, t = lane % 4, h = lane / 4 % 2;  // a group, and the keys of scores' rows 2 t + 8 h, + 1
          const int row = 2 * t + (t & 1) + 8 * h;
          bool k_none = false;
          uint32_t a[kItem], b[kItem];
#pragma unroll
          for (int x = 0; x < kItem; ++x) {
            const uint2 k2 = GROUPS == 4 ? reinterpret_cast<const uint2*>(k_pairs(x))[lane] : make_uint2(k_pairs(x)[lane], 0);
            k_none |= q4::pair_is_none(k2.x) || q4::pair_is_none(k2.y);
            a[x] = v_pairs(x)[row * GROUPS + g];
            b[x] = v_pairs(x)[(row ^ 1) * GROUPS + g];
            half &= half_holds(a[x]) && half_holds(b[x]);
          }
          half = __all_sync(0xffffffffu, half);
#pragma unroll
          for (int x = 0; x < kItem; ++x) {
            uint2 w;
            if (half) {
              w = make_uint2(pack<true>(low_of(a[x]), low_of(b[x])), pack<true>(high_of(a[x]), high_of(b[x])));
            } else {
              if (q4::pair_is_none(a[x])) a[x] = 0;
              if (q4::pair_is_none(b[x])) b[x] = 0;
              w = make_uint2(__byte_perm(a[x], b[x], 0x5410), __byte_perm(a[x], b[x], 0x7632));
            }
            if (lane < 8 * GROUPS) *reinterpret_cast<uint2*>(pairs_out + ((x * GROUPS + g) * 4 + t) * 4 + 2 * h) = w;
          }
          if (__any_sync(0xffffffffu, k_none)) {
#pragma unroll
            for (int x = 0; x < kItem; ++x)
              for (int i = lane; i < 16 * GROUPS; i += 32)
                if (q4::pair_is_none(k_pairs(x)[i])) k_pairs(x)[i] = 0;
            }
          __syncwarp();
        }
        auto body = [&](auto type) {
          constexpr bool HALF = decltype(type)::value;
          // ---- scores
          float s[kItem][NT][4];
#pragma unroll
          for (int x = 0; x < kItem; ++x) {
            uint32_t w[2][GROUPS], pr[2][GROUPS], mine[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const unsigned char* from = blocks + x * L::kBlockBytes + (key_row + 8 * h) * (hd / 2) + t4 * GROUPS * 4;
              const uint32_t* pairs = k_pairs(x) + (key_row + 8 * h) * GROUPS;
              if constexpr (GROUPS == 4) {
                *reinterpret_cast<uint4*>(w[h]) = *reinterpret_cast<const uint4*>(from);
                *reinterpret_cast<uint4*>(pr[h]) = *reinterpret_cast<const uint4*>(pairs);
              } else {
                *reinterpret_cast<uint2*>(w[h]) = *reinterpret_cast<const uint2*>(from);
                *reinterpret_cast<uint2*>(pr[h]) = *reinterpret_cast<const uint2*>(pairs);
              }
              mine[h] = pairs[t4 % GROUPS];
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {  // the pairs with the queries' sums
              mma_new(s[x][nt], mine[0], mine[1], mine[0], mine[1], qs[nt][0], qs[nt][1]);
              mma<false>(s[x][nt], mine[0], mine[1], 0u, 0u, qs[nt][2], 0u);
            }
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
              uint32_t a[2][4];  // 128 + c
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) a[h][i] = masked_or(w[h][g] >> (4 * i), low4, 0x43004300u);
              const float s0 = low_of(pr[0][g]), s1 = low_of(pr[1][g]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float dot[4];
                const uint4 f = L::kKeep ? q[g] : fragment(nt, g);
                mma_new(dot, a[0][0], a[1][0], a[0][1], a[1][1], f.x, f.y);
                mma<false>(dot, a[0][2], a[1][2], a[0][3], a[1][3], f.z, f.w);
                s[x][nt][0] = fmaf(s0, dot[0], s[x][nt][0]);
                s[x][nt][1] = fmaf(s0, dot[1], s[x][nt][1]);
                s[x][nt][2] = fmaf(s1, dot[2], s[x][nt][2]);
                s[x][nt][3] = fmaf(s1, dot[3], s[x][nt][3]);
              }
            }
          }
          if (partly) {
            const int held = held_keys(p, d.keys);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int row = 8 * nt + 2 * t4 + e, pos = d.pos0 + min(row, d.rows - 1) / p.G;
                const int lo = first_seen(p, pos), hi = behind_seen(p, held, pos);
#pragma unroll
                for (int x = 0; x < kItem; ++x)
#pragma unroll
                  for (int h = 0; h < 2; ++h) {
                    const int j = key_row + 8 * h, key = (x ? info.z : info.x) + j;
                    if (j >= (x ? info.w : info.y) || key >= hi || (key < lo && key >= p.c.sinks)) s[x][nt][2 * h + e] = -INFINITY;
                  }
              }
          }
          // ---- weights
          float e[kItem][NT][4];
          bool above = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int x = 0; x < kItem; ++x) {
                e[x][nt][i] = fmaf(s[x][nt][i], p.c.scale_log2, kShift - m[nt][i % 2]);
                above |= e[x][nt][i] > kShift;
              }
          if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                float top = fmaxf(fmaxf(s[0][nt][r], s[0][nt][2 + r]), fmaxf(s[1][nt][r], s[1][nt][2 + r])) * p.c.scale_log2;
#pragma unroll
                for (int w = 4; w < 32; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                if (top > m[nt][r]) {  // of a row: all its lanes
                  const float corr = ex2(m[nt][r] - (top + kAbove));
                  m[nt][r] = top + kAbove;
                  l[nt][r] *= corr;
#pragma unroll
                  for (int i = 0; i < 2 * GROUPS; ++i) {
                    o[nt][i][r] *= corr;
                    o[nt][i][2 + r] *= corr;
                  }
                }
#pragma unroll
                for (int x = 0; x < kItem; ++x)
#pragma unroll
                  for (int h = 0; h < 2; ++h) e[x][nt][2 * h + r] = fmaf(s[x][nt][2 * h + r], p.c.scale_log2, kShift - m[nt][r]);
              }
          }
          uint32_t pb[kItem][NT][2];
#pragma unroll
          for (int x = 0; x < kItem; ++x)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int i = 0; i < 4; ++i) e[x][nt][i] = ex2(e[x][nt][i]);
              l[nt][0] += e[x][nt][0] + e[x][nt][2];
              l[nt][1] += e[x][nt][1] + e[x][nt][3];
              pb[x][nt][0] = transpose8(pack<HALF>(e[x][nt][0], e[x][nt][1]));
              pb[x][nt][1] = transpose8(pack<HALF>(e[x][nt][2], e[x][nt][3]));
            }
          // ---- values
#pragma unroll
          for (int x = 0; x < kItem; ++x) {
            constexpr int W = GROUPS / 2;  // words of a key here
            uint32_t w[4][W];
            uint4 sm[W];  // s and m of the keys of rows 2 t4, + 1, and of those 8 on
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = (k % 2 ? vb : va) + 8 * (k / 2);
              const unsigned char* from = blocks + x * L::kBlockBytes + 8 * hd + row * (hd / 2) + gid * W * 4;
              if constexpr (W == 2) *reinterpret_cast<uint2*>(w[k]) = *reinterpret_cast<const uint2*>(from);
              else w[k][0] = *reinterpret_cast<const uint32_t*>(from);
            }
#pragma unroll
            for (int i = 0; i < W; ++i)
              sm[i] = *reinterpret_cast<const uint4*>(pairs_out + ((x * GROUPS + (gid * W) % GROUPS + i) * 4 + t4) * 4);
            // codes of two keys beside each other: nibbles 0-3 and 4-7 of each word
            uint32_t part[2][W][2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < W; ++i) {
                part[h][i][0] = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x5410);
                part[h][i][1] = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x7632);
              }
            auto value = [&](uint32_t codes, int nibble, uint32_t sc, uint32_t mn) {
              if constexpr (HALF) {
                // the even nibbles as 1024 + c, the odd ones, 4 bits higher in the significand, as 64 + c
                const uint32_t y = nibble >= 2 ? codes >> 8 : codes, zero = nibble % 2 ? 0x54005400u : 0x64006400u;
                const uint32_t c = masked_or(y, nibble % 2 ? high4 : low4, zero);
                const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), *reinterpret_cast<const __half2*>(&zero)),
                                          *reinterpret_cast<const __half2*>(&sc), *reinterpret_cast<const __half2*>(&mn));
                return *reinterpret_cast<const uint32_t*>(&v);
              } else {
                return q4::stands_for(((codes >> (4 * nibble)) & 0x000f000fu) | 0x43004300u, sc, mn);
              }
            };
#pragma unroll
            for (int i = 0; i < 2 * GROUPS; ++i) {
              // rows gid and gid + 8 of the product: nibble i of the lane's two words, or nibbles i and i + 4 of its one
              const int x1 = W - 1, n1 = W == 2 ? i : i + 4;
              const uint32_t a0 = value(part[0][0][i / 4], i % 4, sm[0].x, sm[0].y);
              const uint32_t a1 = value(part[0][x1][n1 / 4], n1 % 4, sm[x1].x, sm[x1].y);
              const uint32_t a2 = value(part[1][0][i / 4], i % 4, sm[0].z, sm[0].w);
              const uint32_t a3 = value(part[1][x1][n1 / 4], n1 % 4, sm[x1].z, sm[x1].w);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma<HALF>(o[nt][i], a0, a1, a2, a3, pb[x][nt][0], pb[x][nt][1]);
            }
          }
        };
        if (half) body(std::true_type{});
        else body(std::false_type{});
        __syncwarp();
        ++computed;
      }
      // ---- the unit's part: a lane has words' 8 elements of rows 2 t4, + 1: of two words, or one
      constexpr int W = GROUPS / 2;
      auto element = [&](int nt, int word, int r, int e) -> float& {  // element e lies in nibble e / 2 + 4 (e % 2)
        const int nibble = e / 2 + 4 * (e % 2);
        return W == 2 ? o[nt][nibble][2 * word + r] : o[nt][nibble % 4][2 * (nibble / 4) + r];
      };
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float sum = l[nt][r];
#pragma unroll
          for (int w = 4; w < 32; w *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
          const int row = 8 * nt + 2 * t4 + r;
          if (row >= d.rows) continue;
          if (d.parts == 1) {
            const int64_t token = d.token0 + row / p.G;
            const int head = d.kvh * p.G + row % p.G;
            float f = sum == 0.f ? 0.f : 1.f / sum;
            if (p.c.gate && sum != 0.f) f *= sigmoid(p.c.gate[token * p.c.gate_stride + head]);
#pragma unroll
            for (int i = 0; i < W; ++i) {
              const int word = gid * W + i;  // of dims 32 (word % GROUPS) + 8 (word / GROUPS) on
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = sum == 0.f ? 0u : pack<false>(element(nt, i, r, 2 * e) * f, element(nt, i, r, 2 * e + 1) * f);
              *reinterpret_cast<uint4*>(p.c.out + token * p.c.out_stride + (int64_t)head * hd + 32 * (word % GROUPS) +
                                        8 * (word / GROUPS)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            if (p.c.lse && gid == 0)
              p.c.lse[token * p.c.Hq + head] = sum == 0.f ? -INFINITY : (m[nt][r] - kShift + log2f(sum)) * 0.6931471805599453f;
          } else {
            const int64_t part = part_slot(d.first, d.index);
#pragma unroll
            for (int i = 0; i < W; ++i) {
              const int word = gid * W + i;
              float* to = p.acc + (part * p.c.rows + row) * hd + 32 * (word % GROUPS) + 8 * (word / GROUPS);
              __stcg(reinterpret_cast<float4*>(to), make_float4(element(nt, i, r, 0), element(nt, i, r, 1), element(nt, i, r, 2), element(nt, i, r, 3)));
              __stcg(reinterpret_cast<float4*>(to) + 1, make_float4(element(nt, i, r, 4), element(nt, i, r, 5), element(nt, i, r, 6), element(nt, i, r, 7)));
            }
            if (gid == 0) {
              __stcg(p.ml + part * 2 * p.c.rows + row, sum == 0.f ? kNone : m[nt][r]);
              __stcg(p.ml + (part * 2 + 1) * p.c.rows + row, sum);
            }
          }
        }
      // ---- parts that are all there are joined, 16 neighbours at a time: into the first one's slot, or to the output
      int index = d.index, parts = d.parts, stride = 1, level = 0;
#pragma unroll 1
      while (parts > 1) {
        __threadfence();
        __syncwarp();
        const int leader = index / kJoin * kJoin, count = min(kJoin, parts - leader);  // in units of `stride` parts
        int last = 0;
        if (lane == 0) {
          // the warps between two first ones are inside the unit: theirs are free for the joins of joined parts
          unsigned* counter = p.counters + ((int64_t)(d.first + leader * stride + level) * 2 + (leader != 0));
          unsigned old = *reinterpret_cast<volatile unsigned*>(counter), seen, arrived;
          do {
            seen = old;
            arrived = (seen >> 12 == p.tag ? seen & 0xfffu : 0u) + 1;
            old = atomicCAS(counter, seen, arrived == (unsigned)count ? 0u : p.tag << 12 | arrived);
          } while (old != seen);
          last = arrived == (unsigned)count;
          __threadfence();
        }
        last = __shfl_sync(0xffffffffu, last, 0);
        if (!last) break;
        const bool final = parts <= kJoin;
        constexpr int kQuads = hd / 4, kTogether = 4, kAtOnce = 2;  // of a lane: rows' pieces, parts whose loads are in flight
        const int64_t to = part_slot(d.first, leader * stride);
#pragma unroll 1
        for (int x0 = lane; x0 < d.rows * kQuads; x0 += 32 * kAtOnce) {
          float top[kAtOnce], sum[kAtOnce], y[kAtOnce][4];
#pragma unroll
          for (int a = 0; a < kAtOnce; ++a) {
            top[a] = kNone;
            sum[a] = y[a][0] = y[a][1] = y[a][2] = y[a][3] = 0.f;
          }
#pragma unroll 1
          for (int i0 = 0; i0 < count; i0 += kTogether) {
            float pm[kAtOnce][kTogether], pl[kAtOnce][kTogether];
            float4 v[kAtOnce][kTogether];
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a)
#pragma unroll
              for (int k = 0; k < kTogether; ++k) {
                const int x = x0 + 32 * a, row = x / kQuads, quad = x % kQuads;
                const bool there = i0 + k < count && row < d.rows;
                const int64_t part = part_slot(d.first, (leader + (there ? i0 + k : 0)) * stride);
                pm[a][k] = there ? __ldcg(p.ml + part * 2 * p.c.rows + row) : kNone;
                pl[a][k] = there ? __ldcg(p.ml + (part * 2 + 1) * p.c.rows + row) : 0.f;
                v[a][k] = there ? __ldcg(reinterpret_cast<const float4*>(p.acc + (part * p.c.rows + row) * hd + quad * 4))
                                : make_float4(0.f, 0.f, 0.f, 0.f);
              }
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) {
              float high = top[a];
#pragma unroll
              for (int k = 0; k < kTogether; ++k) high = fmaxf(high, pm[a][k]);
              const float before = ex2(top[a] - high);
              top[a] = high;
              sum[a] *= before;
#pragma unroll
              for (int e = 0; e < 4; ++e) y[a][e] *= before;
#pragma unroll
              for (int k = 0; k < kTogether; ++k) {
                const float f = ex2(pm[a][k] - high);
                sum[a] = fmaf(pl[a][k], f, sum[a]);
                y[a][0] = fmaf(v[a][k].x, f, y[a][0]), y[a][1] = fmaf(v[a][k].y, f, y[a][1]);
                y[a][2] = fmaf(v[a][k].z, f, y[a][2]), y[a][3] = fmaf(v[a][k].w, f, y[a][3]);
              }
            }
          }
          // (the first part's m and sum are rewritten only when every lane has read them)
          if (!final) __syncwarp();
#pragma unroll
          for (int a = 0; a < kAtOnce; ++a) {
            const int x = x0 + 32 * a, row = x / kQuads, quad = x % kQuads;
            if (row >= d.rows) continue;
            if (final) {
              const int64_t token = d.token0 + row / p.G;
              const int head = d.kvh * p.G + row % p.G;
              float f = sum[a] == 0.f ? 0.f : 1.f / sum[a];
              if (p.c.gate && sum[a] != 0.f) f *= sigmoid(p.c.gate[token * p.c.gate_stride + head]);
              uint2 w;
              w.x = sum[a] == 0.f ? 0u : pack<false>(y[a][0] * f, y[a][1] * f);
              w.y = sum[a] == 0.f ? 0u : pack<false>(y[a][2] * f, y[a][3] * f);
              *reinterpret_cast<uint2*>(p.c.out + token * p.c.out_stride + (int64_t)head * hd + quad * 4) = w;
              if (p.c.lse && quad == 0)
                p.c.lse[token * p.c.Hq + head] = sum[a] == 0.f ? -INFINITY : (top[a] - kShift + log2f(sum[a])) * 0.6931471805599453f;
            } else {
              __stcg(reinterpret_cast<float4*>(p.acc + (to * p.c.rows + row) * hd + quad * 4), make_float4(y[a][0], y[a][1], y[a][2], y[a][3]));
              if (quad == 0) {
                __stcg(p.ml + to * 2 * p.c.rows + row, top[a]);
                __stcg(p.ml + (to * 2 + 1) * p.c.rows + row, sum[a]);
              }
            }
          }
          if (!final) __syncwarp();
        }
        index = leader / kJoin;
        parts = (parts + kJoin - 1) / kJoin;
        stride *= kJoin;
        ++level;
      }
      ++done;
      loaded = false;
    }
    wait_copies<0>();
  }
  // ---- rows of no request, where no other kernel takes them
  if (p.c.only && !refused) {
    const int idle = tl.idle[0] + p.c.kv.N - tl.idle[1];
#pragma unroll 1
    for (int i = worker; i < idle; i += p.workers) {
      const int64_t t = i < tl.idle[0] ? i : tl.idle[1] + i - tl.idle[0];
#pragma unroll 1
      for (int c = lane; c < p.c.Hq * hd / 8; c += 32)
        *reinterpret_cast<uint4*>(p.c.out + t * p.c.out_stride + c * 8) = make_uint4(0, 0, 0, 0);
      if (p.c.lse)
#pragma unroll 1
        for (int h = lane; h < p.c.Hq; h += 32) p.c.lse[t * p.c.Hq + h] = -INFINITY;
    }
  }
}

// The CTAs of a launch: those that are on the GPU at once, or as many as a batch can have a share for.
int ctas_of(int B, int N, int Hkv, int64_t max_keys, int warps) {
  const int64_t items = (max_keys + kItem * q4::kBlock - 1) / (kItem * q4::kBlock) + 1;  // of a unit; sinks may add one
  const int64_t shares = std::min<int64_t>(B, N) * Hkv * (items + kUnitCost) / kMinShare + 1;
  const int64_t most = std::min<int64_t>((int64_t)zb::sm_count() * 2, q4::kFewFlagBytes / 8 / warps - 1);
  return (int)std::max<int64_t>(1, std::min(most, shares));  // a warp of each first: few shares are spread over the SMs
}

template <int GROUPS, int NT>
int launch(FewParams& p, int ctas, cudaStream_t stream) {
  using L = Shape<GROUPS, NT>;
  auto kernel = gqa_few_q4_kernel<GROUPS, NT>;
  constexpr int kSmem = L::kWarps * L::kPerWarp + (int)sizeof(Tail);
  static_assert((kSmem + 1024) * L::kCtas <= 228 * 1024, "shared memory");
  static bool configured[64] = {false};  // the shared-memory attribute, set once per device
  int dev = 0;
  ZB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    ZB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  p.workers = ctas * L::kWarps;
  ZB_CUDA(zb::launch(kernel, dim3((unsigned)ctas), dim3(L::kThreads), (size_t)kSmem, stream, 1, p));
  return zb::check_launch("gqa_chunk_q4");
}

int warps_of(int rows) { return rows <= 8 ? 8 : 6; }

}  // namespace

namespace zb {
namespace q4 {

int few_rows(int hd, int G, int max_new) {
  if (hd != 64 && hd != 128) return 0;
  const int64_t rows = (int64_t)max_new * G;
  if (rows <= 16) return rows <= 8 ? 8 : 16;
  // Requests of many rows are there or may be: the single tokens beside them, by the leaner kernel where it holds them
  return G <= 8 ? 8 : G <= 16 ? 16 : 0;
}

int64_t few_workspace_bytes(int B, int N, int Hkv, int hd, int rows, int64_t max_keys) {
  if (rows == 0 || B < 1 || N < 1) return 0;
  return kFewFlagBytes + (int64_t)ctas_of(B, N, Hkv, max_keys, warps_of(rows)) * warps_of(rows) * 2 * rows * (hd + 2) * 4;
}

int launch_few(const FewCall& call, cudaStream_t stream) {
  FewParams p;
  p.c = call;
  p.G = call.Hq / call.kv.Hkv;
  unsigned l = 0;
  while ((1u << l) < (unsigned)call.kv.page_size) ++l;
  p.page_shift = 31 + l;
  p.page_mul = (unsigned)((((uint64_t)1 << p.page_shift) + call.kv.page_size - 1) / call.kv.page_size);
  const int warps = warps_of(call.rows);
  const int ctas = ctas_of(call.kv.B, call.kv.N, call.kv.Hkv, (int64_t)call.kv.page_size * call.kv.max_pages, warps);
  static std::atomic<unsigned> calls{0};
  do p.tag = (calls.fetch_add(1, std::memory_order_relaxed) + 1) & 0xfffffu;
  while (p.tag == 0);
  p.counters = reinterpret_cast<unsigned*>(call.workspace);
  p.acc = reinterpret_cast<float*>(call.workspace + kFewFlagBytes);
  p.ml = p.acc + (int64_t)ctas * warps * 2 * call.rows * call.kv.hd;
  p.status = device_status_ptr();
  if (call.kv.hd == 128) return call.rows == 8 ? launch<4, 1>(p, ctas, stream) : launch<4, 2>(p, ctas, stream);
  return call.rows == 8 ? launch<2, 1>(p, ctas, stream) : launch<2, 2>(p, ctas, stream);
}

}  // namespace q4
}  // namespace zb
