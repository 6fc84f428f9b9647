// Attention of few rows over a paged KV cache in 4 bits (kv_q4.cuh): the single tokens, and short drafts of them, of a decode
// batch. The mathematics is that of gqa_chunk.cu; requests of more rows are its kernel's.
//
// The rows of a request's score matrix for one KV head are its (token, head of the group) pairs, up to 8 (NT = 1) or 16. A row
// reads every code once, so the work is the codes' way from HBM and their unpacking; the products are few. So they are
// formed from registers (m16n8k16: 16 keys or dims by 8 rows), where a code goes from the loaded word into a matrix fragment
// with two instructions for two codes, and nothing is written out in between as a tensor-memory product would need it:
//   scores^T [16 keys, 8 rows] = sum over groups g of  s_g (c . q)_g + m_g (sum q)_g:  the codes themselves are the operand, as fp16
//     subnormals, which takes one instruction for two of them; the queries, scaled into fp16's range, keep their 8 bits. s goes onto
//     the products' sums in fp32; the second term is a product of its own, the pairs as they lie in the cache times the queries'
//     sums, split into three bf16. So the scores are as good as fp32's, down to 2^-35 of a row's largest element;
//   out^T [16 dims of a group, 8 rows] += c (s_g p^T), and p^T m_g and the sum of p by a product more. Weights are fp16, 2^-12 of
//     each: bf16's 2^-9 would be the largest error here. fp16 has less range, so an item whose pairs are not all within it
//     (half_holds()) and those after it take bf16.
// A weight is 2^(score - m + 15) with m a row's reference, its largest score or up to 2 (log2) above it when it is set; it is set
// anew by a score above it, rarely after the first items. So weights lie in fp16's range: up to 2^15, the largest not below 2^13
// when m is set, and those below 2^-40 of m count as 0. m and the sum cancel in the end. s p is formed in fp16 too and has its
// range: with the smallest step, 2^-12, it is rounded as fp16 does for weights down to 2^-15 of the largest and gone at 2^-26; with
// steps of 2^-4 at 2^-23 and 2^-34. (With m up to 8 above, 65536 keys 2^-20 to 2^-23 of a first one that stands out were off by a
// tenth to a third. 0 above costs 256 tokens over 1628 keys 74.3 us for setting m more often, 1 72.8, 2 72.2, 4 and 8 71.9.)
// The keys of a 16-key block stand in the scores' rows in the order 0 1 3 2 4 5 7 6 and 8 on: the two rows of a quarter of the lanes then
// read other banks, and the four rows that a quarter's values come from too, as far as 64-byte rows allow.
//
// Every warp works for itself. All units' keys are one long run of items (two blocks of 16 keys, at hd 128 2560 bytes
// each), of which a warp takes an equal share (the split is as in gqa_chunk.cu, to warps instead of CTAs): it looks up the places of
// its blocks, has the copies of the next item under way while it computes one, and keeps m, the sum and the accumulator of a unit in
// its registers, where a lane has 8 consecutive elements of up to four rows' outputs. A unit that spans warps leaves a part of each
// in the workspace; the warp that finishes the last of up to 8 neighbouring parts joins them in the order of their keys, and so on
// for the joined ones. No warp waits for another, and results do not depend on timing.
//
// Measured (B200, 16 / 4 heads of 128): 256 tokens over 1628 keys (268 MB) 72 us, 3.7 TB/s, 0.57 of a copy's (90 where values take
// bf16, all steps below 2^-12); the copies alone take 48, the unpacking and products 17 beside them, the joins 4. Issue slots 51 %, the
// logic pipe 46 %, matrix pipe 23 %: a warp's chain of wait, unpack, products, weights leaves slots that more warps (12 to 16 an SM) or
// stages did not fill. 2 tokens over 65001 keys (83 MB) 36 us, 12 of them the three levels of joins; one over 878 keys 16, launch
// and chain.
// Measured ways that were slower (256 tokens of 16 / 4 heads of 128 over 1628 keys): seven warps a CTA that share a unit's items, an eighth
// that starts the copies, the accumulators joined in shared memory: 105-112 us. Each warp waited for copies and at every
// unit's end for the slowest; half of the cycles issued nothing.
#include <algorithm>

#include "few_q4.cuh"

namespace {

namespace q4 = zb::q4;

constexpr int kItem = 2;      // blocks of an item
constexpr int kStages = 2;    // items of a warp: one that is computed, and copies under way
constexpr int kUnitCost = 4;  // of a unit, in items
constexpr int kMinShare = 3;  // items of a warp, its units' cost among them
constexpr int kJoin = 8;      // parts that are joined at once
constexpr float kAbove = 2.f, kShift = 15.f;
constexpr float kNone = -3.0e38f;  // m of a row that has seen no key

struct FewParams {
  q4::FewCall c;
  int G, workers;
  unsigned page_mul, page_shift;  // division by the page size
  // [warp][2]: how many parts have arrived of those that are joined with one of the warp's (the first of them; [0]: of the unit that
  // began there, [1]: of one that had begun before); 0 again when all have
  unsigned* counters;
  float* acc;  // [warp][2][rows][hd]: parts
  float2* ml;  // [warp][2][rows]: m, sum
  unsigned* status;
};

// What a warp does with one unit.
struct Desc {
  int token0, pos0, keys;  // first token row, its key position, keys of the request
  int rows, kvh;
  int items;
  int index, parts, first;  // of the unit's parts this one, their number, and the warp that has the first
  int from;                 // keys from the sinks' end to here are hidden from every row
};
// Where a block lies; its first key; how many of its keys there are, and kPartly if some rows do not see some of its keys.
struct Place {
  const unsigned char* at;
  int key0, exist;
};
constexpr int kPartly = 256;
// A warp's own shared memory, behind its stages and queries.
struct Own {
  int2 info[kStages][kItem];  // of the stages' blocks: a Place's key0 and exist
  alignas(16) Place places[32];
  Desc desc[2];
  // the unit after those opened: how far its request and the share have got
  int64_t at;
  int b, kvh, off;
  int row0, tokens, keys;
  // of the unit opened last: blocks whose places are not looked up yet, and what that takes
  int next, end, n, sink_blocks, gap, of_b, of_kvh, held, all_lo, all_hi;
};

template <int GROUPS, int NT>
struct Shape {
  static constexpr int kHd = GROUPS * q4::kGroup, kBlockBytes = q4::block_bytes(kHd), kRows = 8 * NT;
  static constexpr int kStage = kItem * kBlockBytes;
  static constexpr int kOffQ = kStages * kStage;
  static constexpr int kOffPairs = kOffQ + kRows * kHd * 2;  // pairs of values, as the lanes need them
  static constexpr int kOffOwn = kOffPairs + kItem * GROUPS * 64;
  static constexpr int kPerWarp = (kOffOwn + (int)sizeof(Own) + 127) / 128 * 128;
  // 12 warps an SM have 168 registers a thread. 16 with 128 keep some in memory: 71 us against 72 for 256 tokens over 1628 keys,
  // but 40 against 36 for 2 over 65001.
  static constexpr int kWarps = 6, kCtas = 2, kThreads = 32 * kWarps;
  // The queries' fragments stay in registers, or are read again for every block where the accumulators take those.
  static constexpr bool kKeep = NT == 1;
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
// The same with half the depth, of bf16.
__device__ __forceinline__ void mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ void mma8_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}
// D = A B of fp16
__device__ __forceinline__ void mma_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
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

// Whether fp16 keeps a pair's s and 2^8 m well: s is below 2 and |m| below 2^7 (a sign bit of `over` else), and s is 2^-12 or
// more, or the pair is 0 (`holds`). And whether it is not 0 (`some`), and s 2^-8 or more (`big`).
__device__ __forceinline__ void half_holds(uint32_t pair, uint32_t& over, bool& holds) {
  const uint32_t a = pair & 0x7fff7fffu;
  over |= a + (((0x8000u - 0x4300u) << 16) | (0x8000u - 0x4000u));
  holds &= a << 16 >= 0x3980u << 16 || a == 0;
}
// Bit 7 of the bytes that are not 0.
__device__ __forceinline__ uint32_t bytes_set(uint32_t x) { return (((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) & 0x80808080u; }

__device__ __forceinline__ void fence_gpu() { asm volatile("fence.acq_rel.gpu;" ::: "memory"); }
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
// While the work is split, over the first warp's stages: a round of requests, and their places in it.
struct Round {
  int before[256], cost[256];
  Request request[256];
};
struct Tail {
  int sums[2][16];
  int idle[2];
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

// n / d, whose quotient fits 32 bits; n hardly ever does not.
__device__ __forceinline__ int quotient(int64_t n, int d) { return n <= INT32_MAX ? (int)n / d : (int)(n / d); }

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
__device__ __forceinline__ unsigned part_slot(int first, int index) { return (unsigned)(first + index) * 2 + (index == 0); }

template <int GROUPS, int NT>
__global__ void __launch_bounds__(Shape<GROUPS, NT>::kThreads, Shape<GROUPS, NT>::kCtas)
    gqa_few_q4_kernel(const __grid_constant__ FewParams p) {
  using L = Shape<GROUPS, NT>;
  constexpr int hd = L::kHd, kWarps = L::kWarps, kThreads = L::kThreads;
  extern __shared__ __align__(128) unsigned char gbase[];
  Tail& tl = *reinterpret_cast<Tail*>(gbase + kWarps * L::kPerWarp);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid % 32;
  Round& round = *reinterpret_cast<Round*>(gbase);
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
  const int share = max(kMinShare, quotient(work + p.workers - 1, p.workers));
  const int64_t begin = (int64_t)share * worker, end = min(work, begin + share);
  {
    const int64_t of_head = begin <= INT32_MAX ? (int)begin / Hkv : begin / Hkv;  // how far the share's begin is into the work of one head
    int64_t seen = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < B; b0 += kThreads) {
      int cost = mine_cost, before = mine_before, total = mine_total;
      Request r = mine;
      if (b0 > 0) {
        r = b0 + tid < B ? request(p, b0 + tid, more) : Request{0, 0, 0};
        cost = cost_of(p, r);
        buffer ^= 1;
        before = block_scan<kWarps>(cost, tl, buffer, total);
      }
      if (work > 0) {
        round.before[tid] = before;
        round.cost[tid] = cost;
        round.request[tid] = r;
      }
      __syncthreads();
      if (begin < end && of_head >= seen && of_head < seen + total) {
        const int into = (int)(of_head - seen);
#pragma unroll 2
        for (int i = lane; i < kThreads; i += 32) {
          if (into >= round.before[i] && into - round.before[i] < round.cost[i]) {
            const int64_t rest = begin - (seen + round.before[i]) * Hkv;
            const int kvh = quotient(rest, round.cost[i]);
            my.at = begin;
            my.b = b0 + i;
            my.kvh = kvh;
            my.off = (int)(rest - (int64_t)kvh * round.cost[i]);
            my.row0 = round.request[i].row0;
            my.tokens = round.request[i].tokens;
            my.keys = round.request[i].keys;
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
            d.first = x.n > 0 ? quotient(first, share) : worker;
            d.index = worker - d.first;
            d.parts = x.n > 0 ? quotient(first + unit_items - 1, share) - d.first + 1 : 1;
            d.from = x.lo_first;
            my.desc[opened % 2] = d;
            my.next = from * kItem;
            my.end = to * kItem;
            my.n = x.n;
            my.sink_blocks = x.sink_blocks;
            my.gap = x.gap;
            my.of_b = b;
            my.of_kvh = kvh;
            my.held = held_keys(p, req.keys);
            my.all_lo = x.lo_last;
            my.all_hi = x.hi_first;
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
          const int exist = there ? min(q4::kBlock, my.held - key0) : 0;
          // keys of [all_lo, all_hi), and those below min(sinks, all_hi), are seen by every row
          const bool all = exist == q4::kBlock && key0 + q4::kBlock <= my.all_hi && (key0 >= my.all_lo || key0 + q4::kBlock <= p.c.sinks);
          found.exist = exist | (all ? 0 : kPartly);
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
      const int stage = fetched % kStages;
#pragma unroll
      for (int x = 0; x < kItem; ++x) {
        const Place found = my.places[place + x];
        const uint32_t to = zb::smem_addr(own + stage * L::kStage + x * L::kBlockBytes) + lane * 16;
        if (lane == 0) my.info[stage][x] = make_int2(found.key0, found.exist);
        if (found.exist & (kPartly - 1))
#pragma unroll
          for (int i = 0; i < L::kBlockBytes; i += 512)
            if (i + 512 <= L::kBlockBytes || lane * 16 < L::kBlockBytes - i) copy16(to + i, found.at + i + lane * 16);
      }
      commit_copies();
      place += kItem;
      ++fetched;
    };
    const uint32_t low4 = 0x000f000fu, high4 = 0x00f000f0u, halves = gid < 4 ? 0x5410u : 0x7632u;

#pragma unroll 1
    for (int k = 0; k < kStages; ++k) fetch();
#pragma unroll 1
    while (true) {
      if (opened == done) open_unit();
      if (opened == done) break;
      const Desc& d = my.desc[done % 2];  // not held in registers through the items
      // The copies of the item to be computed, and with them those of its unit's queries.
      auto arrived = [&]() {
        const int behind = fetched - computed - 1;
        if (behind > 1) wait_copies<2>();
        else if (behind > 0) wait_copies<1>();
        else wait_copies<0>();
        __syncwarp();
      };
      if (fetched == computed) fetch();
      arrived();
      // ---- queries, scaled by a power of 2 to a largest element of 2^14 to 2^15: B fragments in fp16, and what a group's m multiplies,
      // the sum of its elements of the query, as three bf16. (c . q) comes with 2^-24 for every code's 1, or with 2^-20 for those 4
      // bits higher, whose elements of the query have 2^-4 less.
      const unsigned char* q_rows = own + L::kOffQ;
      uint4 q[NT][L::kKeep ? GROUPS : 1];
      uint32_t qs[NT][3];
      float scale[NT][2];  // of the scores of rows 2 t4, + 1
      auto fragment = [&](int nt, int g, float by, float& sum) {
        const uint4 w = 8 * nt + gid < d.rows ? *reinterpret_cast<const uint4*>(q_rows + (8 * nt + gid) * hd * 2 + (32 * g + 8 * t4) * 2)
                                              : make_uint4(0, 0, 0, 0);
        const float high = by * 0x1p-4f;
        sum = (low_of(w.x) + high_of(w.x) + (low_of(w.y) + high_of(w.y)) + (low_of(w.z) + high_of(w.z) + (low_of(w.w) + high_of(w.w)))) * by;
        return make_uint4(pack<true>(low_of(w.x) * by, high_of(w.x) * by), pack<true>(low_of(w.y) * high, high_of(w.y) * high),
                          pack<true>(low_of(w.z) * by, high_of(w.z) * by), pack<true>(low_of(w.w) * high, high_of(w.w) * high));
      };
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t top = 0;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
          if (8 * nt + gid < d.rows) {
            const uint4 w = *reinterpret_cast<const uint4*>(q_rows + (8 * nt + gid) * hd * 2 + (32 * g + 8 * t4) * 2);
            top = __vmaxu2(__vmaxu2(top, w.x & 0x7fff7fffu), __vmaxu2(w.y & 0x7fff7fffu, __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
          }
        top = max(top >> 16, top & 0xffffu) >> 7;  // the largest exponent
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(max(top, __shfl_xor_sync(0xffffffffu, top, 2)), 16u);
        const bool none = top >= 244;  // not finite, or at the end of the range: the row's scores become NaN
        const float by = __uint_as_float((268u - min(top, 244u)) << 23);
        float of_group = 0.f;  // t4
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          float sum;
          const uint4 f = fragment(nt, g, by, sum);
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if (g == t4) of_group = none ? NAN : sum * 0x1p-24f;
          if (L::kKeep) q[nt][g] = f;
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) {
          const float kept = zb::bf16_round(of_group);
          qs[nt][i] = pack<false>(0.f, kept);
          of_group -= kept;
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t its = __shfl_sync(0xffffffffu, top, 8 * t4 + 4 * r);
          scale[nt][r] = p.c.scale_log2 * __uint_as_float((min(its, 244u) + 10u) << 23);
        }
        if (!L::kKeep) {  // the fragments over the queries
          __syncwarp();
          uint4 f[GROUPS];
          float ignored;
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) f[g] = fragment(nt, g, by, ignored);
          __syncwarp();
#pragma unroll
          for (int g = 0; g < GROUPS; ++g)
            *reinterpret_cast<uint4*>(own + L::kOffQ + (8 * nt + gid) * hd * 2 + (32 * g + 8 * t4) * 2) = f[g];
          __syncwarp();
        }
      }
      __syncwarp();
      loaded = true;
      // Of rows 2 t4 and 2 t4 + 1 (and 8 on): m; sum of p s c 2^-24, or 2^-20, of 16 elements of a group at a time; and, on lanes
      // 4 g + t4, the sum of 2^8 p m of group g, on lanes 16 + t4 that of p.
      float m[NT][2], o[NT][2 * GROUPS][4], om[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = kNone;
        om[nt][0] = om[nt][1] = om[nt][2] = om[nt][3] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * GROUPS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      }
      uint32_t* s_out = reinterpret_cast<uint32_t*>(own + L::kOffPairs);  // [item's block][t4][rows 2 t4, + 1, or 8 on][group]
      uint32_t* m_out = s_out + kItem * 8 * GROUPS;                         // [item's block][group][t4][rows 2 t4, + 1, or 8 on]
      // Items from `item` on; returns the first that fp16 does not hold, which and those after it bf16 then takes. (Two loops: with
      // the choice inside one, the accumulators changed places between its branches.)
      auto run = [&](auto type, int item) {
        constexpr bool HALF = decltype(type)::value;
        const int items = d.items;
#pragma unroll 1
        for (; item < items; ++item) {
#pragma unroll 1
        for (int k = fetched - computed; k < kStages; ++k) fetch();
        const int stage = computed % kStages;
        arrived();
        int2 info[kItem];
        bool partly = false;
#pragma unroll
        for (int x = 0; x < kItem; ++x) {
          info[x] = my.info[stage][x];
          partly |= (info[x].y & kPartly) != 0;
        }
        unsigned char* blocks = own + stage * L::kStage;
        auto k_pairs = [&](int x) { return reinterpret_cast<uint32_t*>(blocks + x * L::kBlockBytes + 16 * hd); };
        auto v_pairs = [&](int x) { return reinterpret_cast<uint32_t*>(blocks + x * L::kBlockBytes + 18 * hd); };
        if (partly) {  // rows that are no keys hold anything, and what no row sees shall not choose the values' type either
#pragma unroll
          for (int x = 0; x < kItem; ++x)
#pragma unroll 1
            for (int i = lane; i < 16 * GROUPS; i += 32) {
              const int j = i / GROUPS, key = info[x].x + j;
              if (j >= (info[x].y & (kPartly - 1)) || (key >= p.c.sinks && key < d.from)) k_pairs(x)[i] = v_pairs(x)[i] = 0;
            }
          __syncwarp();
        }
        // Pairs: none of the keys' may count as one that is not finite; the values' go to where the lanes that need them read
        // them, two keys' s and m beside each other.
        {
          const int g = lane / 8 % GROUPS, t = lane % 4, h = lane / 4 % 2;  // a group, and the keys of scores' rows 2 t + 8 h, + 1
          const int row = 2 * t + (t & 1) + 8 * h;
          uint32_t none = 0, over = 0, a[kItem][2];
          bool holds = true;
#pragma unroll
          for (int x = 0; x < kItem; ++x) {
            const uint2 k2 = GROUPS == 4 ? reinterpret_cast<const uint2*>(k_pairs(x))[lane] : make_uint2(k_pairs(x)[lane], 0);
            none |= q4::none_bits(k2.x) | q4::none_bits(k2.y);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              a[x][k] = v_pairs(x)[(row ^ k) * GROUPS + g];
              half_holds(a[x][k], over, holds);
            }
          }
          if (HALF && !__all_sync(0xffffffffu, holds && (over & 0x80008000u) == 0)) return item;
#pragma unroll
          for (int x = 0; x < kItem; ++x) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
              if (!HALF && q4::pair_is_none(a[x][k])) a[x][k] = 0;
            const float by = HALF ? 1.f : 0x1p-24f;
            if (lane < 8 * GROUPS) {
              s_out[x * 8 * GROUPS + (t * 2 + h) * GROUPS + g] = pack<HALF>(low_of(a[x][0]) * by, low_of(a[x][1]) * by);
              m_out[x * 8 * GROUPS + (g * 4 + t) * 2 + h] = pack<HALF>(high_of(a[x][0]) * 0x1p8f, high_of(a[x][1]) * 0x1p8f);
            }
          }
          if (__any_sync(0xffffffffu, (none & 0x80008000u) != 0)) {
#pragma unroll
            for (int x = 0; x < kItem; ++x)
              for (int i = lane; i < 16 * GROUPS; i += 32)
                if (q4::pair_is_none(k_pairs(x)[i])) k_pairs(x)[i] = 0;
          }
          __syncwarp();
        }
        {
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
              mma8_new(s[x][nt], mine[0], mine[1], qs[nt][0]);
              mma8(s[x][nt], mine[0], mine[1], qs[nt][1]);
              mma8(s[x][nt], mine[0], mine[1], qs[nt][2]);
            }
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
              // a code in the lowest 4 bits of an fp16 is c 2^-24, one 4 bits higher c 2^-20: no constant to join it to
              uint32_t a[2][4];
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t upper = w[h][g] >> 8;
                a[h][0] = w[h][g] & low4, a[h][1] = w[h][g] & high4, a[h][2] = upper & low4, a[h][3] = upper & high4;
              }
              const float s0 = low_of(pr[0][g]), s1 = low_of(pr[1][g]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float dot[4];
                const uint4 f = L::kKeep ? q[nt][g] : *reinterpret_cast<const uint4*>(q_rows + (8 * nt + gid) * hd * 2 + (32 * g + 8 * t4) * 2);
                mma_new(dot, a[0][0], a[1][0], a[0][1], a[1][1], f.x, f.y);
                mma<true>(dot, a[0][2], a[1][2], a[0][3], a[1][3], f.z, f.w);
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
                    const int j = key_row + 8 * h, key = info[x].x + j;
                    if (j >= (info[x].y & (kPartly - 1)) || key >= hi || (key < lo && key >= p.c.sinks)) s[x][nt][2 * h + e] = -INFINITY;
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
                e[x][nt][i] = fmaf(s[x][nt][i], scale[nt][i % 2], kShift - m[nt][i % 2]);
                above |= e[x][nt][i] > kShift;
              }
          if (__any_sync(0xffffffffu, above)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                float top = fmaxf(s[0][nt][r], s[0][nt][2 + r]);
#pragma unroll
                for (int x = 1; x < kItem; ++x) top = fmaxf(top, fmaxf(s[x][nt][r], s[x][nt][2 + r]));
                top *= scale[nt][r];
#pragma unroll
                for (int w = 4; w < 32; w *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                if (top > m[nt][r]) {  // of a row: all its lanes
                  const float corr = ex2(m[nt][r] - (top + kAbove));
                  m[nt][r] = top + kAbove;
                  om[nt][r] *= corr;
#pragma unroll
                  for (int i = 0; i < 2 * GROUPS; ++i) {
                    o[nt][i][r] *= corr;
                    o[nt][i][2 + r] *= corr;
                  }
                }
#pragma unroll
                for (int x = 0; x < kItem; ++x)
#pragma unroll
                  for (int h = 0; h < 2; ++h) e[x][nt][2 * h + r] = fmaf(s[x][nt][2 * h + r], scale[nt][r], kShift - m[nt][r]);
              }
          }
          uint32_t pb[kItem][NT][2];
#pragma unroll
          for (int x = 0; x < kItem; ++x)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
              for (int i = 0; i < 4; ++i) e[x][nt][i] = ex2(e[x][nt][i]);
              pb[x][nt][0] = transpose8(pack<HALF>(e[x][nt][0], e[x][nt][1]));
              pb[x][nt][1] = transpose8(pack<HALF>(e[x][nt][2], e[x][nt][3]));
            }
          // ---- values: a product's 16 rows are elements of one group, so that s goes onto the weights, two at a time, and the
          // codes are the operand as they are. Lanes of gid 0-3 take nibbles 0-3 of word gid of the group, those of gid 4-7 nibbles
          // 4-7 of word gid - 4.
#pragma unroll
          for (int x = 0; x < kItem; ++x) {
            uint32_t w[4][GROUPS], s2[2][GROUPS], ma[2];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int row = (k % 2 ? vb : va) + 8 * (k / 2);
              const unsigned char* from = blocks + x * L::kBlockBytes + 8 * hd + row * (hd / 2) + gid % 4 * GROUPS * 4;
              if constexpr (GROUPS == 4) *reinterpret_cast<uint4*>(w[k]) = *reinterpret_cast<const uint4*>(from);
              else *reinterpret_cast<uint2*>(w[k]) = *reinterpret_cast<const uint2*>(from);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t* from = s_out + x * 8 * GROUPS + (t4 * 2 + h) * GROUPS;
              if constexpr (GROUPS == 4) *reinterpret_cast<uint4*>(s2[h]) = *reinterpret_cast<const uint4*>(from);
              else *reinterpret_cast<uint2*>(s2[h]) = *reinterpret_cast<const uint2*>(from);
            }
            {
              const uint2 both = *reinterpret_cast<const uint2*>(m_out + x * 8 * GROUPS + (gid % GROUPS * 4 + t4) * 2);
              const uint32_t one = HALF ? 0x3c003c00u : 0x3f803f80u;
              ma[0] = gid < GROUPS ? both.x : gid == 4 ? one : 0u;
              ma[1] = gid < GROUPS ? both.y : gid == 4 ? one : 0u;
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<HALF>(om[nt], ma[0], 0u, ma[1], 0u, pb[x][nt][0], pb[x][nt][1]);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
              uint32_t a[2][4];  // codes of rows' keys 2 t4, + 1 (and 8 on), of a lane's four nibbles
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t y = __byte_perm(w[2 * h][g], w[2 * h + 1][g], halves);
                if constexpr (HALF) {
                  const uint32_t upper = y >> 8;
                  a[h][0] = y & low4, a[h][1] = y & high4, a[h][2] = upper & low4, a[h][3] = upper & high4;
                } else {
#pragma unroll
                  for (int i = 0; i < 4; ++i) {  // s c 2^-24, or 2^-20
                    const uint32_t c = ((y >> (4 * i)) & 0x000f000fu) | 0x43004300u, k128 = 0x43004300u, k16 = 0x41804180u;
                    __nv_bfloat162 v = __hmul2(__hsub2(q4::as_bf162(c), q4::as_bf162(k128)), q4::as_bf162(s2[h][g]));
                    a[h][i] = q4::as_word(i % 2 ? __hmul2(v, q4::as_bf162(k16)) : v);
                  }
                }
              }
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                uint32_t b[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  b[h] = pb[x][nt][h];
                  if constexpr (HALF) {
                    const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&b[h]), *reinterpret_cast<const __half2*>(&s2[h][g]));
                    b[h] = *reinterpret_cast<const uint32_t*>(&v);
                  }
                }
                mma<HALF>(o[nt][2 * g], a[0][0], a[0][1], a[1][0], a[1][1], b[0], b[1]);
                mma<HALF>(o[nt][2 * g + 1], a[0][2], a[0][3], a[1][2], a[1][3], b[0], b[1]);
              }
            }
          }
        }
        __syncwarp();
        ++computed;
        }
        return item;
      };
      const int held_items = run(std::true_type{}, 0);
      if (held_items < d.items) run(std::false_type{}, held_items);
      // ---- the unit's part: every second element of a word is on lane gid, the others on lane gid ^ 4; each takes 4 in a row
      const bool upper_half = gid >= 4;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float sum = __shfl_sync(0xffffffffu, om[nt][r], 16 + t4);
          float y[GROUPS][4];
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            const float mg = __shfl_sync(0xffffffffu, om[nt][r], 4 * g + t4) * 0x1p-8f;
            float x[4] = {fmaf(o[nt][2 * g][r], 0x1p24f, mg), fmaf(o[nt][2 * g][2 + r], 0x1p20f, mg),
                          fmaf(o[nt][2 * g + 1][r], 0x1p24f, mg), fmaf(o[nt][2 * g + 1][2 + r], 0x1p20f, mg)};
            const float z0 = __shfl_xor_sync(0xffffffffu, upper_half ? x[0] : x[2], 16);
            const float z1 = __shfl_xor_sync(0xffffffffu, upper_half ? x[1] : x[3], 16);
            y[g][0] = upper_half ? z0 : x[0], y[g][1] = upper_half ? x[2] : z0;
            y[g][2] = upper_half ? z1 : x[1], y[g][3] = upper_half ? x[3] : z1;
          }
          const int row = 8 * nt + 2 * t4 + r;
          if (row >= d.rows) continue;
          const int dim = 8 * (gid % 4) + 4 * (gid / 4);  // of a group
          if (d.parts == 1) {
            const int64_t token = d.token0 + row / p.G;
            const int head = d.kvh * p.G + row % p.G;
            float f = sum == 0.f ? 0.f : 1.f / sum;
            if (p.c.gate && sum != 0.f) f *= sigmoid(p.c.gate[token * p.c.gate_stride + head]);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
              *reinterpret_cast<uint2*>(p.c.out + token * p.c.out_stride + (int64_t)head * hd + 32 * g + dim) =
                  sum == 0.f ? make_uint2(0u, 0u) : make_uint2(pack<false>(y[g][0] * f, y[g][1] * f), pack<false>(y[g][2] * f, y[g][3] * f));
            if (p.c.lse && gid == 0)
              p.c.lse[token * p.c.Hq + head] = sum == 0.f ? -INFINITY : (m[nt][r] - kShift + log2f(sum)) * 0.6931471805599453f;
          } else {
            const unsigned at = part_slot(d.first, d.index) * L::kRows + row;  // parts of a call fit 2^31 floats
            float* to = p.acc + at * hd + dim;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
              __stcg(reinterpret_cast<float4*>(to + 32 * g), make_float4(y[g][0], y[g][1], y[g][2], y[g][3]));
            if (gid == 0) __stcg(p.ml + at, make_float2(sum == 0.f ? kNone : m[nt][r], sum));
          }
        }
      // ---- parts that are all there are joined, 8 neighbours at a time: into the first one's slot, or to the output
      int index = d.index, parts = d.parts, stride = 1, level = 0;
#pragma unroll 1
      while (parts > 1) {
        __syncwarp();
        const int leader = index / kJoin * kJoin, count = min(kJoin, parts - leader);  // in units of `stride` parts
        int last = 0;
        if (lane == 0) {
          // the warps between two first ones are inside the unit: theirs are free for the joins of joined parts
          unsigned* counter = p.counters + ((int64_t)(d.first + leader * stride + level) * 2 + (leader != 0));
          fence_gpu();  // the warp's part, behind the barrier above, comes before its arrival
          last = atomicAdd(counter, 1u) + 1 == (unsigned)count;
          if (last) *counter = 0;
          if (last) fence_gpu();
        }
        last = __shfl_sync(0xffffffffu, last, 0);
        if (!last) break;
        __syncwarp();  // what lane 0 acquired is before every lane's reads: a shuffle alone orders no memory
        const bool final = parts <= kJoin;
        // What it takes is round trips to L2, of about a microsecond: 4 pieces of 4 elements a lane (4 rows of 128) of 4 parts are
        // loaded together.
        constexpr int kQuads = hd / 4, kPieces = 4, kTogether = 4;
        const unsigned first_at = part_slot(d.first, leader * stride) * L::kRows;
        const unsigned step = (unsigned)stride * 2 * L::kRows, back = leader == 0 ? L::kRows : 0;  // a unit's first part is in a second slot
#pragma unroll 1
        for (int base = 0; base < d.rows * kQuads; base += 32 * kPieces) {  // as often for every lane: the warp meets in it
          const int x0 = base + lane;
          float top[kPieces], sum[kPieces], y[kPieces][4];
          unsigned at[kPieces];
#pragma unroll
          for (int a = 0; a < kPieces; ++a) {
            const int row = (x0 + 32 * a) / kQuads;
            at[a] = first_at + (row < d.rows ? row : 0);
            top[a] = kNone;
            sum[a] = y[a][0] = y[a][1] = y[a][2] = y[a][3] = 0.f;
          }
#pragma unroll 1
          for (int i0 = 0; i0 < count; i0 += kTogether) {
            float2 ml[kPieces][kTogether];
            float4 v[kPieces][kTogether];
#pragma unroll
            for (int k = 0; k < kTogether; ++k) {
              const int i = min(i0 + k, count - 1);
              const unsigned further = i * step - (i > 0 ? back : 0);
#pragma unroll
              for (int a = 0; a < kPieces; ++a) {
                ml[a][k] = __ldcg(p.ml + at[a] + further);
                v[a][k] = __ldcg(reinterpret_cast<const float4*>(p.acc + (at[a] + further) * hd) + x0 % kQuads);
              }
            }
#pragma unroll
            for (int a = 0; a < kPieces; ++a) {
              float high = top[a];
#pragma unroll
              for (int k = 0; k < kTogether; ++k) high = fmaxf(high, ml[a][k].x);  // the last part again where there are none left
              const float before = ex2(top[a] - high);
              top[a] = high;
              sum[a] *= before;
#pragma unroll
              for (int e = 0; e < 4; ++e) y[a][e] *= before;
#pragma unroll
              for (int k = 0; k < kTogether; ++k) {
                const float f = i0 + k < count ? ex2(ml[a][k].x - high) : 0.f;
                sum[a] = fmaf(ml[a][k].y, f, sum[a]);
                y[a][0] = fmaf(v[a][k].x, f, y[a][0]), y[a][1] = fmaf(v[a][k].y, f, y[a][1]);
                y[a][2] = fmaf(v[a][k].z, f, y[a][2]), y[a][3] = fmaf(v[a][k].w, f, y[a][3]);
              }
            }
          }
          if (!final) __syncwarp();  // a row's first m and sum are rewritten when every lane has read them
#pragma unroll
          for (int a = 0; a < kPieces; ++a) {
            const int x = x0 + 32 * a, row = x / kQuads, quad = x % kQuads;
            if (row >= d.rows) continue;
            if (final) {
              const int64_t token = d.token0 + row / p.G;
              const int head = d.kvh * p.G + row % p.G;
              float f = sum[a] == 0.f ? 0.f : 1.f / sum[a];
              if (p.c.gate && sum[a] != 0.f) f *= sigmoid(p.c.gate[token * p.c.gate_stride + head]);
              *reinterpret_cast<uint2*>(p.c.out + token * p.c.out_stride + (int64_t)head * hd + quad * 4) =
                  sum[a] == 0.f ? make_uint2(0u, 0u) : make_uint2(pack<false>(y[a][0] * f, y[a][1] * f), pack<false>(y[a][2] * f, y[a][3] * f));
              if (p.c.lse && quad == 0)
                p.c.lse[token * p.c.Hq + head] = sum[a] == 0.f ? -INFINITY : (top[a] - kShift + log2f(sum[a])) * 0.6931471805599453f;
            } else {
              __stcg(reinterpret_cast<float4*>(p.acc + at[a] * hd) + quad, make_float4(y[a][0], y[a][1], y[a][2], y[a][3]));
              if (quad == 0) __stcg(p.ml + at[a], make_float2(top[a], sum[a]));
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
  static_assert(sizeof(Round) <= L::kOffQ && L::kThreads <= 256, "a round of requests");
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

int warps_of(int rows) { return rows <= 8 ? Shape<4, 1>::kWarps : Shape<4, 2>::kWarps; }

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
  p.counters = reinterpret_cast<unsigned*>(call.workspace);
  p.acc = reinterpret_cast<float*>(call.workspace + kFewFlagBytes);
  p.ml = reinterpret_cast<float2*>(p.acc + (int64_t)ctas * warps * 2 * call.rows * call.kv.hd);
  p.status = device_status_ptr();
  if (call.kv.hd == 128) return call.rows == 8 ? launch<4, 1>(p, ctas, stream) : launch<4, 2>(p, ctas, stream);
  return call.rows == 8 ? launch<2, 1>(p, ctas, stream) : launch<2, 2>(p, ctas, stream);
}

}  // namespace q4
}  // namespace zb
