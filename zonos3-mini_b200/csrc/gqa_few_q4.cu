// Attention of few rows over a paged KV cache in 4 bits (kv_q4.cuh): the single tokens, and short drafts of them, of a decode
// batch. The mathematics is that of gqa_chunk.cu; requests of more rows are its kernel's.
//
// The rows of a request's score matrix for one KV head are its (token, head of the group) pairs, up to 8 (NT = 1) or 16. A row
// reads every code once, so the work is the codes' way from HBM and their unpacking; the products are few. So they are
// formed from registers (m16n8k16: 16 keys or dims by 8 rows), where a code goes from the loaded word into a matrix fragment
// with two instructions for two codes, and nothing is written out in between as a tensor-memory product would need it:
//   scores^T [16 keys, 8 rows] = sum over groups g of  s_g (c . q)_g + m_g (sum q)_g:  the codes themselves are the operand, as
//     128 + c in bf16 (exact), the products' sums are fp32, and the pair of a key's group goes onto them in fp32: the scores have
//     the precision of fp32;
//   out^T [16 dims, 8 rows] += V^T p^T with V = m + s c and the weights in fp16, 2^-12 of each: bf16's 2^-9 would be the largest
//     error here. fp16 has less range, so a block whose pairs are not all within it (magnitudes of 2^-10 to 2^14, or 0) takes bf16.
// A weight is 2^(score - m + 15) with m a row's reference, its largest score or up to 8 (log2) above it when it is set; it is set
// anew by a score above it, hardly ever after the first block. So weights lie in fp16's range: up to 2^15, the largest not below 2^7
// when m is set, and those below 2^-39 of m count as 0. m and the sum cancel in the end.
// The keys of a 16-key block stand in the scores' rows in the order 0 1 3 2 4 5 7 6 and 8 on: the two rows of a quarter of the lanes then
// read other banks, and the four rows that a lane's values come from too, as far as 64-byte rows allow.
//
// A warp takes one block of 16 keys at a time (at hd 128 one bulk copy of 2560 bytes), its products and its own m, sum and
// accumulator; 7 such warps are a CTA, two CTAs an SM. An eighth warp looks up pages and starts the copies, 24 blocks ahead and across
// units. The CTAs take equal runs of all units' blocks (as in gqa_chunk.cu); at the end of a unit's part the warps'
// accumulators are joined through shared memory in order, and where a unit spans CTAs the last one to arrive joins the parts
// in the order of their keys: no CTA waits for another, and results do not depend on timing.
#include <algorithm>

#include "few_q4.cuh"

namespace {

namespace q4 = zb::q4;

// Warps that compute. With the one that copies, 8 a CTA: of nine, an SM's quarter would get five of two CTAs, and a thread 96
// registers instead of 128.
constexpr int kWarps = 7;
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kCtas = 2;                        // of an SM
constexpr int kStages = 24, kDescs = 4;
constexpr int kUnitCost = 8;                    // of a unit, in blocks
constexpr int kMinShare = 16;                   // blocks of a CTA, its units' cost among them
constexpr float kAbove = 8.f, kShift = 15.f;
constexpr float kNone = -3.0e38f;               // m of a row that has seen no key

struct FewParams {
  q4::FewCall c;
  int G;
  unsigned page_mul, page_shift;  // division by the page size
  // [CTA]: the call's tag and, below it, the parts that have arrived of the unit that began there and goes on; 0 again when
  // all have. What a call whose waits gave up has left has another tag.
  unsigned* counters;
  unsigned tag;
  float* acc;                     // [CTA][2][rows][hd]
  float* ml;                      // [CTA][2][2][rows]: m, sum
  unsigned* status;
};

struct Desc {
  int token0, pos0, keys;  // first token row, its key position, keys of the request
  int rows, kvh;
  int item0, items;  // blocks here; -1: the end
  int index, parts;  // of the unit's parts, this one and their number
  int first_cta;     // where the unit's first part is
  int from;          // keys from the sinks' end to here are hidden from every row
  int all_lo, all_hi;  // keys of [all_lo, all_hi), and those below min(sinks, all_hi), are seen by every row
};

template <int GROUPS, int NT>
struct Shape {
  static constexpr int kHd = GROUPS * q4::kGroup, kBlockBytes = q4::block_bytes(kHd), kRows = 8 * NT;
  static constexpr int kJoinRow = kHd + 4;  // floats of a row in the join's buffer: rows 2 t of its writers begin 8 banks apart
  static constexpr int kOffQ = kStages * kBlockBytes;
  static constexpr int kOffJoin = kOffQ + kDescs * kRows * kHd * 2;
  static constexpr int kOffSums = kOffJoin + kWarps * 8 * kJoinRow * 4;  // the groups' sums of the queries, of a unit
  static constexpr int kOffTail = kOffSums + kWarps * GROUPS * kRows * 4;
  // The queries' fragments stay in registers, or are read again for every block where the accumulators take those.
  static constexpr bool kKeep = NT == 1;
};
struct Tail {
  uint64_t full[kStages], empty[kStages];
  uint64_t desc_full[kDescs], desc_empty[kDescs], met;
  int2 info[kStages];  // a block's first key, and how many of its keys there are
  Desc desc[kDescs];
  float m[kWarps][16], l[kWarps][16];
  int sums[2][kWarps + 1];
  int64_t start_off;
  int start_b;
  int idle[2];
  int last;
  int abort;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool HALF>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (HALF)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
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

// Whether m + s c of a pair and its neighbours keep fp16's 11 bits, or near them: the larger of |m| and 16 s lies in [2^-10, 2^14),
// or the pair is 0.
__device__ __forceinline__ bool half_holds(uint32_t pair) {
  const uint32_t a = pair & 0x7fff7fffu, top = max(a >> 16, (a & 0xffffu) + 0x200u);  // 16 s: the exponent 4 more
  return a == 0 || top - 0x3a80u < 0x4680u - 0x3a80u;
}

// A wait that gives up after about a second, and at once after any earlier one of the CTA did.
__device__ __forceinline__ bool wait(const uint64_t& bar, uint32_t parity, int* abort) {
  const uint32_t at = zb::smem_addr(&bar);
  if (zb::mbar_try_wait(at, parity)) return true;
#pragma unroll 1
  for (int i = 0; i < 250000; ++i) {
    if (zb::mbar_try_wait_sleep(at, parity, 20000u)) return true;
    if (*reinterpret_cast<volatile int*>(abort) != 0) return false;
  }
  *reinterpret_cast<volatile int*>(abort) = 1;
  return false;
}
__device__ __forceinline__ void arrive(const uint64_t& bar) { zb::mbar_arrive(zb::smem_addr(&bar)); }
// What was written to shared memory comes before the next copy over it.
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// A request's new rows (none where they are another kernel's) and its blocks of keys. Blocks from sink_blocks on are counted
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
  return r.tokens > 0 ? kUnitCost + blocks_of(p, r).n : 0;
}

// Exclusive prefix of v over the block's threads; `total` the sum. `buffer` alternates from call to call.
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
  for (int w = 0; w <= kWarps; ++w) {
    const int s = tl.sums[buffer][w];
    if (w < warp) before += s;
    total += s;
  }
  return before + in - v;
}

__device__ __forceinline__ float sigmoid(__nv_bfloat16 x) { return 1.f / (1.f + ex2(-1.4426950408889634f * __bfloat162float(x))); }

// Part `index` of a unit whose first part is CTA `first`'s: the slots are its own second one, then the first ones of the CTAs after it.
__device__ __forceinline__ int64_t part_slot(int first, int index) { return (int64_t)(first + index) * 2 + (index == 0); }

template <int GROUPS, int NT>
__global__ void __launch_bounds__(kThreads, kCtas) gqa_few_q4_kernel(const __grid_constant__ FewParams p) {
  using L = Shape<GROUPS, NT>;
  extern __shared__ __align__(128) unsigned char gbase[];
  Tail& tl = *reinterpret_cast<Tail*>(gbase + L::kOffTail);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid / 32, 0), lane = tid % 32;
  const int B = p.c.kv.B, Hkv = p.c.kv.Hkv;
  const int ctas = gridDim.x, cta = blockIdx.x;
  constexpr int hd = L::kHd;
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      zb::mbar_init(zb::smem_addr(&tl.full[s]), 1);
      zb::mbar_init(zb::smem_addr(&tl.empty[s]), 1);
    }
    for (int s = 0; s < kDescs; ++s) {
      zb::mbar_init(zb::smem_addr(&tl.desc_full[s]), 1);
      zb::mbar_init(zb::smem_addr(&tl.desc_empty[s]), kWarps);
    }
    zb::mbar_init(zb::smem_addr(&tl.met), 32 * kWarps);
    zb::fence_mbar_init();
    tl.abort = 0;
  }
  zb::pdl_enter();

  // ---- the plan: the work of all units, and where this CTA's begins
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
    const int before = block_scan(cost, tl, buffer, total);
    if (b0 == 0) {
      mine_before = before;
      mine_total = total;
    }
    work += total;
  }
  const bool refused = __syncthreads_or(out_of_order);
  const bool left_out = __syncthreads_or(more) && p.c.only;
  if (cta == 0 && tid == 0 && p.status && (refused || left_out))
    atomicOr(p.status, refused ? zb::kStatusAttnChunkBatch : zb::kStatusAttnFewRows);
  work = refused ? 0 : work * Hkv;
  const int64_t share = max((int64_t)kMinShare, (work + ctas - 1) / ctas);
  const int64_t begin = share * cta, end = min(work, begin + share);
  if (begin < end) {
    int64_t seen = 0;
#pragma unroll 1
    for (int b0 = 0; b0 < B; b0 += kThreads) {
      int cost = mine_cost, before = mine_before, total = mine_total;
      if (b0 > 0) {
        cost = b0 + tid < B ? cost_of(p, request(p, b0 + tid, more)) : 0;
        buffer ^= 1;
        before = block_scan(cost, tl, buffer, total);
      }
      const int64_t at = (seen + before) * Hkv;
      if (cost > 0 && begin >= at && begin < at + (int64_t)cost * Hkv) {
        tl.start_b = b0 + tid;
        tl.start_off = begin - at;
      }
      seen += total;
      if (begin < seen * Hkv) break;
    }
  }
  __syncthreads();
  int* abort = &tl.abort;

  if (begin >= end) {
    // nothing for this CTA
  } else if (warp == kWarps) {
    // =============================================================================================== copies
    int b = tl.start_b, item = 0, n = 0;
    bool ignored = false, going = true;
    Request req = request(p, b, ignored);
    int cost = max(cost_of(p, req), 1);
    int kvh = (int)(tl.start_off / cost), off = (int)(tl.start_off % cost);
    int64_t at = begin;
    int window0 = -1;
    Request window{};
    auto room = [&](const uint64_t& bar, uint32_t parity) {
      going = __all_sync(0xffffffffu, wait(bar, parity, abort));
      return going;
    };
    while (going && at < end) {
      const Blocks x = blocks_of(p, req);
      const int to_cost = (int)min((int64_t)cost, off + (end - at));
      const int from = max(off - kUnitCost, 0), to = max(to_cost - kUnitCost, 0);
      if (to > from || (x.n == 0 && off == 0)) {
        const int slot = n % kDescs;
        if (n >= kDescs && !room(tl.desc_empty[slot], (n / kDescs - 1) & 1)) break;
        const int64_t first = at - off + kUnitCost;  // of the unit's blocks
        if (lane == 0) {
          Desc d;
          d.token0 = req.row0;
          d.pos0 = req.keys - req.tokens;
          d.keys = req.keys;
          d.rows = req.tokens * p.G;
          d.kvh = kvh;
          d.item0 = item;
          d.items = to - from;
          d.first_cta = x.n > 0 ? (int)(first / share) : cta;
          d.index = cta - d.first_cta;
          d.parts = x.n > 0 ? (int)((first + x.n - 1) / share) - d.first_cta + 1 : 1;
          d.from = x.lo_first;
          d.all_lo = x.lo_last;
          d.all_hi = x.hi_first;
          tl.desc[slot] = d;
          zb::mbar_arrive_expect_tx(zb::smem_addr(&tl.desc_full[slot]), (uint32_t)(req.tokens * p.G * hd * 2));
        }
        __syncwarp();
        if (lane < req.tokens)  // the queries: a token's heads of the group lie side by side
          zb::bulk_g2s(zb::smem_addr(gbase + L::kOffQ + slot * (L::kRows * hd * 2) + lane * p.G * hd * 2),
                       p.c.q + (int64_t)(req.row0 + lane) * p.c.q_stride + (int64_t)kvh * p.G * hd, (uint32_t)(p.G * hd * 2),
                       zb::smem_addr(&tl.desc_full[slot]));
        ++n;
        const int held = held_keys(p, req.keys);
        const int32_t* table = p.c.kv.table + (int64_t)b * p.c.kv.table_stride;
#pragma unroll 1
        for (int j0 = from; j0 < to && going; j0 += 32) {  // a lane's block
          const int j = j0 + lane, block = j < x.sink_blocks ? j : j + x.gap, key0 = block * q4::kBlock;
          const int column = (int)(((uint64_t)(unsigned)key0 * p.page_mul) >> p.page_shift);
          const int page = j < to && key0 < held ? table[column] : -1;
          const bool there = page >= 0 && page < p.c.kv.num_pages;
          const unsigned char* src = reinterpret_cast<const unsigned char*>(p.c.kv.k) + (there ? (int64_t)page * p.c.kv.page_stride : 0) +
                                     (int64_t)kvh * p.c.kv.head_stride +
                                     (int64_t)(key0 - column * p.c.kv.page_size) / q4::kBlock * L::kBlockBytes;
          const int exist = there ? min(q4::kBlock, held - key0) : 0;
#pragma unroll 1
          for (int g = 0; g < 32 && j0 + g < to; g += 8) {  // 8 at a time: waiting for room for all would drain the ring
            const bool own = lane / 8 == g / 8 && j < to;
            const int i = item + j - from, stage = i % kStages;
            bool ready = true;
            if (own && i >= kStages) ready = wait(tl.empty[stage], (i / kStages - 1) & 1, abort);
            going = __all_sync(0xffffffffu, ready);
            if (!going) break;
            if (own) {
              tl.info[stage] = make_int2(key0, exist);
              if (there) {
                zb::mbar_arrive_expect_tx(zb::smem_addr(&tl.full[stage]), L::kBlockBytes);
                zb::bulk_g2s(zb::smem_addr(gbase + stage * L::kBlockBytes), src, L::kBlockBytes, zb::smem_addr(&tl.full[stage]));
              } else {
                arrive(tl.full[stage]);
              }
            }
            __syncwarp();
          }
        }
        item += to - from;
      }
      // ---- the next unit: KV head, then request
      at += to_cost - off;
      off = 0;
      if (at >= end) break;
      if (++kvh == Hkv) {
        kvh = 0;
        do {
          ++b;
          if (b / 32 != window0) {
            window0 = b / 32;
            const int i = window0 * 32 + lane;
            window = i < B ? request(p, i, ignored) : Request{0, 0, 0};
          }
          req.row0 = __shfl_sync(0xffffffffu, window.row0, b % 32);
          req.tokens = __shfl_sync(0xffffffffu, window.tokens, b % 32);
          req.keys = __shfl_sync(0xffffffffu, window.keys, b % 32);
        } while (b < B - 1 && req.tokens == 0);
        cost = cost_of(p, req);
        if (cost == 0) break;  // not while the lengths stay as they were when the work was added up
      }
    }
    const int slot = n % kDescs;
    if (going && (n < kDescs || room(tl.desc_empty[slot], (n / kDescs - 1) & 1))) {
      if (lane == 0) {
        tl.desc[slot].items = -1;
        arrive(tl.desc_full[slot]);
      }
      ++n;
    }
    __syncwarp();
    // nothing is in flight when the CTA's shared memory goes to another, also where a wait gave up
    if (lane < min(kStages, item))
      zb::mbar_wait_bounded(zb::smem_addr(&tl.full[lane]), (item - 1 - lane) / kStages & 1, p.status, zb::kStatusAttnChunkTimeout);
    if (lane < min(kDescs, n))
      zb::mbar_wait_bounded(zb::smem_addr(&tl.desc_full[lane]), (n - 1 - lane) / kDescs & 1, p.status, zb::kStatusAttnChunkTimeout);
  } else {
    // =============================================================================================== blocks
    const int gid = lane / 4, t4 = lane % 4;
    const int key_row = gid ^ ((gid >> 1) & 1);             // the key of scores' row gid; 8 more for row gid + 8
    const int va = 2 * t4 + (t4 & 1), vb = va ^ 1;  // the keys of rows 2 t4 and 2 t4 + 1
    int meetings = 0;
    auto meet = [&]() {  // the warps that compute; a wait with a limit, as all are
      arrive(tl.met);
      wait(tl.met, meetings & 1, abort);
      ++meetings;
    };
    for (int n = 0;; ++n) {
      const int slot = n % kDescs;
      if (!wait(tl.desc_full[slot], (n / kDescs) & 1, abort)) break;
      const Desc d = tl.desc[slot];
      if (d.items < 0) break;
      // ---- queries: B fragments, and their groups' sums
      const unsigned char* q_rows = gbase + L::kOffQ + slot * (L::kRows * hd * 2);
      float* sums = reinterpret_cast<float*>(gbase + L::kOffSums) + warp * GROUPS * L::kRows;
      auto fragment = [&](int nt, int g) {
        return 8 * nt + gid < d.rows ? *reinterpret_cast<const uint4*>(q_rows + (8 * nt + gid) * hd * 2 + (32 * g + 8 * t4) * 2)
                                     : make_uint4(0, 0, 0, 0);
      };
      uint4 q[L::kKeep ? GROUPS : 1];
      float2 qs[L::kKeep ? GROUPS : 1];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          const uint4 w = fragment(nt, g);
          float sum = low_of(w.x) + high_of(w.x) + (low_of(w.y) + high_of(w.y)) + (low_of(w.z) + high_of(w.z)) + (low_of(w.w) + high_of(w.w));
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          if (L::kKeep) {
            q[g] = w;
            qs[g].x = __shfl_sync(0xffffffffu, sum, 8 * t4);
            qs[g].y = __shfl_sync(0xffffffffu, sum, 8 * t4 + 4);
          } else if (t4 == 0) {
            sums[g * L::kRows + 8 * nt + gid] = sum;
          }
        }
      __syncwarp();
      if (L::kKeep && lane == 0) arrive(tl.desc_empty[slot]);
      // hidden keys: of the lane's rows 2 t4, 2 t4 + 1 (and 8 on)
      float m[NT][2], l[NT][2], o[NT][2 * GROUPS][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = kNone;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * GROUPS; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      }
      const int item_end = d.item0 + d.items, turn = d.item0 % kWarps;
      auto skips = [&](int w) { return w >= turn ? w - turn : w - turn + kWarps; };  // blocks before warp w's first one
#pragma unroll 1
      for (int item = d.item0 + skips(warp); item < item_end; item += kWarps) {
        const int stage = item % kStages;
        wait(tl.full[stage], (item / kStages) & 1, abort);
        const int2 info = tl.info[stage];
        unsigned char* block = gbase + stage * L::kBlockBytes;
        uint32_t* k_pairs = reinterpret_cast<uint32_t*>(block + 16 * hd);
        uint32_t* v_pairs = reinterpret_cast<uint32_t*>(block + 18 * hd);
        const int key0 = info.x;
        if (info.y < q4::kBlock || (key0 < d.from && key0 + q4::kBlock > p.c.sinks)) {
          // rows that are no keys hold anything, and what no row sees shall not choose the values' type either
          for (int i = lane; i < 16 * GROUPS; i += 32) {
            const int j = i / GROUPS, key = key0 + j;
            if (j >= info.y || (key >= p.c.sinks && key < d.from)) k_pairs[i] = v_pairs[i] = 0;
          }
          fence_proxy_async();
          __syncwarp();
        }
        bool half = true;
        {
          bool k_none = false;
#pragma unroll
          for (int i = 0; i < GROUPS / 2; ++i) {
            k_none |= q4::pair_is_none(k_pairs[lane + 32 * i]);
            half &= half_holds(v_pairs[lane + 32 * i]);
          }
          if (__any_sync(0xffffffffu, k_none)) {
#pragma unroll
            for (int i = 0; i < GROUPS / 2; ++i)
              if (q4::pair_is_none(k_pairs[lane + 32 * i])) k_pairs[lane + 32 * i] = 0;
            fence_proxy_async();
            __syncwarp();
          }
          half = __all_sync(0xffffffffu, half);
        }
        // ---- scores
        float s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
        {
          uint32_t w[2][GROUPS], pr[2][GROUPS];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const unsigned char* from = block + (key_row + 8 * h) * (hd / 2) + t4 * GROUPS * 4;
            const uint32_t* pairs = k_pairs + (key_row + 8 * h) * GROUPS;
            if constexpr (GROUPS == 4) {
              *reinterpret_cast<uint4*>(w[h]) = *reinterpret_cast<const uint4*>(from);
              *reinterpret_cast<uint4*>(pr[h]) = *reinterpret_cast<const uint4*>(pairs);
            } else {
              *reinterpret_cast<uint2*>(w[h]) = *reinterpret_cast<const uint2*>(from);
              *reinterpret_cast<uint2*>(pr[h]) = *reinterpret_cast<const uint2*>(pairs);
            }
          }
#pragma unroll
          for (int g = 0; g < GROUPS; ++g) {
            const uint32_t a[2][4] = {{q4::codes_128<0>(w[0][g]), q4::codes_128<1>(w[0][g]), q4::codes_128<2>(w[0][g]), q4::codes_128<3>(w[0][g])},
                                      {q4::codes_128<0>(w[1][g]), q4::codes_128<1>(w[1][g]), q4::codes_128<2>(w[1][g]), q4::codes_128<3>(w[1][g])}};
            const float s0 = low_of(pr[0][g]), s1 = low_of(pr[1][g]);
            const float m0 = fmaf(-128.f, s0, high_of(pr[0][g])), m1 = fmaf(-128.f, s1, high_of(pr[1][g]));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float dot[4] = {0.f, 0.f, 0.f, 0.f};
              const uint4 f = L::kKeep ? q[g] : fragment(nt, g);
              const float2 sum = L::kKeep ? qs[g] : *reinterpret_cast<const float2*>(sums + g * L::kRows + 8 * nt + 2 * t4);
              mma<false>(dot, a[0][0], a[1][0], a[0][1], a[1][1], f.x, f.y);
              mma<false>(dot, a[0][2], a[1][2], a[0][3], a[1][3], f.z, f.w);
              s[nt][0] = fmaf(s0, dot[0], fmaf(m0, sum.x, s[nt][0]));
              s[nt][1] = fmaf(s0, dot[1], fmaf(m0, sum.y, s[nt][1]));
              s[nt][2] = fmaf(s1, dot[2], fmaf(m1, sum.x, s[nt][2]));
              s[nt][3] = fmaf(s1, dot[3], fmaf(m1, sum.y, s[nt][3]));
            }
          }
        }
        if (info.y < q4::kBlock || key0 + q4::kBlock > d.all_hi || (key0 < d.all_lo && key0 + q4::kBlock > p.c.sinks)) {
          const int held = held_keys(p, d.keys);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int row = 8 * nt + 2 * t4 + e, pos = d.pos0 + min(row, d.rows - 1) / p.G;
              const int lo = first_seen(p, pos), hi = behind_seen(p, held, pos);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int j = key_row + 8 * h, key = key0 + j;
                if (j >= info.y || key >= hi || (key < lo && key >= p.c.sinks)) s[nt][2 * h + e] = -INFINITY;
              }
            }
        }
        // ---- weights
        float e[NT][4];
        bool above = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[nt][i] = fmaf(s[nt][i], p.c.scale_log2, kShift - m[nt][i % 2]);
            above |= e[nt][i] > kShift;
          }
        if (__any_sync(0xffffffffu, above)) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float top = fmaxf(s[nt][r], s[nt][2 + r]) * p.c.scale_log2;
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
              for (int h = 0; h < 2; ++h) e[nt][2 * h + r] = fmaf(s[nt][2 * h + r], p.c.scale_log2, kShift - m[nt][r]);
            }
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int i = 0; i < 4; ++i) e[nt][i] = ex2(e[nt][i]);
          l[nt][0] += e[nt][0] + e[nt][2];
          l[nt][1] += e[nt][1] + e[nt][3];
        }
        // ---- values
        auto values = [&](auto type) {
          constexpr bool HALF = decltype(type)::value;
          uint32_t pb[NT][2];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            pb[nt][0] = transpose8(pack<HALF>(e[nt][0], e[nt][1]));
            pb[nt][1] = transpose8(pack<HALF>(e[nt][2], e[nt][3]));
          }
          constexpr int W = GROUPS / 2;  // words of a key here
          uint32_t w[4][W], pr[4][W];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = (k % 2 ? vb : va) + 8 * (k / 2);
            const unsigned char* from = block + 8 * hd + row * (hd / 2) + gid * W * 4;
            const uint32_t* pairs = v_pairs + row * GROUPS + (gid * W) % GROUPS;
            if constexpr (W == 2) {
              *reinterpret_cast<uint2*>(w[k]) = *reinterpret_cast<const uint2*>(from);
              *reinterpret_cast<uint2*>(pr[k]) = *reinterpret_cast<const uint2*>(pairs);
            } else {
              w[k][0] = *reinterpret_cast<const uint32_t*>(from);
              pr[k][0] = *pairs;
            }
            if constexpr (!HALF)
#pragma unroll
              for (int i = 0; i < W; ++i) pr[k][i] = q4::pair_is_none(pr[k][i]) ? 0u : pr[k][i];
          }
          // codes of two keys beside each other: nibbles 0-3 and 4-7 of each word; and the keys' s and m
          uint32_t part[2][W][2], s2[2][W], m2[2][W];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < W; ++i) {
              part[h][i][0] = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x5410);
              part[h][i][1] = __byte_perm(w[2 * h][i], w[2 * h + 1][i], 0x7632);
              if constexpr (HALF) {
                s2[h][i] = pack<true>(low_of(pr[2 * h][i]), low_of(pr[2 * h + 1][i]));
                m2[h][i] = pack<true>(high_of(pr[2 * h][i]), high_of(pr[2 * h + 1][i]));
              } else {
                s2[h][i] = __byte_perm(pr[2 * h][i], pr[2 * h + 1][i], 0x5410);
                m2[h][i] = __byte_perm(pr[2 * h][i], pr[2 * h + 1][i], 0x7632);
              }
            }
          auto value = [&](uint32_t codes, uint32_t sc, uint32_t mn) {
            if constexpr (HALF) {
              const uint32_t c = codes | 0x64006400u, k1024 = 0x64006400u;  // 1024 + c
              const __half2 x = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), *reinterpret_cast<const __half2*>(&k1024)),
                                        *reinterpret_cast<const __half2*>(&sc), *reinterpret_cast<const __half2*>(&mn));
              return *reinterpret_cast<const uint32_t*>(&x);
            } else {
              return q4::stands_for(codes | 0x43004300u, sc, mn);
            }
          };
#pragma unroll
          for (int i = 0; i < 2 * GROUPS; ++i) {
            // rows gid and gid + 8 of the product: nibble i of the lane's two words, or nibbles i and i + 4 of its one
            const int x0 = 0, x1 = W - 1, n0 = i, n1 = W == 2 ? i : i + 4;
            const uint32_t a0 = value((part[0][x0][n0 / 4] >> (4 * (n0 % 4))) & 0x000f000fu, s2[0][x0], m2[0][x0]);
            const uint32_t a1 = value((part[0][x1][n1 / 4] >> (4 * (n1 % 4))) & 0x000f000fu, s2[0][x1], m2[0][x1]);
            const uint32_t a2 = value((part[1][x0][n0 / 4] >> (4 * (n0 % 4))) & 0x000f000fu, s2[1][x0], m2[1][x0]);
            const uint32_t a3 = value((part[1][x1][n1 / 4] >> (4 * (n1 % 4))) & 0x000f000fu, s2[1][x1], m2[1][x1]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma<HALF>(o[nt][i], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
        };
        if (half) values(std::true_type{});
        else values(std::false_type{});
        __syncwarp();
        if (lane == 0) arrive(tl.empty[stage]);
      }
      __syncwarp();
      if (!L::kKeep && lane == 0) arrive(tl.desc_empty[slot]);
      // ---- the warps' accumulators together
      const bool whole = d.parts == 1;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (8 * nt >= d.rows) break;
        float* join = reinterpret_cast<float*>(gbase + L::kOffJoin);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float sum = l[nt][r];
#pragma unroll
          for (int w = 4; w < 32; w *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, w);
          if (gid == 0) {
            tl.m[warp][8 * nt + 2 * t4 + r] = m[nt][r];
            tl.l[warp][8 * nt + 2 * t4 + r] = sum;
          }
        }
        const bool any = d.items > skips(warp);  // the warp had a block
        if (any && 8 * nt + 2 * t4 < d.rows)
#pragma unroll
          for (int i = 0; i < 2 * GROUPS; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) join[(warp * 8 + 2 * t4 + r % 2) * L::kJoinRow + 16 * i + gid + 8 * (r / 2)] = o[nt][i][r];
        meet();
        // a thread takes 4 elements of a row: element e of word w lies in nibble e / 2 + 4 (e % 2) of it
        constexpr int kQuads = hd / 4;
        for (int x = tid; x < 8 * kQuads; x += 32 * kWarps) {
          const int row = 8 * nt + x / kQuads, quad = x % kQuads, word = quad / 2;
          if (row >= d.rows) break;
          int at[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int nibble = (quad % 2 * 4 + e) / 2 + 4 * (e % 2);
            at[e] = GROUPS == 4 ? 16 * nibble + word / 2 + 8 * (word % 2) : 16 * (nibble % 4) + word + 8 * (nibble / 4);
          }
          float top = kNone;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, tl.m[w][row]);
          float sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            if (d.items <= skips(w)) continue;
            const float f = ex2(tl.m[w][row] - top);
            sum = fmaf(tl.l[w][row], f, sum);
            const float* from = join + (w * 8 + x / kQuads) * L::kJoinRow;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = fmaf(from[at[e]], f, y[e]);
          }
          // the quad's dims: word t * GROUPS + g holds 32 g + 8 t on
          const int dim = 32 * (word % GROUPS) + 8 * (word / GROUPS) + quad % 2 * 4;
          if (whole) {
            const int64_t token = d.token0 + row / p.G;
            const int head = d.kvh * p.G + row % p.G;
            float f = sum == 0.f ? 0.f : 1.f / sum;
            if (p.c.gate && sum != 0.f) f *= sigmoid(p.c.gate[token * p.c.gate_stride + head]);
            uint2 w;
            w.x = sum == 0.f ? 0u : pack<false>(y[0] * f, y[1] * f);
            w.y = sum == 0.f ? 0u : pack<false>(y[2] * f, y[3] * f);
            *reinterpret_cast<uint2*>(p.c.out + token * p.c.out_stride + (int64_t)head * hd + dim) = w;
            if (p.c.lse && quad == 0)
              p.c.lse[token * p.c.Hq + head] = sum == 0.f ? -INFINITY : (top - kShift + log2f(sum)) * 0.6931471805599453f;
          } else {
            const int64_t part = part_slot(d.first_cta, d.index);
            __stcg(reinterpret_cast<float4*>(p.acc + (part * p.c.rows + row) * hd + dim), make_float4(y[0], y[1], y[2], y[3]));
            if (quad == 0) {
              __stcg(p.ml + part * 2 * p.c.rows + row, sum == 0.f ? kNone : top);
              __stcg(p.ml + (part * 2 + 1) * p.c.rows + row, sum);
            }
          }
        }
        if (!whole) __threadfence();
        meet();  // the buffer is free, the part is written
      }
      if (!whole) {
        if (tid == 0) {
          unsigned* counter = p.counters + d.first_cta;
          unsigned old = *reinterpret_cast<volatile unsigned*>(counter), seen, arrived;
          do {
            seen = old;
            arrived = (seen >> 12 == p.tag ? seen & 0xfffu : 0u) + 1;
            old = atomicCAS(counter, seen, arrived == (unsigned)d.parts ? 0u : p.tag << 12 | arrived);
          } while (old != seen);
          tl.last = arrived == (unsigned)d.parts;
          __threadfence();
        }
        meet();
        if (tl.last) {
          constexpr int kQuads = hd / 4, kTogether = 8;
          for (int x = tid; x < d.rows * kQuads; x += 32 * kWarps) {
            const int row = x / kQuads, quad = x % kQuads;
            float top = kNone, sum = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
            for (int i0 = 0; i0 < d.parts; i0 += kTogether) {
              float pm[kTogether], pl[kTogether], high = top;
              float4 v[kTogether];
#pragma unroll
              for (int k = 0; k < kTogether; ++k) {
                const bool there = i0 + k < d.parts;
                const int64_t part = part_slot(d.first_cta, there ? i0 + k : 0);
                pm[k] = there ? __ldcg(p.ml + part * 2 * p.c.rows + row) : kNone;
                pl[k] = there ? __ldcg(p.ml + (part * 2 + 1) * p.c.rows + row) : 0.f;
                v[k] = there ? __ldcg(reinterpret_cast<const float4*>(p.acc + (part * p.c.rows + row) * hd + quad * 4))
                             : make_float4(0.f, 0.f, 0.f, 0.f);
              }
#pragma unroll
              for (int k = 0; k < kTogether; ++k) high = fmaxf(high, pm[k]);
              const float before = ex2(top - high);
              top = high;
              sum *= before;
#pragma unroll
              for (int e = 0; e < 4; ++e) y[e] *= before;
#pragma unroll
              for (int k = 0; k < kTogether; ++k) {
                const float f = ex2(pm[k] - top);
                sum = fmaf(pl[k], f, sum);
                y[0] = fmaf(v[k].x, f, y[0]), y[1] = fmaf(v[k].y, f, y[1]);
                y[2] = fmaf(v[k].z, f, y[2]), y[3] = fmaf(v[k].w, f, y[3]);
              }
            }
            const int64_t token = d.token0 + row / p.G;
            const int head = d.kvh * p.G + row % p.G;
            float f = sum == 0.f ? 0.f : 1.f / sum;
            if (p.c.gate && sum != 0.f) f *= sigmoid(p.c.gate[token * p.c.gate_stride + head]);
            uint2 w;
            w.x = sum == 0.f ? 0u : pack<false>(y[0] * f, y[1] * f);
            w.y = sum == 0.f ? 0u : pack<false>(y[2] * f, y[3] * f);
            *reinterpret_cast<uint2*>(p.c.out + token * p.c.out_stride + (int64_t)head * hd + quad * 4) = w;
            if (p.c.lse && quad == 0)
              p.c.lse[token * p.c.Hq + head] = sum == 0.f ? -INFINITY : (top - kShift + log2f(sum)) * 0.6931471805599453f;
          }
        }
        meet();  // tl.last has been read
      }
    }
  }
  // ---- rows of no request, where no other kernel takes them
  if (p.c.only && !refused) {
    const int idle = tl.idle[0] + p.c.kv.N - tl.idle[1];
#pragma unroll 1
    for (int i = cta * (kWarps + 1) + warp; i < idle; i += ctas * (kWarps + 1)) {
      const int64_t t = i < tl.idle[0] ? i : tl.idle[1] + i - tl.idle[0];
#pragma unroll 1
      for (int c = lane; c < p.c.Hq * hd / 8; c += 32)
        *reinterpret_cast<uint4*>(p.c.out + t * p.c.out_stride + c * 8) = make_uint4(0, 0, 0, 0);
      if (p.c.lse)
#pragma unroll 1
        for (int h = lane; h < p.c.Hq; h += 32) p.c.lse[t * p.c.Hq + h] = -INFINITY;
    }
  }
  __syncthreads();
  if (tid == 0 && *abort != 0 && p.status) atomicOr(p.status, zb::kStatusAttnChunkTimeout);
}

template <int GROUPS, int NT>
int launch(FewParams& p, int ctas, cudaStream_t stream) {
  auto kernel = gqa_few_q4_kernel<GROUPS, NT>;
  constexpr int kSmem = Shape<GROUPS, NT>::kOffTail + (int)sizeof(Tail);
  static_assert(kSmem * kCtas <= 227 * 1024, "shared memory");
  static bool configured[64] = {false};  // the shared-memory attribute, set once per device
  int dev = 0;
  ZB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    ZB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  ZB_CUDA(zb::launch(kernel, dim3((unsigned)ctas), dim3(kThreads), (size_t)kSmem, stream, 1, p));
  return zb::check_launch("gqa_chunk_q4");
}

int ctas_of() { return (int)std::min<int64_t>((int64_t)zb::sm_count() * kCtas, q4::kFewFlagBytes / 4); }

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

int64_t few_workspace_bytes(int B, int N, int Hkv, int hd, int rows) {
  if (rows == 0 || B < 1 || N < 1) return 0;
  return kFewFlagBytes + (int64_t)ctas_of() * 2 * rows * (hd + 2) * 4;
}

int launch_few(const FewCall& call, cudaStream_t stream) {
  FewParams p;
  p.c = call;
  p.G = call.Hq / call.kv.Hkv;
  unsigned l = 0;
  while ((1u << l) < (unsigned)call.kv.page_size) ++l;
  p.page_shift = 31 + l;
  p.page_mul = (unsigned)((((uint64_t)1 << p.page_shift) + call.kv.page_size - 1) / call.kv.page_size);
  const int ctas = ctas_of();
  static std::atomic<unsigned> calls{0};
  do p.tag = (calls.fetch_add(1, std::memory_order_relaxed) + 1) & 0xfffffu;
  while (p.tag == 0);
  p.counters = reinterpret_cast<unsigned*>(call.workspace);
  p.acc = reinterpret_cast<float*>(call.workspace + kFewFlagBytes);
  p.ml = p.acc + (int64_t)ctas * 2 * call.rows * call.kv.hd;
  p.status = device_status_ptr();
  if (call.kv.hd == 128) return call.rows == 8 ? launch<4, 1>(p, ctas, stream) : launch<4, 2>(p, ctas, stream);
  return call.rows == 8 ? launch<2, 1>(p, ctas, stream) : launch<2, 2>(p, ctas, stream);
}

}  // namespace q4
}  // namespace zb
