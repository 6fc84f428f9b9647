// Attention of every request's new tokens over its pages of a KV cache.
//
// Token t of request b at key position p (paged.cuh) sees the keys j <= p (causal; every key of the request otherwise)
// with j > p - window (or j < sinks) when there is a window, and whose page is in the cache. With s_j = scale q . k_j over them,
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  lse = m + log sum_j e^(s_j - m),  m = max_j s_j;
// a token that sees no key, or belongs to no request, gives 0 (lse -inf). Query head h reads KV head h / (Hq / Hkv).
// The layer's output gate multiplies head h's row by sigmoid(gate[t, h]) before the one rounding to bf16.
//
// Both products run on the tensor cores. The G = Hq / Hkv heads of a KV head share its keys, so the rows of a
// request's score matrix are its (token, head of the group) pairs, token-major; a unit of work is 256 such rows of one
// (request, KV head), as two streams of 128 rows (the lanes of tensor memory), against a range of 128-key tiles. Per
// stream and tile: S = Q K^T (tcgen05, fp32 in tensor memory); a thread takes a row, finds its maximum, forms p = 2^(s
// scale log2 e - m), adds up its sum in fp32 and writes p back over S as bf16; O += P V with P read from tensor memory.
// The two streams share each tile's K and V in shared memory and take turns: one's exponentials run while the tensor
// cores work for the other. The subtracted m cancels in the final division, so it need not be the maximum: it lies at it
// or up to 24 (log2) above it, and moves to 24 above a tile's largest score when that is larger than m. So no p is above 1, as
// with the maximum itself: the accumulator stays below sum |v_j|, and no finite values overflow that do not with the maximum;
// and the largest p is at least 2^-24, so that weights below 2^-102 of it count as 0, and values down to 2^-100 keep their
// precision. m starts at 24, which holds for first keys whose largest score is 0 to 12 (for larger ones it would be reached
// too soon). So the search for the maximum runs beside the exponentials instead of before them, and the accumulator is hardly
// ever rescaled: 4 x 512 tokens behind 8192 take 131 us with scores that spread by 1 nat, 134 by 4, 141 by 8, 190 by 16.
// p is rounded to bf16 because the tensor cores multiply bf16; its sum is kept from before the rounding. Where that would
// be the largest error for nothing it is avoided: units of few rows multiply what the rounding left off too, and rows whose
// first keys lie in a partly visible tile start with m 24 above their largest score, whose p is 2^-24 and exact.
//
// The lengths live on the device, so the split of the work does too: every CTA adds up the tiles of all units (a scan
// over the requests) and takes an equal run of them. A unit that spans CTAs leaves partial results (accumulator,
// maximum, sum) in the workspace, and the CTA where it began joins them in order (the others hand theirs over as the
// first thing they do); so one token over a long cache uses the whole GPU, a ragged batch is balanced whatever its
// lengths, and the result does not depend on timing.
//
// Warps: 0-3 and 4-7 the rows of stream 0 and 1; 8 issues the tensor-core work; 9-11 look up pages and copy K, V and Q
// rows (any page size, any strides) into shared memory, several tiles ahead and across units (9-15 for 4 bits, below).
//
// A key hidden from some rows of a tile must not reach them even when its value is not finite, and 0 x inf is NaN in a
// matrix product. So where a tile's keys are visible to some of its rows only, warps 10 and 11 look through the V tile while
// the scores are being worked on; values that are not finite are added to the rows that see them one by one, then zeroed.
//
// What bounds it, and what it measured (B200, 16 query and 4 KV heads of 128; calls one after the other without end, and in
// brackets bursts of 20 captured calls, before the power limit lowers the clock):
// * A long prompt (8192 tokens, causal; 275 GFLOP): 278 us, 988 TFLOP/s (231 us, 1190), 0.60 (0.73) of the 1638 that a library
//   product of 8192^3 reaches in a burst. Per stream and tile the chain scores (512 cycles), weights (1024 of the exponential
//   unit, 2048 with the other stream's beside them), hand-over, values' product (its second half 256) comes to 3100-3500
//   cycles for two tiles' 2048 cycles of tensor-core work; without the row warps' work the loop takes 195 us. At the power
//   limit the clock falls from 1.95 to 1.62 GHz. 4 x 512 tokens behind 8192 cached ones (142 GFLOP): 156 us, 908 TFLOP/s (131).
// * Single tokens are bound by HBM and power: 256 requests of 1628 keys (856 MB), 171 us, 5.0 TB/s, 0.78 of a copy's 6.46
//   (153 us, 0.87); 2 of 65000 keys over all CTAs, 57 us, 4.7 TB/s. Products 64 rows high for the 4 rows of a token are what
//   takes the power; with pages of one row the decode kernel, whose products are 16 wide, takes 155 us and this one 237.
// * Many short units (256 prompts of up to 128 tokens) are bound by the latency of a unit's steps, 8000-10000 cycles,
//   and by their balance, not by bytes (26 us of them): 72 us. Each unit runs through about 30 KB of code once, more than
//   the instruction cache keeps beside the other warps' (a fifth of its requests miss at the present 147 KB of kernel). So code
//   that runs once a unit is kept small before it is kept fast: loops over 32 keys or dims instead of whole rows (unrolled
//   whole, the epilogue made it 75 -> 79 us), one place for each stream's products (70.7 -> 69.2), waits that count (73.7 ->
//   70.7).
// * One request of one token: 15 us, about 7 of them the way from the launch to the first scores.
//
// Pages: with rows of 64 or 128 elements and a page size with a factor of 8 or more, a lane copies a page's rows in one
// tensor copy; 16-byte copies by three warps otherwise. On 128 requests of 2000 keys and pages of 8 the first takes 125 us
// against 158 with heads of 128, 120 against 120 with heads of 64. The 16-byte copies cost most on pages of one row: the 4 x 512
// tokens take 199 us, the prompts 84; and where a head dim is padded: 96 dims 192 us for the 4 x 512 tokens, 32 dims 180 us for
// 256 single tokens, more than 64 dims do (115, 127).
//
// First keys that stay visible (SINKS): with a window, keys j < sinks are seen too. A unit's tiles are then those of the sinks
// and those from its first row's window on; nothing between them is read. Kernels without it keep their registers: one kernel
// for both spilled. A prompt of 8192 with a window of 1024 and 4 first keys (65 GFLOP) takes 106 us, the whole
// prompt without a window 270; 64 single tokens behind 16383 keys 41 us.
//
// A cache in 4 bits (Q4, kv_q4.cuh): the same two products, so keys and values have to lie as 16-bit numbers where the tensor
// cores read them. Warp 9 copies blocks of 16 keys as they are, 64 keys a stage, three stages ahead (a bulk copy each); warps
// 10-12 write out a tile's keys and 13-15 its values. The row warps and these share the registers 184 to 72 a thread. Keys are
// bf16 as the queries are; values and weights are fp16 in every block of 16 keys that fp16 holds (else bf16): errors on
// 4 x 512 tokens behind 8192 are 0.0023 of the outputs' norm, with bf16 0.0032, the plain form's 0.0017. The rows wait for a tile's
// values before they form its weights, which costs 177 us for 160 there; with 12 warps a CTA, three for all of this, it was 277.
// What is left above the bf16 cache's 146 us is the row warps' slots, of which six more warps take half, and that wait.
// fp16's range asks for an m nearer to the largest score than bf16's (kAboveQ4), so wider scores set it anew more often: 4 x 512
// tokens over 8704 keys 192 us with scores that spread by 1 nat, 215 by 4, 223 by 16 (193, 195 and 219 with bf16's distance). Scores
// beyond 2^22 (log2) are past what fp32 resolves within it.
// Requests of few rows are gqa_few_q4.cu's: a product of 64 rows for the 4 of a token would cost what reading less gains.
#include <algorithm>

#include "few_q4.cuh"
#include "tc.cuh"
#include "tc_pair.cuh"

namespace {

namespace tc = zb::tc;

constexpr int kTile = 128;       // keys of a tile
constexpr int kStreamRows = 128;  // rows of a stream
// What a unit and each of its tiles cost, in fifths of a tile of one stream of rows: 1 for such a unit, 2 for one of two
// streams. Of eight sets around the measured times the one that is within 3 % of the best on every batch.
constexpr int kUnitCost1 = 14, kTileCost1 = 5, kUnitCost2 = 20, kTileCost2 = 7;
constexpr int kFewRows = 32;     // up to here the row warps share a unit's rows in joining its parts
// Up to here a unit's rows are lanes 0-15 of products that are 64 rows high instead of 128, and a thread takes 64 of two
// rows' scores. The time of a product hardly matters with so few rows, so a second one takes what rounding a weight to bf16
// leaves off, which leaves 2^-16 of a weight instead of 2^-8: the output of single tokens is then as good as fp32's, 0.0017 of
// its norm from the exact one (its own rounding) instead of 0.0023. The second product costs 256 single tokens over 1628 keys
// 149 -> 152 us, 161 -> 168 where the GPU is held by its power limit (before it, products of 64 rows instead of 128 had taken
// that time from 181 to 167 on another GPU).
constexpr int kFineRows = 16;
constexpr int kSoftWarps = 8, kMmaWarp = 8, kLoadWarp = 9, kLoadWarps = 3;
constexpr int kThreads = 32 * (kLoadWarp + kLoadWarps);
// 4 bits: three warps write out the keys and three the values, which with the products' and the copies' warp are two warpgroups.
constexpr int kOutWarps = 3, kThreadsQ4 = 32 * (kLoadWarp + 1 + 2 * kOutWarps);
constexpr int kMaxSlots = 10, kDescs = 4;
// 4 bits: stages of 64 keys (their values too) as they lie in the cache, which six warps write out as tiles of 16-bit numbers.
constexpr int kRawStages = 3, kRawBlocks = 4;
constexpr int kMasks = 8;  // of key masks and of looked-through tiles: the loaders run at most 5 tiles ahead of the rows
// How far (log2) the m that is subtracted may lie above a row's largest score, and how far a unit's first m has to lie above it.
constexpr float kAbove = 24.f, kRoom = 12.f;
// 4 bits: the weights come 2^15 larger, so that fp16, whose rounding is an eighth of bf16's, holds them. m lies at most 8 above the
// largest score, so a row's largest weight is 2^7 to 2^15, weights are rounded as fp16 does down to 2^-21 of it (2^-14), and what
// they lack below that is 2^-32 of it a key: 2^-12 at a million keys. With 24, keys 11 nats below a first one that stands out were gone.
// They are summed before they are rounded: that takes no instruction, and the roundings above 2^-21 have either sign.
constexpr float kAboveQ4 = 8.f, kRoomQ4 = 2.f, kShiftQ4 = 15.f;
constexpr int kMaxRequests = 16384;
// The flags' part of a workspace, of every call's alike: calls of different grids take turns on one workspace, and what one
// leaves in its parts must not lie where another has its flags.
constexpr int64_t kFlagBytes = 4096;

// n / d and n % d for 0 <= n < 2^31 by a multiplication: m = ceil(2^(31 + l) / d) with 2^l >= d.
struct Divisor {
  unsigned d, m, shift;
  __host__ void set(int by) {
    unsigned l = 0;
    while ((1u << l) < (unsigned)by) ++l;
    d = (unsigned)by;
    shift = 31 + l;
    m = (unsigned)((((uint64_t)1 << shift) + d - 1) / d);
  }
  __device__ __forceinline__ int quotient(int n) const { return (int)(((uint64_t)(unsigned)n * m) >> shift); }
  __device__ __forceinline__ int rest(int n) const { return n - quotient(n) * (int)d; }
};

struct ChunkParams {
  zb::PagedBatch kv;
  Divisor by_page, by_group, by_pair;  // page size, G, tokens of a pair of streams
  const __nv_bfloat16* q;  // [N, Hq, hd], row stride q_stride
  int64_t q_stride;
  int Hq, G;
  int tokens;  // of a stream: kStreamRows / G
  float scale_log2;  // softmax scale * log2(e)
  int causal, window, sinks;
  int few;  // requests of up to so many rows (more than 0) are another kernel's
  const __nv_bfloat16* gate;  // [N, Hq] or null
  int64_t gate_stride;
  __nv_bfloat16* out;  // [N, Hq, hd]
  int64_t out_stride;
  float* lse;  // [N, Hq] or null
  // workspace: per CTA a flag (raised to the call's `raised`, put back to 0 by the CTA that waited for it) and two slots of
  // partial results, rows_max rows each: of the unit that began before this CTA, and of the one that goes on after it
  unsigned* flags;
  unsigned raised;  // of every call another, so that a flag left by a call whose waits gave up is no other call's
  float* acc;  // [CTA][2][HD / 4][rows_max][4]
  float* ml;   // [CTA][2][2][rows_max]: maximum, sum
  int rows_max;
  unsigned* status;
  int box, box_shift;  // rows of a page that one tensor copy brings; 0: K and V rows come by 16-byte copies
  int head_atoms, page_heads;  // a KV head's atom offset, and a page's index step, in the tensor maps
};
struct Maps {
  CUtensorMap q, k, v;
};

// What a CTA does with one unit.
struct Desc {
  int token0;     // the unit's first token row
  int pos0;       // and its key position
  int keys;       // of the request (not negative)
  int rows;       // (token, head) rows
  int kvh;
  int tile0, tiles;  // tiles of keys; 0: no row sees a key
  int sink_tiles, gap;  // tiles from sink_tiles on are counted without the `gap` tiles that lie between sinks and window
  int from;             // keys from the sinks' end to here are hidden from every row
  int mode;          // kFinal, kPart0, kPart1, kStop
  int parts;
  int all_lo, all_hi;  // no key of [all_lo, all_hi) is hidden from some row (a key the request does not have is a zero)
};
enum Mode { kFinal = 0, kPart0 = 1, kPart1 = 2, kStop = 3 };

struct Tail {
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  uint64_t q_full[2], q_empty[2];
  uint64_t s_full[2], p_half[2], p_full[2], o_full[2];
  uint64_t armed[kMasks], scanned[kMasks], drained, halves;  // with 4 bits, armed: a stage is there; scanned: it is free
  uint64_t desc_full[kDescs], desc_empty[kDescs];
  alignas(16) unsigned mask[kMasks][4];  // keys of a tile that exist
  Desc desc[kDescs];
  int idle[2];        // rows of no request: those before the first, those from the second on
  int start[5];       // this CTA's first unit: request, its row, tokens and keys, and the pair of streams
  int64_t start_off;  // how far into the pair's work, all KV heads, the CTA begins
  float ml[2][kStreamRows][2];  // maximum and sum of the rows' two halves, when the streams share rows
  uint32_t tmem;
  int abort;
  int found[kMasks][2];  // either half of the tile's values holds some that are not finite; with 4 bits a byte for each block, 1: bf16
};

template <int HD, bool Q4 = false>
struct Shape {
  // A tile of 128 rows: 8 rows x 64 dims (128 swizzled bytes each) are an atom; an 8-row group's atoms lie together, so
  // that one tensor copy of whole rows of a page, of any multiple of 8, lands in place.
  static constexpr uint32_t kGroup = HD / 64 * 1024;
  static constexpr uint32_t kItem = kTile / 8 * kGroup;
  static constexpr uint32_t kQAtom = kStreamRows * 128;  // the queries lie dims apart: 64 dims of all rows, then the next
  static constexpr int kSlots = Q4 ? (HD == 128 ? 4 : 6) : HD == 128 ? 5 : 10;
  static constexpr uint32_t kRaw = Q4 ? kRawBlocks * zb::q4::block_bytes(HD) : 0;  // a stage
  static constexpr uint32_t kOffQ = kSlots * kItem;
  static constexpr uint32_t kOffRaw = kOffQ + 2 * kItem;
  static constexpr uint32_t kOffTail = kOffRaw + kRawStages * kRaw;
  static constexpr size_t kSmem = kOffTail + sizeof(Tail);
  static constexpr int kThreads = Q4 ? kThreadsQ4 : ::kThreads;
  static_assert(kSlots * kItem >= kMaxRequests * 4 + kThreads * 16, "the plan's tables fit the ring");
  static_assert(kSmem <= 232448, "shared memory");
  static constexpr uint32_t kColS = 0, kColO = 2 * kTile;  // stream s: S at s * 128, O at 256 + s * HD
};

// Byte offset of 16-byte piece c of row r in a tile.
template <int HD>
__device__ __forceinline__ uint32_t piece(int r, int c) {
  return (uint32_t)(r / 8) * Shape<HD>::kGroup + (uint32_t)(c / 8) * 1024 + tc::sw128(r % 8, c % 8);
}

// Rows of a page, of one KV head: a box of 64 dims x 8 rows x atoms x row groups.
__device__ __forceinline__ void load_rows(uint32_t dst, const CUtensorMap* map, int atom, int group, int page, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(0), "r"(atom), "r"(group), "r"(page), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void load_queries(uint32_t dst, const CUtensorMap* map, int dim, int head, int token,
                                             uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(dim), "r"(head), "r"(token), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
// Arrives on `bar` once every cp.async this thread issued before has completed (counts as one expected arrival).
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// D[tmem] (+)= A[tmem] B[smem]
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// 16 columns of 16 lanes (of those from taddr's on): thread T gets, for block b of 8 columns, columns 2 (T % 4), + 1 of
// lane T / 4 in r[4 b], r[4 b + 1] and of lane T / 4 + 8 in the next two.
__device__ __forceinline__ void ld_across(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}
// 16 rows' 128 columns: thread T gets, for block b of 8, columns 2 (T % 4), + 1 of row T / 4 in r[4 b], r[4 b + 1] and of
// row T / 4 + 8 in the next two.
__device__ __forceinline__ void ld_fine(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                 "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                 "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                 "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
                 "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
                 "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
                 "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
                 "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr));
}
// 16 rows' 64 columns: thread T's r[2 b] goes to column 4 b + T % 4 of row T / 4, r[2 b + 1] to the row 8 further.
__device__ __forceinline__ void st_fine(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
      "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// What threads 4 r of the warp hold of rows r and r + 8, for the lane's row.
__device__ __forceinline__ float of_row(float a, float b, int lane) {
  const float x = __shfl_sync(0xffffffffu, a, 4 * (lane % 8)), y = __shfl_sync(0xffffffffu, b, 4 * (lane % 8));
  return lane & 8 ? y : x;
}
__device__ __forceinline__ uint32_t ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr));
  return r;
}
__device__ __forceinline__ void st1(uint32_t taddr, uint32_t r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(r) : "memory");
}
// A value that is the same on every lane, told to the compiler: it and what follows from it stay in uniform registers,
// which the tensor-core instructions take their operands from.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ Desc uniform(const Desc& d) {
  Desc u;
  u.token0 = uniform(d.token0);
  u.pos0 = uniform(d.pos0);
  u.keys = uniform(d.keys);
  u.rows = uniform(d.rows);
  u.kvh = uniform(d.kvh);
  u.tile0 = uniform(d.tile0);
  u.tiles = uniform(d.tiles);
  u.sink_tiles = uniform(d.sink_tiles);
  u.gap = uniform(d.gap);
  u.mode = uniform(d.mode);
  u.parts = uniform(d.parts);
  u.all_lo = uniform(d.all_lo);
  u.all_hi = uniform(d.all_hi);
  return u;
}
// One lane of a converged warp, always the same. Code under it stays uniform for the compiler, so that the operands of
// the tensor-core instructions are kept in uniform registers.
__device__ __forceinline__ bool elect() {
  uint32_t yes;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(yes));
  return yes != 0;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm volatile("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm volatile("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint32_t to_bf16x2(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t to_fp16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Sign bits set where the bf16 values are not finite (all exponent bits set: one more carries into the sign).
__device__ __forceinline__ unsigned not_finite(unsigned pair) { return (pair & 0x7f807f80u) + 0x00800080u; }
__device__ __forceinline__ unsigned not_finite(const uint4& v) {
  return not_finite(v.x) | not_finite(v.y) | not_finite(v.z) | not_finite(v.w);
}
// Whether a tile of keys from `first` on has keys that some of the unit's rows see and others do not.
template <bool SINKS>
__device__ __forceinline__ bool mixed_tile(const Desc& u, int first, int sinks) {
  return first + kTile > u.all_hi || (first < u.all_lo && (!SINKS || first + kTile > sinks));
}
// The first key of tile t of a unit.
template <bool SINKS>
__device__ __forceinline__ int first_key(const Desc& u, int t) {
  const int tile = u.tile0 + t;
  return (SINKS && tile >= u.sink_tiles ? tile + u.gap : tile) * kTile;
}

// A wait that gives up after about a second (a try that may sleep comes back after 4 us), and at once after any earlier one
// of the CTA did. Short, because it stands in many places of loops that fill the instruction cache: the status is set at
// the kernel's end. False: it gave up. Only those who copy into what they waited for have to stop then; what the others go on
// to read and write is the CTA's own, up to the end of the unit.
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
// The same answer for every lane of the warp.
__device__ __forceinline__ bool gave_up(int* abort) {
  return __any_sync(0xffffffffu, *reinterpret_cast<volatile int*>(abort) != 0);
}
__device__ __forceinline__ void arrive(const uint64_t& bar) { zb::mbar_arrive(zb::smem_addr(&bar)); }

struct Request {
  int row0, tokens, keys;
};
__device__ __forceinline__ Request request(const ChunkParams& p, int b) {
  Request r;
  r.row0 = min(max(p.kv.cu[b], 0), p.kv.N);
  r.tokens = min(max(p.kv.cu[b + 1], r.row0), p.kv.N) - r.row0;
  if (r.tokens * p.G <= p.few) r.tokens = 0;
  r.keys = max(p.kv.keys[b], 0);
  return r;
}

// Keys of a request that the page table's columns can hold.
__device__ __forceinline__ int held_keys(const ChunkParams& p, int keys) {
  return min(keys, p.kv.max_pages * p.kv.page_size);
}
// Keys [lo, hi) that the token at position pos of a request with `keys` keys sees, beside those below min(sinks, hi).
__device__ __forceinline__ void visible(const ChunkParams& p, int keys, int pos, int& lo, int& hi) {
  const int held = held_keys(p, keys);
  hi = max(p.causal ? min(held, pos + 1) : held, 0);
  lo = p.window > 0 ? (int)max((int64_t)0, (int64_t)pos + 1 - p.window) : 0;
  if (lo <= p.sinks) lo = 0;
}

// Streams of a request's rows come in pairs; a pair's unit of work for one KV head: its rows and key tiles.
__device__ __forceinline__ int stream_pairs(const ChunkParams& p, int tokens) {
  return p.by_pair.quotient(tokens + 2 * p.tokens - 1);
}
__device__ __forceinline__ void unit_tiles(const ChunkParams& p, const Request& r, int pair, Desc& d) {
  const int first = pair * 2 * p.tokens, tokens = min(r.tokens - first, 2 * p.tokens);
  d.token0 = r.row0 + first;
  d.pos0 = r.keys - r.tokens + first;
  d.keys = r.keys;
  d.rows = tokens * p.G;
  int lo0, hi0, lo1, hi1;
  visible(p, r.keys, d.pos0, lo0, hi0);
  visible(p, r.keys, d.pos0 + tokens - 1, lo1, hi1);
  d.all_lo = lo1;
  d.all_hi = hi0 == held_keys(p, r.keys) ? INT32_MAX : hi0;
  d.from = lo0;
  d.tile0 = lo0 / kTile;
  d.tiles = hi1 > lo0 ? (hi1 + kTile - 1) / kTile - d.tile0 : 0;
  d.sink_tiles = d.gap = 0;
  const int seen_first = min(p.sinks, hi1);
  if (lo0 > 0 && seen_first > 0) {  // the sinks' tiles come before the window's, the last of them may be its first
    const int tiles = (seen_first + kTile - 1) / kTile;
    d.sink_tiles = d.tiles > 0 ? min(tiles, d.tile0) : tiles;  // no window: the table ends before it
    d.gap = d.tile0 - d.sink_tiles;
    d.tiles += d.sink_tiles;
    d.tile0 = 0;
  }
}

// A unit's cost, and the first of its tiles that begin at or behind a given cost into it.
__device__ __forceinline__ int unit_cost(const ChunkParams& p, const Desc& d) {
  const bool two = d.rows > p.tokens * p.G;
  return two ? kUnitCost2 + d.tiles * kTileCost2 : kUnitCost1 + d.tiles * kTileCost1;
}
__device__ __forceinline__ int tile_behind(const ChunkParams& p, const Desc& d, int cost) {
  const bool two = d.rows > p.tokens * p.G;
  const int into = cost - (two ? kUnitCost2 : kUnitCost1);
  return into <= 0 ? 0 : two ? (into + kTileCost2 - 1) / kTileCost2 : (into + kTileCost1 - 1) / kTileCost1;
}

// Exclusive prefix of v over the block's threads; `total` the sum. `buffer` alternates from call to call.
template <int THREADS>
__device__ __forceinline__ int block_scan(int v, Tail& tl, int buffer, int& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  int in = v;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const int u = __shfl_up_sync(0xffffffffu, in, o);
    if (lane >= o) in += u;
  }
  int* sums = reinterpret_cast<int*>(tl.ml) + buffer * (THREADS / 32);  // the rows' maxima come later
  if (lane == 31) sums[warp] = in;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const int s = sums[w];
    if (w < warp) before += s;
    total += s;
  }
  return before + in - v;
}

// 1 / x to an ulp; the sums and 1 + e^-x that it is called on are far from fp32's limits, or infinite (0) or NaN (NaN).
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid(__nv_bfloat16 x) { return reciprocal(1.f + ex2(-1.4426950408889634f * __bfloat162float(x))); }

__device__ __forceinline__ void raise_flag(unsigned* flag, unsigned raised) {
  asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(flag), "r"(raised) : "memory");
}
// Whether the flag was raised within a second.
__device__ __forceinline__ bool wait_flag(const unsigned* flag, unsigned raised) {
  const uint64_t start = zb::globaltimer_ns();
  for (;;) {
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
    if (v == raised) return true;
    if (zb::globaltimer_ns() - start > 1000000000ull) return false;
  }
}

// Waits for the parts of a unit that began in this CTA: those of the CTAs after it, every warp for itself.
__device__ __forceinline__ bool wait_parts(const ChunkParams& p, const Desc& u, int cta, int lane) {
  bool there = true;
#pragma unroll 1
  for (int i = 1 + lane; i < u.parts; i += 32) there = wait_flag(p.flags + cta + i, p.raised) && there;
  there = __all_sync(0xffffffffu, there);
  if (!there && p.status && lane == 0) atomicOr(p.status, zb::kStatusAttnChunkTimeout);
  return there;
}
// Part i of a unit that began in CTA cta: the CTA's own, then those of the CTAs after it.
__device__ __forceinline__ int64_t part_slot(int cta, int i) { return (int64_t)(cta + i) * 2 + (i == 0); }

// Joins the parts of a unit of few rows, in the order of their keys: a thread of the row warps takes 8 dims of a row, the
// loads of 8 parts in flight together.
template <int HD>
__device__ __forceinline__ void join_few(const ChunkParams& p, const Desc& u, int cta, int tid, float shift) {
  constexpr int kTogether = 8;
  const int sharers = 32 * kSoftWarps / u.rows, r = tid % u.rows;  // threads of a row
  if (tid / u.rows >= sharers) return;
  const int h = u.kvh * p.G + p.by_group.rest(r);
  const int64_t token = u.token0 + p.by_group.quotient(r);
  const __nv_bfloat16 gate = p.gate ? p.gate[token * p.gate_stride + h] : __float2bfloat16_rn(0.f);
#pragma unroll 1
  for (int piece = tid / u.rows; piece < HD / 8; piece += sharers) {
    float y[8] = {}, top = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int i0 = 0; i0 < u.parts; i0 += kTogether) {
      float m[kTogether], sum[kTogether], hi = top;
      float4 v[kTogether][2];
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        const bool there = i0 + k < u.parts;
        const int64_t part = part_slot(cta, there ? i0 + k : 0);
        const float* ml = p.ml + part * 2 * p.rows_max + r;
        const float4* a = reinterpret_cast<const float4*>(p.acc + (part * (HD / 4) + piece * 2) * p.rows_max * 4 + r * 4);
        m[k] = there ? __ldcg(ml) : -INFINITY;
        sum[k] = there ? __ldcg(ml + p.rows_max) : 0.f;
        v[k][0] = there ? __ldcg(a) : make_float4(0.f, 0.f, 0.f, 0.f);
        v[k][1] = there ? __ldcg(a + p.rows_max) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int k = 0; k < kTogether; ++k) hi = fmaxf(hi, m[k]);
      const float mb = hi == -INFINITY ? 0.f : hi, before = ex2(top - mb);
      top = hi;
      l *= before;
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= before;
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        const float w = ex2(m[k] - mb);  // 0 for a part none of whose keys the row sees; its accumulator is 0 too
        l += sum[k] * w;
        y[0] += v[k][0].x * w, y[1] += v[k][0].y * w, y[2] += v[k][0].z * w, y[3] += v[k][0].w * w;
        y[4] += v[k][1].x * w, y[5] += v[k][1].y * w, y[6] += v[k][1].z * w, y[7] += v[k][1].w * w;
      }
    }
    const float f = l == 0.f ? 0.f : (p.gate ? sigmoid(gate) : 1.f) * reciprocal(l);
    if (piece * 8 < p.kv.hd)
      *reinterpret_cast<uint4*>(p.out + token * p.out_stride + (int64_t)h * p.kv.hd + piece * 8) =
          make_uint4(to_bf16x2(y[0] * f, y[1] * f), to_bf16x2(y[2] * f, y[3] * f), to_bf16x2(y[4] * f, y[5] * f),
                     to_bf16x2(y[6] * f, y[7] * f));
    if (p.lse && piece == 0) p.lse[token * p.Hq + h] = l == 0.f ? -INFINITY : (top - shift + log2f(l)) * 0.6931471805599453f;
  }
}

// Q4: the cache holds 4 bits (and may leave requests of few rows to another kernel). SINKS: there are first keys that stay
// visible; a kernel of its own, as the few registers it takes would be spilled ones for the rest.
template <int HD, bool Q4, bool SINKS>
__global__ void __launch_bounds__(Shape<HD, Q4>::kThreads, 1) gqa_chunk_kernel(const __grid_constant__ ChunkParams p,
                                                                const __grid_constant__ Maps maps) {
  using L = Shape<HD, Q4>;
  constexpr int kThreads = L::kThreads;
  constexpr float kShift = Q4 ? kShiftQ4 : 0.f, kAbove = Q4 ? kAboveQ4 : ::kAbove, kRoom = Q4 ? kRoomQ4 : ::kRoom;
  extern __shared__ __align__(1024) unsigned char gbase[];
  const uint32_t base = zb::smem_addr(gbase);
  if (base % 1024 != 0) {  // the swizzled tiles ask for it; there is no static shared memory before them
    if (p.status) atomicOr(p.status, zb::kStatusAttnChunkTimeout);
    return;
  }
  Tail& tl = *reinterpret_cast<Tail*>(gbase + L::kOffTail);
  const int tid = threadIdx.x, warp = uniform(tid / 32), lane = tid % 32;
  const int B = p.kv.B, Hkv = p.kv.Hkv, hd = p.kv.hd, G = p.G;
  // The work goes backwards over the blocks: a block that joins a unit's parts waits for blocks with lower indices, which
  // were started before it, and they have nothing to wait for before they hand their parts over.
  const int ctas = gridDim.x, cta = ctas - 1 - (int)blockIdx.x;

  if (tid == 0) {
    for (int s = 0; s < L::kSlots; ++s) {
      zb::mbar_init(zb::smem_addr(&tl.full[s]), Q4 ? kOutWarps : p.box ? 1 : kLoadWarps * 32 + 1);
      zb::mbar_init(zb::smem_addr(&tl.empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      zb::mbar_init(zb::smem_addr(&tl.q_full[s]), 1);
      zb::mbar_init(zb::smem_addr(&tl.q_empty[s]), 1);
      zb::mbar_init(zb::smem_addr(&tl.s_full[s]), 2);
      zb::mbar_init(zb::smem_addr(&tl.p_half[s]), kSoftWarps / 2);
      zb::mbar_init(zb::smem_addr(&tl.p_full[s]), kSoftWarps / 2);
      zb::mbar_init(zb::smem_addr(&tl.o_full[s]), 1);
    }
    for (int s = 0; s < kMasks; ++s) {
      zb::mbar_init(zb::smem_addr(&tl.armed[s]), 1);
      zb::mbar_init(zb::smem_addr(&tl.scanned[s]), Q4 ? 2 * kOutWarps : kLoadWarps - 1);
    }
    zb::mbar_init(zb::smem_addr(&tl.drained), 1);
    zb::mbar_init(zb::smem_addr(&tl.halves), 32 * kSoftWarps);
    for (int s = 0; s < kDescs; ++s) {
      zb::mbar_init(zb::smem_addr(&tl.desc_full[s]), 1);
      zb::mbar_init(zb::smem_addr(&tl.desc_empty[s]), kSoftWarps + 1);
    }
    zb::fence_mbar_init();
    tl.abort = 0;
  }
  if (warp == kMmaWarp) tc::alloc(zb::smem_addr(&tl.tmem), 512);
  if (warp == kLoadWarp && lane < 3)
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(lane == 0 ? &maps.q : lane == 1 ? &maps.k : &maps.v))
                 : "memory");
  zb::pdl_enter();  // nothing before it touches memory that another kernel may still write

  // ---- the plan: the work of all units, and this CTA's first one
  // Requests (and below, pairs of streams) go by the block's threads, kThreads at a time; the first ones' stay at hand.
  const Request mine = tid < B ? request(p, tid) : Request{0, 0, 0};
  if (tid == 0) {
    tl.idle[0] = min(max(p.kv.cu[0], 0), p.kv.N);
    tl.idle[1] = min(max(p.kv.cu[B], tl.idle[0]), p.kv.N);
  }
  int* pairs_before = reinterpret_cast<int*>(gbase);                             // [B], over the ring
  Request* requests = reinterpret_cast<Request*>(gbase + kMaxRequests * 4);  // [kThreads], the first requests
  if (tid < B) requests[tid] = mine;
  int64_t all_pairs = 0;
  int buffer = 0;
  bool out_of_order = false;  // bounds that decrease or leave the rows: two requests would write the same ones
#pragma unroll 1
  for (int b0 = 0; b0 < B; b0 += kThreads, buffer ^= 1) {
    const int b = b0 + tid;
    const int n = b < B ? stream_pairs(p, b0 == 0 ? mine.tokens : request(p, b).tokens) : 0;
    if (b < B) out_of_order |= p.kv.cu[b + 1] < p.kv.cu[b] || p.kv.cu[b] < 0 || p.kv.cu[b + 1] > p.kv.N;
    int total;
    const int before = block_scan<kThreads>(n, tl, buffer, total);
    if (b < B) pairs_before[b] = (int)(all_pairs + before);
    all_pairs += total;
  }
  const bool refused = __syncthreads_or(out_of_order);  // nothing is done then
  const int pairs = refused ? 0 : (int)all_pairs;
  if (refused && blockIdx.x == 0 && tid == 0 && p.status) atomicOr(p.status, zb::kStatusAttnChunkBatch);
  struct Pair {
    int b, pair, work;  // work: for one KV head
  };
  auto at_hand = [&](int b) { return b < kThreads ? requests[b] : request(p, b); };
  auto pair_of = [&](int j) {
    if (j >= pairs) return Pair{0, 0, 0};
    int lo = 0, hi = B;  // the last b with pairs_before[b] <= j
#pragma unroll 1
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (pairs_before[mid] <= j) lo = mid;
      else hi = mid;
    }
    Desc d;
    unit_tiles(p, at_hand(lo), j - pairs_before[lo], d);
    return Pair{lo, j - pairs_before[lo], unit_cost(p, d)};
  };
  const Pair first_pair = pair_of(tid);
  int first_total = 0;
  const int first_before = block_scan<kThreads>(first_pair.work, tl, buffer, first_total);
  int64_t work = first_total;
#pragma unroll 1
  for (int j0 = kThreads; j0 < pairs; j0 += kThreads) {
    int total;
    buffer ^= 1;
    block_scan<kThreads>(pair_of(j0 + tid).work, tl, buffer, total);
    work += total;
  }
  work *= Hkv;
  const int64_t share =
      max((int64_t)kTileCost2, work < INT32_MAX - ctas ? ((int)work + ctas - 1) / ctas : (work + ctas - 1) / ctas);
  const int64_t begin = share * cta, end = min(work, begin + share);
  if (begin < end) {
    int64_t seen = 0;
#pragma unroll 1
    for (int j0 = 0; j0 < pairs; j0 += kThreads) {
      Pair q = first_pair;
      int before = first_before, total = first_total;
      if (j0 > 0) {
        q = pair_of(j0 + tid);
        buffer ^= 1;
        before = block_scan<kThreads>(q.work, tl, buffer, total);
      }
      const int64_t at = (seen + before) * Hkv;
      if (q.work > 0 && begin >= at && begin < at + (int64_t)q.work * Hkv) {
        const Request r = at_hand(q.b);
        tl.start[0] = q.b;
        tl.start[1] = r.row0;
        tl.start[2] = r.tokens;
        tl.start[3] = r.keys;
        tl.start[4] = q.pair;
        tl.start_off = begin - at;
      }
      seen += total;
      if (begin < seen * Hkv) break;
    }
  }
  if (hd < HD) {  // the padding dims of every tile stay zero
    __syncthreads();
#pragma unroll 1
    for (uint32_t i = tid; i < L::kOffTail / 16; i += kThreads) reinterpret_cast<uint4*>(gbase)[i] = make_uint4(0, 0, 0, 0);
  }
  tc::fence_proxy_async();  // the plan's tables and the zeros come before the tensor copies over them
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  const uint32_t tmem = uniform((int)tl.tmem);
  int* abort = &tl.abort;

  if (begin >= end) {
    // nothing for this CTA
  } else if (warp >= kLoadWarp) {
    // =============================================================================================== loaders
    if constexpr (Q4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
    const int lw = warp - kLoadWarp;
    constexpr int kChunks = HD / 8;          // 16-byte pieces of a row
    constexpr int kPass = 32 / kChunks;      // rows of a warp's copy instruction
    constexpr int kCopies = kTile / kPass;   // instructions of a tile
    const int chunk = lane % kChunks, sub = lane / kChunks;
    const bool carries = chunk * 8 < hd;
    // Rows 32 k + l of a tile are at element offset off[k] of lane l (negative: absent, zeros). The three warps take 32
    // rows each and share the last 32. The addresses of kAhead copies are formed before they are issued, as each copy
    // takes its row's offset from another lane.
    constexpr int kAhead = 4, kGroups = kCopies / 4 / kAhead;  // groups of copies of 32 rows
    auto copy_group = [&](uint32_t dst, const __nv_bfloat16* src, int64_t off, int row0, int g) {
      int64_t o[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) o[i] = __shfl_sync(0xffffffffu, off, (g * kAhead + i) * kPass + sub);
      if (!carries) return;
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
        cp_async16(dst + piece<HD>(row0 + (g * kAhead + i) * kPass + sub, chunk), src + (o[i] < 0 ? 0 : o[i]) + chunk * 8, o[i] >= 0);
    };
    auto copy_tile = [&](uint32_t dst, const __nv_bfloat16* src, const int64_t (&off)[4], int turn) {
      const int64_t own = lw == 0 ? off[0] : lw == 1 ? off[1] : off[2];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) copy_group(dst, src, own, 32 * lw, g);
#pragma unroll 1
      for (int g = (lw + turn) % kLoadWarps; g < kGroups; g += kLoadWarps) copy_group(dst, src, off[3], 96, g);
    };
    // this lane's request of the window of 32 requests around the current one
    int window0 = -1;
    Request window{};
    auto fetch_window = [&](int b) {
      if (b / 32 != window0) {
        window0 = b / 32;
        const int i = window0 * 32 + lane;
        window = i < B ? request(p, i) : Request{0, 0, 0};
      }
    };
    int b = tl.start[0], pair = tl.start[4];
    Request req{tl.start[1], tl.start[2], tl.start[3]};
    auto take = [&](int i) {
      req.row0 = __shfl_sync(0xffffffffu, window.row0, i % 32);
      req.tokens = __shfl_sync(0xffffffffu, window.tokens, i % 32);
      req.keys = __shfl_sync(0xffffffffu, window.keys, i % 32);
    };
    Desc d;
    unit_tiles(p, req, pair, d);
    int64_t at = begin;
    const int unit0 = unit_cost(p, d);
    int kvh = (int)(tl.start_off / unit0), off = (int)(tl.start_off % unit0);
    int item = 0, tile_no = 0, q_item = 0, scans = 0, n = 0, raws = 0;
    bool going = true;  // until a wait for room gave up
    auto room = [&](const uint64_t& bar, uint32_t parity) {
      going = __all_sync(0xffffffffu, wait(bar, parity, abort));
      return going;
    };
    while (going) {
      // ---- the unit's tiles here: those that begin in this CTA's share, at least as long as any tile
      const int unit = unit_cost(p, d), to = (int)min((int64_t)unit, off + (end - at));
      const int from_tile = tile_behind(p, d, off), to_tile = tile_behind(p, d, to);
      const bool here = d.tiles > 0 ? to_tile > from_tile : off == 0;
      Desc u = d;
      u.kvh = kvh;
      const int held = held_keys(p, req.keys);
      const int32_t* table = p.kv.table + (int64_t)min(b, B - 1) * p.kv.table_stride;
      // Page lookups, a tile ahead of their use and before anything that can wait. A lane's box of a tile:
      const int boxes = p.box ? kTile >> p.box_shift : 0;
      auto look_box = [&](int t) {  // of tile t of the unit's from from_tile on
        const int pos = first_key<SINKS>(d, from_tile + t) + lane * p.box;
        const bool hidden = SINKS && pos >= p.sinks && pos + p.box <= d.from;  // from every row: not brought
        return lane < boxes && pos < held && !hidden ? table[p.by_page.quotient(pos)] : -1;
      };
      int next = -1;
      if (p.box && here && warp == kLoadWarp) next = look_box(0);
      if (here || at >= end) {
        u.tile0 = d.tile0 + from_tile;
        u.tiles = to_tile - from_tile;
        const bool starts = from_tile == 0, ends = to_tile == d.tiles;
        u.mode = at >= end ? kStop : starts && ends ? kFinal : starts ? kPart1 : kPart0;
        // CTAs that hold a part of it from this one on
        const int64_t last = at - off + unit - (u.rows > p.tokens * G ? kTileCost2 : kTileCost1);  // its last tile
        u.parts = ends ? 1 : last < INT32_MAX ? (int)last / (int)share - cta + 1 : (int)(last / share) - cta + 1;
        if (warp == kLoadWarp) {
          const int slot = n % kDescs;
          if (n >= kDescs && !room(tl.desc_empty[slot], (n / kDescs - 1) & 1)) break;
          if (lane == 0) {
            tl.desc[slot] = u;
            arrive(tl.desc_full[slot]);
          }
          __syncwarp();
        }
        ++n;
        if (u.mode == kStop) break;
      } else {
        u.tiles = 0;
      }
      if (u.tiles > 0) {
        if (warp == kLoadWarp + 1) {  // the unit's queries: a stream's tokens, the group's heads of each
#pragma unroll 1
          for (int s = 0; s < (u.rows > p.tokens * G ? 2 : 1); ++s, ++q_item) {
            const int slot = q_item % 2;
            if (q_item >= 2 && !room(tl.q_empty[slot], (q_item / 2 - 1) & 1)) break;
            if (lane == 0) {
              zb::mbar_arrive_expect_tx(zb::smem_addr(&tl.q_full[slot]), (uint32_t)(p.tokens * G * HD * 2));
#pragma unroll 1
              for (int a = 0; a < HD / 64; ++a)
                load_queries(base + L::kOffQ + slot * L::kItem + a * L::kQAtom, &maps.q, a * 64, kvh * G,
                             u.token0 + s * p.tokens, zb::smem_addr(&tl.q_full[slot]));
            }
            __syncwarp();
          }
        }
        // The last two warps look through the values of tiles that hold keys hidden from some rows, half of a tile each.
        // A phase's parity says that the phase is over only to those who know that it is the current one or the last. With
        // tensor copies these warps pass over whole tiles, so they would get to one whose slot is phases behind, and take an
        // older phase for the tile's: they wait until the tile's copies have been started.
        auto look_through = [&](int t, int v_item) {
          const int first = first_key<SINKS>(u, t), slot = scans % kMasks;
          if (warp == kLoadWarp || !mixed_tile<SINKS>(u, first, p.sinks)) return;
          if (p.box) wait(tl.armed[slot], (scans / kMasks) & 1, abort);
          wait(tl.full[v_item % L::kSlots], (v_item / L::kSlots) & 1, abort);
          // groups of 8 rows in turn; rows past the request's keys are no values (warp 8 zeroes them)
          const uint4* v = reinterpret_cast<const uint4*>(gbase + (v_item % L::kSlots) * L::kItem);
          unsigned bad = 0;
          const int rows = min(kTile, held - first);
#pragma unroll 1
          for (int g = lw - 1; g * 8 < rows; g += kLoadWarps - 1)
#pragma unroll
            for (int i = 0; i < L::kGroup / 512; ++i) {
              const unsigned b = not_finite(v[g * (L::kGroup / 16) + 32 * i + lane]);
              bad |= g * 8 + i % 2 * 4 + lane / 8 < rows ? b : 0u;
            }
          const bool found = __any_sync(0xffffffffu, (bad & 0x80008000u) != 0);
          if (lane == 0) {
            tl.found[slot][lw - 1] = found;
            arrive(tl.scanned[slot]);
          }
          ++scans;
        };
        if (Q4) {
          const int block = zb::q4::block_bytes(hd);
          if (warp == kLoadWarp) {  // blocks of 16 keys as they lie in the cache, a bulk copy each
#pragma unroll 1
            for (int t = 0; t < u.tiles && going; ++t, ++tile_no) {
              const int first = first_key<SINKS>(u, t), pos = first + lane * zb::q4::kBlock;
              const bool there = next >= 0 && next < p.kv.num_pages;
              const int64_t from = there ? (int64_t)next * p.kv.page_stride + (int64_t)kvh * p.kv.head_stride +
                                               (int64_t)(p.by_page.rest(pos) / zb::q4::kBlock) * block
                                         : 0;
              const unsigned live = __ballot_sync(0xffffffffu, there);
              unsigned bits[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int r = 32 * k + lane;
                const bool hidden = first + r >= p.sinks && first + r < d.from;  // from every row
                bits[k] = __ballot_sync(0xffffffffu, first + r < held && !hidden && (live >> (r / zb::q4::kBlock) & 1u));
              }
              if (t + 1 < u.tiles) next = look_box(t + 1);
#pragma unroll 1
              for (int half = 0; half < 2; ++half, ++raws) {
                const int slot = raws % kRawStages;
                if (raws >= kRawStages && !room(tl.scanned[slot], (raws / kRawStages - 1) & 1)) break;
                if (lane == 0) {
                  if (half == 0) *reinterpret_cast<uint4*>(tl.mask[tile_no % kMasks]) = make_uint4(bits[0], bits[1], bits[2], bits[3]);
                  zb::mbar_arrive_expect_tx(zb::smem_addr(&tl.armed[slot]),
                                            (uint32_t)(__popc(live >> (kRawBlocks * half) & ((1u << kRawBlocks) - 1)) * block));
                }
                __syncwarp();
                if (there && lane / kRawBlocks == half)
                  zb::bulk_g2s(base + L::kOffRaw + slot * L::kRaw + lane % kRawBlocks * block,
                               reinterpret_cast<const unsigned char*>(p.kv.k) + from, (uint32_t)block,
                               zb::smem_addr(&tl.armed[slot]));
              }
            }
          } else {  // the keys (warps 10-12) and values (13-15) of a tile as bf16, absent ones as zeros
            // A lane takes one group of a row, so its pair is looked at once for four words; it takes those in an order that the row
            // shifts, so that a warp's rows, 64 (or 32) bytes of codes each, are in different banks.
            constexpr int kLanes = HD / 32, kRows = 32 / kLanes, kPasses = zb::q4::kBlock / kRows;  // of a row, of a pass, of a block
            const int kv = (lw - 1) / kOutWarps, share = (lw - 1) % kOutWarps, groups = hd / zb::q4::kGroup;
            const int g = lane % kLanes, sub = lane / kLanes, turn = sub * kLanes / 8;
#pragma unroll 1
            for (int t = 0; t < u.tiles && going; ++t, ++tile_no, item += 2) {
              const int slot = (item + kv) % L::kSlots;
              uint4 exist{};
#pragma unroll 1
              for (int half = 0; half < 2; ++half, ++raws) {
                const int stage = raws % kRawStages;
                if (!wait(tl.armed[stage], (raws / kRawStages) & 1, abort)) going = false;
                if (half == 0) {
                  if (item >= L::kSlots && !room(tl.empty[slot], (item / L::kSlots - 1) & 1)) break;
                  exist = *reinterpret_cast<const uint4*>(tl.mask[tile_no % kMasks]);
                }
                const unsigned char* raw = gbase + L::kOffRaw + stage * L::kRaw;
                const unsigned lower = half ? exist.z : exist.x, upper = half ? exist.w : exist.y;
                // A warp takes whole blocks. Values are written as fp16, whose rounding is an eighth of bf16's, in blocks that fp16
                // holds: one product of the tensor cores takes the 16 keys of a block, so each block has a type of its own and the
                // warps need not agree on it (on one type for a stage: 181 us for 4 x 512 tokens behind 8192, now 177).
#pragma unroll 1
                for (int blk = (share + kOutWarps - raws % kOutWarps) % kOutWarps; blk < kRawBlocks; blk += kOutWarps) {
                  const unsigned char* from = raw + blk * block;
                  const unsigned exists = (blk & 2 ? upper : lower) >> (blk & 1) * zb::q4::kBlock;
                  uint32_t pair[kPasses], over = 0;
                  bool holds = kv != 0;
                  if (g < groups) {
#pragma unroll
                    for (int i = 0; i < kPasses; ++i) {
                      const int in = kRows * i + sub;
                      pair[i] = reinterpret_cast<const uint32_t*>(from + (16 + 2 * kv) * hd)[in * groups + g];
                      if (!(exists >> in & 1u) || zb::q4::pair_is_none(pair[i])) pair[i] = 0;
                      zb::q4::fp16_holds(pair[i], over, holds);
                    }
                  }
                  const bool half_type = __all_sync(0xffffffffu, holds && (over & 0x80008000u) == 0);
                  if (kv && lane == 0) reinterpret_cast<unsigned char*>(tl.found[tile_no % kMasks])[kRawBlocks * half + blk] = !half_type;
                  if (g < groups) {
#pragma unroll
                    for (int i = 0; i < kPasses; ++i) {
                      const int in = kRows * i + sub;
                      const uint32_t* w = reinterpret_cast<const uint32_t*>(from + 8 * kv * hd + in * (hd / 2)) + g;
                      uint32_t words[4];
#pragma unroll
                      for (int k = 0; k < 4; ++k) words[k] = w[((k + turn) & 3) * groups];
                      auto to = [&](int k) {
                        return reinterpret_cast<uint4*>(gbase + slot * L::kItem +
                                                        piece<HD>(64 * half + zb::q4::kBlock * blk + in, 4 * g + ((k + turn) & 3)));
                      };
                      if (half_type) {
                        const zb::q4::HalfPair halves(pair[i]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) *to(k) = halves.read_word(words[k]);
                      } else {
#pragma unroll
                        for (int k = 0; k < 4; ++k) *to(k) = zb::q4::read_word(words[k], pair[i]);
                      }
                    }
                  }
                }
                __syncwarp();
                if (lane == 0) arrive(tl.scanned[stage]);
              }
              tc::fence_proxy_async();  // what was written -> the tensor cores
              __syncwarp();
              if (lane == 0) arrive(tl.full[slot]);
            }
          }
        } else if (p.box) {
          if (warp == kLoadWarp) {
#pragma unroll 1
            for (int t = 0; t < u.tiles && going; ++t, ++tile_no) {
              const int first = first_key<SINKS>(u, t), pos = first + lane * p.box;
              const bool mixed = mixed_tile<SINKS>(u, first, p.sinks);
              const bool there = next >= 0 && next < p.kv.num_pages;
              const int page = there ? next * p.page_heads + (p.page_heads > 1 ? kvh : 0)
                                     : (int)(p.kv.num_pages * p.page_heads);  // past the end: zeros
              const int group = there ? p.by_page.rest(pos) / 8 : 0;
              const unsigned live = __ballot_sync(0xffffffffu, there);
              unsigned bits[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int r = 32 * k + lane;
                bits[k] = __ballot_sync(0xffffffffu, first + r < held && (live >> (r >> p.box_shift) & 1u));
              }
              if (t + 1 < u.tiles) next = look_box(t + 1);
#pragma unroll 1
              for (int kv = 0; kv < 2; ++kv, ++item) {
                const int slot = item % L::kSlots;
                if (item >= L::kSlots && !room(tl.empty[slot], (item / L::kSlots - 1) & 1)) break;
                if (lane == 0) {
                  if (kv == 0) *reinterpret_cast<uint4*>(tl.mask[tile_no % kMasks]) = make_uint4(bits[0], bits[1], bits[2], bits[3]);
                  zb::mbar_arrive_expect_tx(zb::smem_addr(&tl.full[slot]), L::kItem);
                  if (kv == 1 && mixed) arrive(tl.armed[scans % kMasks]);
                }
                __syncwarp();
                if (lane < boxes)
                  load_rows(base + slot * L::kItem + lane * (p.box / 8) * L::kGroup, kv ? &maps.v : &maps.k,
                            kvh * p.head_atoms, group, page, zb::smem_addr(&tl.full[slot]));
              }
              scans += mixed;
            }
          } else {
#pragma unroll 1
            for (int t = 0; t < u.tiles; ++t, item += 2) look_through(t, item + 1);
          }
        } else {
          int pages[4];
          auto look = [&](int t) {  // pages of the lane's rows of tile t
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int pos = first_key<SINKS>(u, t) + 32 * k + lane;
              const bool hidden = SINKS && pos >= p.sinks && pos < u.from;  // from every row: not brought
              pages[k] = pos < held && !hidden ? table[p.by_page.quotient(pos)] : -1;
            }
          };
          look(0);
#pragma unroll 1
          for (int t = 0; t < u.tiles && going; ++t, ++tile_no) {
            int64_t off[4];
            unsigned bits[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int pos = first_key<SINKS>(u, t) + 32 * k + lane;
              const bool there = pages[k] >= 0 && pages[k] < p.kv.num_pages;
              off[k] = there ? (int64_t)pages[k] * p.kv.page_stride + (int64_t)p.by_page.rest(pos) * p.kv.slot_stride +
                                   (int64_t)kvh * p.kv.head_stride
                             : -1;
              bits[k] = __ballot_sync(0xffffffffu, there);
            }
            if (t + 1 < u.tiles) look(t + 1);
#pragma unroll 1
            for (int kv = 0; kv < 2; ++kv, ++item) {
              const int slot = item % L::kSlots;
              if (item >= L::kSlots && !room(tl.empty[slot], (item / L::kSlots - 1) & 1)) break;
              copy_tile(base + slot * L::kItem, kv ? p.kv.v : p.kv.k, off, item);
              cp_async_arrive(zb::smem_addr(&tl.full[slot]));
              if (warp == kLoadWarp && lane == 0) {
                if (kv == 0) *reinterpret_cast<uint4*>(tl.mask[tile_no % kMasks]) = make_uint4(bits[0], bits[1], bits[2], bits[3]);
                arrive(tl.full[slot]);
              }
            }
            if (going) look_through(t, item - 1);
          }
        }
      }
      // ---- the next unit: KV head, then pair, then request
      at += to - off;
      off = 0;
      if (at >= end) continue;  // the stop descriptor
      if (++kvh == Hkv) {
        kvh = 0;
        if (pair + 1 < stream_pairs(p, req.tokens)) {
          ++pair;
        } else {
          pair = 0;
          do {
            ++b;
            fetch_window(min(b, B - 1));
            take(min(b, B - 1));
          } while (b < B && req.tokens == 0);
        }
        unit_tiles(p, req, pair, d);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // Nothing is in flight when the CTA's shared memory goes to another, also where a wait gave up: a lane waits for the last
    // copies into a slot.
    auto landed = [&](const uint64_t* full, int slots, int items) {
      if (lane < min(slots, items))
        zb::mbar_wait_bounded(zb::smem_addr(full + lane), (items - 1 - lane) / slots & 1, p.status, zb::kStatusAttnChunkTimeout);
      __syncwarp();
    };
    if (warp == kLoadWarp && p.box && !Q4) landed(tl.full, L::kSlots, item);
    if (warp == kLoadWarp && Q4) landed(tl.armed, kRawStages, raws);
    if (warp == kLoadWarp + 1) landed(tl.q_full, 2, q_item);
  } else if (warp == kMmaWarp) {
    // =============================================================================================== tensor cores
    if constexpr (Q4) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    else asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
    constexpr uint32_t kIdS = tc::idesc_bf16(0, kTile), kIdO = tc::idesc_bf16(0, HD, false, /*b_mn=*/true);
    constexpr uint32_t kFp16 = (1u << 7) | (1u << 10);  // bits that make the operands bf16; off where values are fp16
    int types[2] = {0, 0};  // 4 bits: whether the blocks of either half of a tile are bf16, a byte each
    uint32_t height = 0;  // the rest of the descriptors: the unit's rows
    // This warp's own time between two products is time the tensor cores stand still once their short queue is empty: ring
    // positions are kept instead of divided out, and one lane issues a stream's products and commits in one go.
    struct Ring {
      int slot;
      uint32_t phase;
      __device__ __forceinline__ Ring after(int items) const {
        const int to = slot + items;
        return to >= L::kSlots ? Ring{to - L::kSlots, phase ^ 1u} : Ring{to, phase};
      }
    };
    Ring at{0, 0};  // of the unit's next tile's keys; its values lie one further
    int q_item = 0, scans = 0, tile_no = 0;
    uint32_t parity = 0;  // bit s: of stream s's weights
    auto full = [&](const Ring& i) { wait(tl.full[i.slot], i.phase, abort); };
    auto commit = [&](const uint64_t& bar) { tc::commit(zb::smem_addr(&bar)); };
    const uint64_t k_desc = tc::desc_mnmajor(base, 16, L::kGroup), v_desc = tc::desc_mnmajor(base, 1024, L::kGroup);
    const uint64_t q_desc = tc::desc_kmajor(base + L::kOffQ);
    // By one lane: S_s = Q K^T of a ring slot and query buffer q.
    auto issue_s = [&](int s, int slot, int q) {
      const uint64_t kd = k_desc + (uint32_t)slot * (L::kItem / 16), qd = q_desc + (uint32_t)(q % 2) * (L::kItem / 16);
#pragma unroll
      for (int ks = 0; ks < HD / 16; ++ks)
        tc::mma(tmem + L::kColS + s * kTile, qd + ((ks / 4) * L::kQAtom + (ks % 4) * 32) / 16,
                kd + ((ks / 4) * 1024 + (ks % 4) * 32) / 16, kIdS | height, ks > 0);
      commit(tl.s_full[s]);
      arrive(tl.s_full[s]);  // passes on the tile's key mask, which this thread got with the tile
    };
    // By one lane: O_s (+)= P_s V of a ring slot, half of its keys; the product of the weights' rests too where they have some.
    auto issue_o = [&](int s, int slot, int half, bool accumulate, bool fine) {
      const uint64_t vd = v_desc + (uint32_t)slot * (L::kItem / 16);
#pragma unroll
      for (int k0 = 0; k0 < kTile / 32; ++k0) {
        const int ks = k0 + half * (kTile / 32);
        mma_ts(tmem + L::kColO + s * HD, tmem + L::kColS + s * kTile + 8 * ks, vd + ks * 2 * L::kGroup / 16,
               Q4 && !(types[half] >> 8 * k0 & 1) ? (kIdO | height) & ~kFp16 : kIdO | height, accumulate || ks > 0);
      }
      if (fine)
#pragma unroll
        for (int k0 = 0; k0 < kTile / 32; ++k0) {
          const int ks = k0 + half * (kTile / 32);
          mma_ts(tmem + L::kColO + s * HD, tmem + L::kColS + s * kTile + kTile / 2 + 8 * ks, vd + ks * 2 * L::kGroup / 16,
                 kIdO | height, true);
        }
    };
    for (int n = 0;; ++n) {
      const int slot = n % kDescs;
      wait(tl.desc_full[slot], (n / kDescs) & 1, abort);
      const Desc u = uniform(tl.desc[slot]);
      if (lane == 0) arrive(tl.desc_empty[slot]);
      if (u.mode == kStop || gave_up(abort)) break;
      if (u.tiles == 0) continue;
      const bool two = u.rows > p.tokens * G;  // two streams of rows share each tile, or one's two halves take turns
      const bool fine = !Q4 && u.rows <= kFineRows;
      height = tc::idesc_bf16(fine ? 64 : kStreamRows, 0) & ~tc::idesc_bf16(0, 0);
      const int stride = two ? 1 : 2;          // tiles from one of a stream to its next
      const int held = held_keys(p, u.keys);
      Ring ahead = at;  // of the next tile whose scores are due
#pragma unroll 1
      for (int t = -stride; t < u.tiles; ++t) {
        // O_s += P_s(t) V(t) as soon as P_s(t) is there, then the stream's next scores; before the first tile, those alone
        const bool more = t + stride < u.tiles, ends = t + stride == u.tiles - 1;
        const int s0 = two ? 0 : t & 1, s1 = two ? 1 : s0, first = first_key<SINKS>(u, t);
        const Ring v = at.after(1), k = ahead;
        unsigned char* v_tile = gbase + v.slot * L::kItem;
        bool found = false;
        if (t >= 0) {
          full(v);
          if constexpr (Q4) {
            const int* found = tl.found[tile_no % kMasks];
            types[0] = uniform(found[0]);
            types[1] = uniform(found[1]);
            ++tile_no;
          }
          // rows of the last page past the request's keys came along with a tensor copy: no key, so no value either
          if (!Q4 && p.box && first + kTile > held && held % p.box != 0) {
            const int r0 = held - first, r1 = (r0 + p.box - 1) / p.box * p.box;
#pragma unroll 1
            for (int i = r0 * (HD / 8) + lane; i < r1 * (HD / 8); i += 32)
              *reinterpret_cast<uint4*>(v_tile + piece<HD>(i / (HD / 8), i % (HD / 8))) = make_uint4(0, 0, 0, 0);
            tc::fence_proxy_async();
            __syncwarp();
          }
          if (!Q4 && mixed_tile<SINKS>(u, first, p.sinks)) {
            const int slot = scans % kMasks;
            wait(tl.scanned[slot], (scans / kMasks) & 1, abort);
            ++scans;
            found = uniform(tl.found[slot][0] | tl.found[slot][1]) != 0;
            if (found) {  // every stream adds what it sees before it hands over P; then the values are zeroed
#pragma unroll 1
              for (int s = s0; s <= s1; ++s) wait(tl.p_full[s], (parity >> s) & 1u, abort);
              uint16_t* e = reinterpret_cast<uint16_t*>(v_tile);
#pragma unroll 1
              for (uint32_t i = lane; i < L::kItem / 2; i += 32)
                if ((e[i] & 0x7f80u) == 0x7f80u) e[i] = 0;
              tc::fence_proxy_async();
              __syncwarp();
            }
          }
          if (p.box == 0) tc::fence_proxy_async();  // 16-byte copies -> the tensor cores
          at = at.after(2);
        }
#pragma unroll 1
        for (int s = s0; s <= s1; ++s) {
          if (t >= 0) {
            wait(tl.p_half[s], (parity >> s) & 1u, abort);
            tc::fence_after();
            if (elect()) issue_o(s, v.slot, 0, t >= stride || found, fine);
            __syncwarp();
            wait(tl.p_full[s], (parity >> s) & 1u, abort);
            tc::fence_after();
            if (elect()) {
              issue_o(s, v.slot, 1, true, fine);
              if (s == s1) commit(tl.empty[v.slot]);
              if (!more) commit(tl.o_full[s]);
            }
            __syncwarp();
            parity ^= 1u << s;
          }
          if (more) {
            const int q = q_item + (two ? s : 0);
            if (t < 0) wait(tl.q_full[q % 2], (q / 2) & 1, abort);
            if (s == s0) {
              full(k);
              if (p.box == 0) tc::fence_proxy_async();
            }
            if (elect()) {
              issue_s(s, k.slot, q);
              if (s == s1) commit(tl.empty[k.slot]);
              if (ends) commit(tl.q_empty[q % 2]);
            }
            __syncwarp();
          }
        }
        if (more) ahead = ahead.after(2);
      }
      q_item += two ? 2 : 1;
    }
    if (elect()) commit(tl.drained);  // nothing is in flight when the tensor memory is given back, also after a wait that
    __syncwarp();                     // gave up
    zb::mbar_wait_bounded(zb::smem_addr(&tl.drained), 0, p.status, zb::kStatusAttnChunkTimeout);
    __syncwarp();
  } else {
    // =============================================================================================== rows
    // 8 x 32 x 192 + 4 x 32 x 120 registers are the 384 x 168 that the CTA was launched with
    if constexpr (Q4) asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");  // with 8 x 32 x 72 of the others, the 512 x 128 of the launch
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    const int s = warp / 4;  // stream
    const uint32_t tlane = tmem + ((uint32_t)(32 * (warp % 4)) << 16);
    const uint32_t col_s = tlane + L::kColS + s * kTile, col_o = tlane + L::kColO + s * HD;
    int tile_no = 0, mine = 0, units = 0, scans = 0, meetings = 0;  // counters of what this CTA, or this stream, has done
    auto meet = [&]() {  // the 8 row warps
      arrive(tl.halves);
      wait(tl.halves, meetings & 1, abort);
      ++meetings;
    };
    for (int n = 0;; ++n) {
      const int slot = n % kDescs;
      wait(tl.desc_full[slot], (n / kDescs) & 1, abort);
      const Desc u = uniform(tl.desc[slot]);
      if (lane == 0) arrive(tl.desc_empty[slot]);
      if (u.mode == kStop || gave_up(abort)) break;
      const int stream_rows = p.tokens * G;
      const bool two = u.rows > stream_rows;
      const int first_row = two ? s * stream_rows : 0, rows = min(stream_rows, u.rows - first_row);
      const bool fine = !Q4 && u.rows <= kFineRows;
      const bool idle = 32 * (warp % 4) >= rows;  // no lane of the warp has a row
      const int stride = two ? 1 : 2;
      float m = kAbove, l = 0.f;
      float m2[2] = {}, l2[2] = {};  // fine: of rows lane / 4 and 8 further; l of this thread's keys only
      bool any2[2] = {};             // whether they saw a key
      __nv_bfloat16 gate_raw = __float2bfloat16_rn(0.f);  // on its way while the tiles are worked on
      {
        int lo = 0, hi = INT32_MAX;  // a lane without a row sees everything; it is not stored
        if (32 * (warp % 4) + lane < rows)
          visible(p, u.keys, u.pos0 + p.by_group.quotient(first_row + 32 * (warp % 4) + lane), lo, hi);
        if (p.gate && u.mode != kPart0 && 32 * (warp % 4) + lane < rows) {
          const int r = first_row + 32 * (warp % 4) + lane;
          gate_raw = p.gate[(int64_t)(u.token0 + p.by_group.quotient(r)) * p.gate_stride + u.kvh * G + p.by_group.rest(r)];
        }
#pragma unroll 1
        for (int t = 0; t < u.tiles; ++t) {
          const int first = first_key<SINKS>(u, t);
          const bool scan = !Q4 && mixed_tile<SINKS>(u, first, p.sinks);
          if (!two && (t & 1) != s) {  // the other half's tile
            scans += scan;
            continue;
          }
          wait(tl.s_full[s], mine & 1, abort);
          ++mine;
          tc::fence_after();
          if (idle) {  // its rows are stored nowhere; zeros, because products of them take less power than of scores
            scans += scan;
            const uint32_t zero[32] = {};
#pragma unroll 1
            for (int c = 0; c < (fine ? 4 : 2); ++c) st32(col_s + 32 * c, zero);
            tc::st_wait();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) {
              arrive(tl.p_half[s]);
              arrive(tl.p_full[s]);
            }
            continue;
          }
          bool half_types = true;  // all values of the tile are fp16
          if constexpr (Q4) {
            const int v_item = 2 * (tile_no + t) + 1;
            wait(tl.full[v_item % L::kSlots], (v_item / L::kSlots) & 1, abort);  // this stream's last product has waited for the one before
            half_types = !(tl.found[(tile_no + t) % kMasks][0] | tl.found[(tile_no + t) % kMasks][1]);
          }
          const unsigned* there = tl.mask[(tile_no + t) % kMasks];
          const uint4 all4 = *reinterpret_cast<const uint4*>(there);
          const bool partly = __any_sync(0xffffffffu, (first < lo && (!SINKS || first + kTile > p.sinks)) || first + kTile > hi ||
                                                          (all4.x & all4.y & all4.z & all4.w) != 0xffffffffu);
          auto seen = [&](int c) {  // which of keys 32 c .. of the tile the row sees
            const int a = min(max(lo - first - 32 * c, 0), 32), z = min(max(hi - first - 32 * c, 0), 32);
            const unsigned below = z >= 32 ? 0xffffffffu : (1u << z) - 1u;
            const unsigned under = a >= 32 ? 0xffffffffu : (1u << a) - 1u;
            if (!SINKS) return there[c] & below & ~under;
            const int k = min(max(p.sinks - first - 32 * c, 0), 32);
            const unsigned kept = k >= 32 ? 0xffffffffu : (1u << k) - 1u;
            return there[c] & below & (~under | kept);
          };
          const uint64_t scale2 = pack2(p.scale_log2, p.scale_log2);
          uint64_t minus, sum2[2] = {0, 0};
          auto rescale = [&](float corr) {  // the lane's row of the accumulator
            if (t >= stride) {
#pragma unroll 1
              for (int c = 0; c < HD / 16; ++c) {
                uint32_t o[16];
                tc::ld16(col_o + 16 * c, o);
                tc::ld_wait();
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * corr);
                tc::st16(col_o + 16 * c, o);
              }
            }
          };
          // Whether the weights formed with m hold for a tile whose largest score is `top` (NaN: they do); if not, m is set
          // by it, and the sum and the accumulator follow. A row's m goes by its own scores alone: with those of the warp's
          // other rows in it, what rounding makes of a token's output would hang on tokens behind it, and on what lies in
          // lanes without a row. `set`: first keys set m whatever it is.
          auto holds = [&](float top, bool set) {
            top *= p.scale_log2;
            const bool off = l != 0.f ? top > m : (set || top > m - kRoom || top < m - kAbove) && top > -INFINITY;
            if (!__any_sync(0xffffffffu, off)) return true;
            top += kAbove;
            const float corr = off && l != 0.f ? ex2(m - top) : 1.f;  // without a key so far both are 0
            l *= corr;
            rescale(corr);
            if (off) m = top;
            return false;
          };
          auto hand_over = [&](const uint64_t& bar) {
            tc::st_wait();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) arrive(bar);
          };
          if (fine) {
            // Two rows' keys 8 b + 2 (lane % 4), + 1: x[4 b], x[4 b + 1] of row lane / 4, the next two of the row 8 further.
            uint32_t x[64], hi16[32], rest[32];
            ld_fine(col_s, x);
            const uint64_t less = pack2(-1.f + 0x1p-24f, -1.f + 0x1p-24f);
            tc::ld_wait();
            if (partly) {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const unsigned word = seen(c);
                  const unsigned wa = __shfl_sync(0xffffffffu, word, lane / 4) >> 2 * (lane % 4);
                  const unsigned wb = __shfl_sync(0xffffffffu, word, lane / 4 + 8) >> 2 * (lane % 4);
#pragma unroll
                  for (int b = 0; b < 4; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                      if (!((e < 2 ? wa : wb) >> (8 * b + e % 2) & 1u)) x[16 * c + 4 * b + e] = 0xff800000u;
                }
            }
            float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int q = 0; q < 32; ++q)
              top[q % 2] = fmaxf(fmaxf(top[q % 2], __uint_as_float(x[2 * q])), __uint_as_float(x[2 * q + 1]));
            bool off[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
              top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2)) * p.scale_log2;
              off[r] = top[r] > m2[r] || (!any2[r] && top[r] > -INFINITY);
            }
            if (__any_sync(0xffffffffu, off[0] || off[1])) {
              float corr[2];
#pragma unroll
              for (int r = 0; r < 2; ++r) {
                corr[r] = off[r] && any2[r] ? ex2(m2[r] - (top[r] + kAbove)) : 1.f;
                l2[r] *= corr[r];
                if (off[r]) m2[r] = top[r] + kAbove;
              }
              rescale(of_row(corr[0], corr[1], lane));
            }
            any2[0] |= top[0] > -INFINITY;
            any2[1] |= top[1] > -INFINITY;
            const uint64_t minus_a = pack2(-m2[0], -m2[0]), minus_b = pack2(-m2[1], -m2[1]);
            sum2[0] = sum2[1] = 0;
            constexpr int kPairs = 4, kGroups = 32 / kPairs;
            float e[2][2 * kPairs];
#pragma unroll
            for (int g = 0; g <= kGroups; ++g)
#pragma unroll
              for (int i = 0; i < kPairs; ++i) {
                if (g < kGroups) {
                  const int q = g * kPairs + i;
                  float a, z;
                  unpack2(fma2(pack2(__uint_as_float(x[2 * q]), __uint_as_float(x[2 * q + 1])), scale2, q % 2 ? minus_b : minus_a),
                          a, z);
                  e[g % 2][2 * i] = ex2(a);
                  e[g % 2][2 * i + 1] = ex2(z);
                }
                if (g > 0) {
                  // A weight's upper 16 bits, and the rest. 2^-24 of the weight stays in the rest, so that it is not 0 where the
                  // weight is not: 0 times an infinite value would be NaN.
                  const int q = (g - 1) * kPairs + i;
                  const uint64_t w = pack2(e[(g + 1) % 2][2 * i], e[(g + 1) % 2][2 * i + 1]);
                  const uint32_t a = __float_as_uint(e[(g + 1) % 2][2 * i]) & 0xffff0000u;
                  const uint32_t z = __float_as_uint(e[(g + 1) % 2][2 * i + 1]) & 0xffff0000u;
                  sum2[i % 2] = add2(sum2[i % 2], w);
                  hi16[q] = a >> 16 | z;
                  float r0, r1;
                  unpack2(fma2(pack2(__uint_as_float(a), __uint_as_float(z)), less, w), r0, r1);
                  rest[q] = to_bf16x2(r0, r1);
                }
              }
            st_fine(col_s, hi16);
            st_fine(col_s + kTile / 2, rest);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float a, z;
              unpack2(sum2[r], a, z);
              l2[r] += a + z;
            }
            sum2[0] = sum2[1] = 0;
            if (!scan) hand_over(tl.p_half[s]);
          } else if (partly || (Q4 && !half_types)) {  // 32 keys at a time, without those that no row of the warp sees; first their largest score
            float top = -INFINITY;
            auto scores = [&](int c, uint32_t (&y)[32]) {  // those that the row does not see as -infinity; whether any row sees one
              const unsigned word = seen(c);
              if (!__any_sync(0xffffffffu, word != 0)) return false;
              ld32(col_s + 32 * c, y);
              const bool all = __all_sync(0xffffffffu, word == 0xffffffffu);
              tc::ld_wait();
              if (!all) {
#pragma unroll
                for (int j = 0; j < 32; ++j) y[j] = (word >> j) & 1u ? y[j] : 0xff800000u;
              }
              return true;
            };
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t y[32];
              if (!scores(c, y)) continue;
              float t2 = -INFINITY;
#pragma unroll
              for (int j = 0; j < 32; j += 4) {
                top = fmaxf(fmaxf(top, __uint_as_float(y[j])), __uint_as_float(y[j + 1]));
                t2 = fmaxf(fmaxf(t2, __uint_as_float(y[j + 2])), __uint_as_float(y[j + 3]));
              }
              top = fmaxf(top, t2);
            }
            // The first keys of a unit's row set m by their largest score, whose weight is a power of 2 then, and exact.
            holds(top, t < stride);
            minus = pack2(kShift - m, kShift - m);
            sum2[0] = sum2[1] = 0;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {  // the weights take half of the scores' columns: those of scores already read
              uint32_t y[32], packed[16] = {};
              if (scores(c, y)) {
                const int bf16 = Q4 ? tl.found[(tile_no + t) % kMasks][c / 2] >> 16 * (c & 1) : 0;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                  float a, z;
                  unpack2(fma2(pack2(__uint_as_float(y[2 * j]), __uint_as_float(y[2 * j + 1])), scale2, minus), a, z);
                  a = ex2(a);
                  z = ex2(z);
                  sum2[j % 2] = add2(sum2[j % 2], pack2(a, z));
                  packed[j] = Q4 && !(bf16 & (j < 8 ? 1 : 256)) ? to_fp16x2(a, z) : to_bf16x2(a, z);
                }
              }
              tc::st16(col_s + 16 * c, packed);
            }
            if (!scan) hand_over(tl.p_half[s]);
          } else {
            // The weights are formed with the m there is, and the tile's largest score is found beside them; nothing is
            // written over the scores before it is known that they hold. A second turn is rare, and the last.
            uint32_t x[kTile];
            // p of a half of the keys. The exponential unit takes 8 cycles an instruction, so everything else has to run in
            // its shadow: the scaling of the next group, the sum and the packing of the one before, and in the first half
            // the search for the largest score are written between a group's exponentials.
            float part[4];
            auto weigh = [&](int half, uint32_t (&packed)[32]) {
              constexpr int kPairs = 4, kGroups = kTile / 4 / kPairs;
              uint64_t a2[kPairs];
              float e[2][2 * kPairs];
              auto scaled = [&](int g, int i) {
                const int k = 64 * half + 2 * (g * kPairs + i);
                return fma2(pack2(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), scale2, minus);
              };
#pragma unroll
              for (int i = 0; i < kPairs; ++i) a2[i] = scaled(0, i);
#pragma unroll
              for (int g = 0; g <= kGroups; ++g) {
#pragma unroll
                for (int i = 0; i < kPairs; ++i) {
                  if (g < kGroups) {
                    float a, z;
                    unpack2(a2[i], a, z);
                    e[g % 2][2 * i] = ex2(a);
                    e[g % 2][2 * i + 1] = ex2(z);
                    if (g + 1 < kGroups) a2[i] = scaled(g + 1, i);
                    if (half == 0) {  // 4 scores to each of the group's pairs
                      const int k = 16 * g + 4 * i;
                      const float hi = fmaxf(__uint_as_float(x[k + 2]), __uint_as_float(x[k + 3]));
                      part[i] = g == 0 ? __uint_as_float(x[k]) : fmaxf(part[i], __uint_as_float(x[k]));
                      part[i] = fmaxf(fmaxf(part[i], __uint_as_float(x[k + 1])), hi);
                    }
                  }
                  if (g > 0) {
                    const float a = e[(g + 1) % 2][2 * i], z = e[(g + 1) % 2][2 * i + 1];
                    sum2[i % 2] = add2(sum2[i % 2], pack2(a, z));
                    packed[(g - 1) * kPairs + i] = Q4 ? to_fp16x2(a, z) : to_bf16x2(a, z);
                  }
                }
              }
            };
            uint32_t packed[32];
            bool again = false;
            do {
#pragma unroll
              for (int c = 0; c < 4; ++c) ld32(col_s + 32 * c, x + 32 * c);
              minus = pack2(kShift - m, kShift - m);
              sum2[0] = sum2[1] = 0;
              tc::ld_wait();
              weigh(0, packed);
              again = !again && !holds(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])), false);
            } while (again);
            st32(col_s, packed);
            if (!scan) hand_over(tl.p_half[s]);
            weigh(1, packed);
            st32(col_s + 32, packed);
          }
          {
            float a, z;
            unpack2(add2(sum2[0], sum2[1]), a, z);
            l += a + z;
          }
          if (scan) {
            const int slot = scans % kMasks;
            wait(tl.scanned[slot], (scans / kMasks) & 1, abort);
            ++scans;
            if (tl.found[slot][0] | tl.found[slot][1]) {  // values that are not finite, one by one
              if (t < stride) {  // the tile's product adds to the accumulator then
                uint32_t zero[32] = {};
#pragma unroll
                for (int c = 0; c < HD / 32; ++c) st32(col_o + 32 * c, zero);
              }
              tc::st_wait();
              const unsigned char* v = gbase + (size_t)((2 * (tile_no + t) + 1) % L::kSlots) * L::kItem;
#pragma unroll 1
              for (int j = 0; j < kTile; ++j) {
                const bool sees = (seen(j / 32) >> (j % 32)) & 1u;
#pragma unroll 1
                for (int c = 0; c < HD / 8; ++c) {
                  const uint4 w = *reinterpret_cast<const uint4*>(v + piece<HD>(j, c));
                  if (!(not_finite(w) & 0x80008000u)) continue;  // the same for every lane
                  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                  for (int e = 0; e < 8; ++e) {
                    const float val = __uint_as_float(e % 2 ? q[e / 2] & 0xffff0000u : q[e / 2] << 16);
                    if ((__float_as_uint(val) & 0x7f800000u) != 0x7f800000u) continue;
                    const float o = __uint_as_float(ld1(col_o + c * 8 + e));
                    tc::ld_wait();
                    st1(col_o + c * 8 + e, __float_as_uint(sees ? o + val : o));
                    tc::st_wait();
                  }
                }
              }
            }
          }
          if (scan) hand_over(tl.p_half[s]);
          hand_over(tl.p_full[s]);
        }
      }
      auto wait_o = [&]() {  // the stream's last product
        if (u.tiles > (two ? 0 : s)) {
          wait(tl.o_full[s], units & 1, abort);
          ++units;
        }
        tc::fence_after();
      };
      if (fine) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          l2[r] += __shfl_xor_sync(0xffffffffu, l2[r], 1);
          l2[r] += __shfl_xor_sync(0xffffffffu, l2[r], 2);
        }
        m = of_row(m2[0], m2[1], lane);
        l = of_row(l2[0], l2[1], lane);
      }
      tile_no += u.tiles;
      if (l == 0.f) m = -INFINITY;  // no key seen: the row counts for nothing where parts are joined
      int own = 32 * (warp % 4) + lane;
      asm volatile("" : "+r"(own));  // the row is worked out here anew: kept through the tiles it would cost registers
      const bool live = own < rows;
      const int r = first_row + own, h = u.kvh * G + p.by_group.rest(r);
      const int64_t token = u.token0 + p.by_group.quotient(r);
      // The accumulator of the row: its stream's, or both halves' of it, each half of the dims by one of the streams.
      float own_c = 1.f, other_c = 0.f;
      int c0 = 0, c1 = HD / 32;
      const bool halves = !two && u.tiles > 1;
      if (halves) {
        wait_o();
        tl.ml[s][own][0] = m;
        tl.ml[s][own][1] = l;
        tc::fence_before();
        meet();
        tc::fence_after();
        const float m2 = tl.ml[1 - s][own][0], l2 = tl.ml[1 - s][own][1];
        const float top = fmaxf(m, m2), mb = top == -INFINITY ? 0.f : top;
        own_c = ex2(m - mb);
        other_c = ex2(m2 - mb);
        l = s == 0 ? l * own_c + l2 * other_c : l2 * other_c + l * own_c;
        m = top;
        c0 = s * (HD / 64);
        c1 = c0 + HD / 64;
      }
      const uint32_t col_other = tlane + L::kColO + (1 - s) * HD;
      // A unit that began here and goes on in other CTAs: they handed their parts over as the first thing they did. With
      // many rows each row adds them to its own accumulator; few rows are joined by all the warps, below.
      const bool few = u.rows <= kFewRows, adds = u.mode == kPart1 && !few;
      float own_w = 1.f;
      if (adds && wait_parts(p, u, cta, lane)) {
        float top = m;
#pragma unroll 4
        for (int i = 1; i < u.parts; ++i) top = fmaxf(top, live ? __ldcg(p.ml + part_slot(cta, i) * 2 * p.rows_max + r) : top);
        const float mb = top == -INFINITY ? 0.f : top;
        own_w = ex2(m - mb);
        l *= own_w;
#pragma unroll 4
        for (int i = 1; i < u.parts; ++i)
          if (live) {
            const float* ml = p.ml + part_slot(cta, i) * 2 * p.rows_max + r;
            l += __ldcg(ml + p.rows_max) * ex2(__ldcg(ml) - mb);
          }
        m = top;
      }
      const bool done = u.mode == kFinal || adds;  // the row's output is formed here
      const float f = l == 0.f ? 0.f : (p.gate ? sigmoid(gate_raw) : 1.f) * reciprocal(l);  // 0 for a row that saw no key; a NaN sum stays NaN
      int64_t rows4[4];  // where the rows go that this lane stores: lane / 4 and every 8th
      {
        const int64_t row = live ? token * p.out_stride + (int64_t)h * hd : -1;
#pragma unroll
        for (int k = 0; k < 4; ++k) rows4[k] = __shfl_sync(0xffffffffu, row, 8 * k + lane / 4);
      }
      if (!halves) wait_o();  // all that does not need it comes before
      if ((two || s == 0 || u.tiles > 1) && !gave_up(abort)) {
        const int64_t part = (int64_t)cta * 2 + (u.mode == kPart1);
        float* acc = p.acc + part * HD * p.rows_max;
        auto chunk = [&](int c) {  // 32 dims of the row's accumulator
          uint32_t o[32] = {};
          if (u.tiles > 0) {
            ld32(col_o + 32 * c, o);
            if (c1 - c0 < HD / 32) {
              uint32_t o2[32];
              ld32(col_other + 32 * c, o2);
              tc::ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float a = __uint_as_float(o[j]) * own_c, z = __uint_as_float(o2[j]) * other_c;
                o[j] = __float_as_uint(s == 0 ? a + z : z + a);
              }
            }
            tc::ld_wait();
          }
          if (adds) {
            const float mb = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * own_w);
#pragma unroll 1
            for (int i = 1; i < u.parts && live; ++i) {
              const float4* a = reinterpret_cast<const float4*>(p.acc + (part_slot(cta, i) * (HD / 4) + 8 * c) * p.rows_max * 4 + r * 4);
              float4 v[8];
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = __ldcg(a + (int64_t)j * p.rows_max);
              const float w = ex2(__ldcg(p.ml + part_slot(cta, i) * 2 * p.rows_max + r) - mb);
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                o[4 * j] = __float_as_uint(fmaf(v[j].x, w, __uint_as_float(o[4 * j])));
                o[4 * j + 1] = __float_as_uint(fmaf(v[j].y, w, __uint_as_float(o[4 * j + 1])));
                o[4 * j + 2] = __float_as_uint(fmaf(v[j].z, w, __uint_as_float(o[4 * j + 2])));
                o[4 * j + 3] = __float_as_uint(fmaf(v[j].w, w, __uint_as_float(o[4 * j + 3])));
              }
            }
          }
          if (done) {
            // packed over the columns that this chunk was read from, so that 4 lanes then hold 64 bytes of a row
            uint32_t w[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {  // column j takes word 4 (j / 2 % 4) + 2 (j / 8) + j % 2 of the chunk
              const int e = 2 * (4 * (j / 2 % 4) + 2 * (j / 8) + j % 2);
              w[j] = l == 0.f ? 0u : to_bf16x2(__uint_as_float(o[e]) * f, __uint_as_float(o[e + 1]) * f);
            }
            tc::st16(col_o + 16 * (c0 + c), w);
          } else if (live) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(acc + ((int64_t)(8 * c + j) * p.rows_max + r) * 4) =
                  make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          }
        };
#pragma unroll 1
        for (int c = c0; c < c1; ++c) chunk(c);
        if (done) {
          tc::st_wait();
#pragma unroll 1
          for (int c = c0; c < c1; ++c) {
            const int dim = 32 * c + 8 * (lane % 4);
            uint32_t w[2][8];
#pragma unroll
            for (int k = 0; k < 2; ++k) ld_across(col_o + 16 * (c0 + c) + ((uint32_t)(16 * k) << 16), w[k]);
            tc::ld_wait();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t* q = w[k / 2] + 2 * (k % 2);
              if (rows4[k] >= 0 && dim < hd)
                *reinterpret_cast<uint4*>(p.out + rows4[k] + dim) = make_uint4(q[0], q[1], q[4], q[5]);
            }
          }
        }
        if (live && c0 == 0) {
          if (!done) {
            p.ml[part * 2 * p.rows_max + r] = m;
            p.ml[(part * 2 + 1) * p.rows_max + r] = l;
          } else if (p.lse) {
            p.lse[token * p.Hq + h] = l == 0.f ? -INFINITY : (m - kShift + log2f(l)) * 0.6931471805599453f;
          }
        }
      }
      tc::fence_before();  // the accumulator's reads come before the next unit's products
      if (u.mode != kFinal) {
        if (!done) __threadfence();
        meet();
        if (u.mode == kPart0) {
          if (tid == 0) raise_flag(p.flags + cta, p.raised);
        } else {
          if (few && wait_parts(p, u, cta, lane)) join_few<HD>(p, u, cta, tid, kShift);
          meet();  // every thread is done with the parts
          if (tid < u.parts - 1) p.flags[cta + 1 + tid] = 0;
        }
      } else if (!two && u.tiles > 1) {
        meet();
      }
    }
  }
  // ---- rows of no request
  const int idle = refused ? 0 : tl.idle[0] + p.kv.N - tl.idle[1];
#pragma unroll 1
  for (int i = cta * (kThreads / 32) + warp; i < idle; i += ctas * (kThreads / 32)) {
    const int64_t t = i < tl.idle[0] ? i : tl.idle[1] + i - tl.idle[0];
#pragma unroll 1
    for (int c = lane; c < p.Hq * hd / 8; c += 32)
      *reinterpret_cast<uint4*>(p.out + t * p.out_stride + c * 8) = make_uint4(0, 0, 0, 0);
    if (p.lse)
#pragma unroll 1
      for (int h = lane; h < p.Hq; h += 32) p.lse[t * p.Hq + h] = -INFINITY;
  }
  tc::fence_before();
  __syncthreads();
  tc::fence_after();
  if (tid == 0 && *abort != 0 && p.status) atomicOr(p.status, zb::kStatusAttnChunkTimeout);
  if (warp == kMmaWarp) tc::dealloc(tmem, 512);
}

// The launch: CTAs, and whether a unit can span several of them.
struct Launch {
  int ctas, rows_max;
  bool splits;
  int64_t flag_bytes, acc_bytes, ml_bytes;
};
Launch plan(int B, int64_t N, int Hq, int Hkv, int hd, int64_t max_keys) {
  Launch l{};
  if (Hkv < 1 || B < 1 || N < 1 || Hq < Hkv || Hq / Hkv > kStreamRows) return l;
  const int G = Hq / Hkv, pair_tokens = 2 * (kStreamRows / G);
  const int64_t tiles = std::max<int64_t>((max_keys + kTile - 1) / kTile, 1);
  const int64_t pairs = N / pair_tokens + std::min<int64_t>(B, N);  // units of a KV head, at most
  l.ctas = (int)std::min<int64_t>(std::min<int64_t>(zb::sm_count(), kFlagBytes / 4), pairs * Hkv * (tiles + kUnitCost2 / kTileCost2));
  l.splits = tiles > 1 && l.ctas > 1;
  l.rows_max = (int)std::min<int64_t>(N, pair_tokens) * G;
  if (l.splits) {
    const int64_t width = hd <= 64 ? 64 : 128;
    l.flag_bytes = kFlagBytes;
    l.acc_bytes = (int64_t)l.ctas * 2 * l.rows_max * width * 4;
    l.ml_bytes = (int64_t)l.ctas * 4 * l.rows_max * 4;
  }
  return l;
}

// Tensor maps: the queries, and over the caches for copies of whole page rows: [64 dims, 8 rows, atoms, row groups, pages], with the KV
// heads folded into the atoms (a row's heads side by side) or the pages (a page's heads one after the other). p.box
// stays 0 where the layout, the page size or the head dim does not allow them.
template <int HD, bool Q4>
int make_maps(ChunkParams& p, Maps& maps) {
  const zb::PagedBatch& c = p.kv;
  auto fn = zb::tcp::encode_fn();
  if (fn == nullptr) return zb::fail(zb::kCudaError, "gqa_chunk: cuTensorMapEncodeTiled unavailable");
  auto encode = [&](CUtensorMap* map, int rank, const void* at, const cuuint64_t* dims, const cuuint64_t* strides,
                    const cuuint32_t* boxes) {
    const cuuint32_t step[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(at), dims, strides, boxes, step,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? zb::kOk : zb::fail(zb::kCudaError, "gqa_chunk: cuTensorMapEncodeTiled failed (%d)", (int)r);
  };
  {  // the queries: [dims, heads, tokens], a box of 64 dims of the group's heads of a stream's tokens
    const cuuint64_t dims[3] = {(cuuint64_t)c.hd, (cuuint64_t)p.Hq, (cuuint64_t)c.N};
    const cuuint64_t strides[2] = {(cuuint64_t)c.hd * 2, (cuuint64_t)p.q_stride * 2};
    const cuuint32_t boxes[3] = {64, (cuuint32_t)p.G, (cuuint32_t)p.tokens};
    ZB_REQUIRE(p.q_stride < (int64_t)1 << 38, "gqa_chunk: q_stride %lld", (long long)p.q_stride);
    if (int rc = encode(&maps.q, 3, p.q, dims, strides, boxes)) return rc;
  }
  if (Q4) {  // blocks come by bulk copies
    p.box = zb::q4::kBlock;
    p.box_shift = 4;
    return zb::kOk;
  }
  p.box = 0;
  int box = 1;
  while (box < kTile && c.page_size % (2 * box) == 0) box *= 2;
  const bool beside = c.head_stride == c.hd || c.Hkv == 1;
  const bool behind = c.page_stride == c.Hkv * c.head_stride && c.num_pages * c.Hkv < INT32_MAX;
  if (box < 8 || c.hd != HD || !(beside || behind) || c.num_pages < 1 || c.num_pages >= INT32_MAX || c.slot_stride < HD ||
      c.page_stride < HD || c.page_stride >= (int64_t)1 << 38 || c.slot_stride >= (int64_t)1 << 34)
    return zb::kOk;
  const int64_t page = beside ? c.page_stride : c.head_stride;
  const cuuint64_t dims[5] = {64, 8, (cuuint64_t)(HD / 64 * (beside ? c.Hkv : 1)), (cuuint64_t)(c.page_size / 8),
                              (cuuint64_t)(c.num_pages * (beside ? 1 : c.Hkv))};
  const cuuint64_t strides[4] = {(cuuint64_t)c.slot_stride * 2, 128, (cuuint64_t)c.slot_stride * 16, (cuuint64_t)page * 2};
  const cuuint32_t boxes[5] = {64, 8, HD / 64, (cuuint32_t)(box / 8), 1};
  if (int rc = encode(&maps.k, 5, c.k, dims, strides, boxes)) return rc;
  if (int rc = encode(&maps.v, 5, c.v, dims, strides, boxes)) return rc;
  p.box = box;
  p.box_shift = __builtin_ctz((unsigned)box);
  p.head_atoms = beside ? HD / 64 : 0;
  p.page_heads = beside ? 1 : c.Hkv;
  return zb::kOk;
}

template <int HD, bool Q4, bool SINKS>
int launch_chunk(ChunkParams& p, const Launch& l, cudaStream_t stream) {
  Maps maps = {};
  if (int rc = make_maps<HD, Q4>(p, maps)) return rc;
  auto kernel = gqa_chunk_kernel<HD, Q4, SINKS>;
  static bool configured[64] = {false};  // the shared-memory attribute, set once per device
  int dev = 0;
  ZB_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    ZB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Shape<HD, Q4>::kSmem));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  ZB_CUDA(zb::launch(kernel, dim3((unsigned)l.ctas), dim3(Shape<HD, Q4>::kThreads), Shape<HD, Q4>::kSmem, stream, 1, p, maps));
  return zb::check_launch("gqa_chunk");
}

// 4 bits: both kernels' flags, then the partial results of whichever runs.
int64_t q4_workspace_bytes(const Launch& l, int B, int N, int Hkv, int hd, int64_t max_keys, int few, bool only_few) {
  const int64_t parts = only_few ? 0 : l.acc_bytes + l.ml_bytes;
  const int64_t few_parts = few > 0 ? zb::q4::few_workspace_bytes(B, N, Hkv, hd, few, max_keys) - zb::q4::kFewFlagBytes : 0;
  return parts + few_parts > 0 ? kFlagBytes + zb::q4::kFewFlagBytes + std::max(parts, few_parts) : 0;
}

// What both caches' entry points do once the cache has been checked; `who` names the entry point.
template <bool Q4>
int chunk(ChunkParams& p, const char* who, const uint16_t* q, int64_t q_stride, int Hq, float softmax_scale, int causal,
          int window, int sinks, int max_new, const uint16_t* gate, int64_t gate_stride, uint16_t* out, int64_t out_stride,
          float* lse, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  const int B = p.kv.B, N = p.kv.N, Hkv = p.kv.Hkv, hd = p.kv.hd;
  ZB_REQUIRE(Hq > 0 && Hq % Hkv == 0, "%s: %d query heads do not group over %d KV heads", who, Hq, Hkv);
  ZB_REQUIRE(softmax_scale > 0.f && softmax_scale < INFINITY, "%s: softmax_scale %g must be positive", who,
             (double)softmax_scale);
  ZB_REQUIRE(window >= 0 && (causal || window == 0), "%s: window %d (>= 0, and only with causal)", who, window);
  ZB_REQUIRE(sinks >= 0, "%s: sinks %d must not be negative", who, sinks);
  ZB_REQUIRE(q_stride >= (int64_t)Hq * hd && q_stride % 8 == 0 && out_stride >= (int64_t)Hq * hd && out_stride % 8 == 0 &&
                 (!gate || gate_stride >= Hq),
             "%s: strides (q %lld, out %lld, gate %lld)", who, (long long)q_stride, (long long)out_stride,
             (long long)gate_stride);
  ZB_REQUIRE((int64_t)N * Hq < (int64_t)1 << 31, "%s: %d tokens x %d heads", who, N, Hq);
  if (Hq / Hkv > kStreamRows)
    return zb::fail(zb::kUnsupported, "%s: %d query heads a KV head (at most %d)", who, Hq / Hkv, kStreamRows);
  if (B > kMaxRequests) return zb::fail(zb::kUnsupported, "%s: %d requests (at most %d)", who, B, kMaxRequests);
  if (N == 0) return zb::kOk;
  ZB_REQUIRE(B > 0, "%s: %d tokens of no request", who, N);
  ZB_REQUIRE(q && out, "%s: null pointer", who);
  ZB_REQUIRE((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) % 16 == 0,
             "%s: q, out and workspace must be 16-byte aligned", who);
  const Launch l = plan(B, N, Hq, Hkv, hd, (int64_t)p.kv.page_size * p.kv.max_pages);
  const int few = Q4 ? zb::q4::few_rows(hd, Hq / Hkv, max_new) : 0;
  const bool only_few = few > 0 && (int64_t)max_new * (Hq / Hkv) <= few;
  const int64_t need = Q4 ? q4_workspace_bytes(l, B, N, Hkv, hd, (int64_t)p.kv.page_size * p.kv.max_pages, few, only_few) : l.flag_bytes + l.acc_bytes + l.ml_bytes;
  ZB_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "%s: a workspace of %lld bytes, got %lld", who,
             (long long)need, (long long)workspace_bytes);
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.Hq = Hq;
  p.G = Hq / Hkv;
  p.tokens = kStreamRows / p.G;
  p.by_page.set(p.kv.page_size);
  p.by_group.set(p.G);
  p.by_pair.set(2 * p.tokens);
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.causal = causal;
  p.window = window;
  p.sinks = window > 0 ? sinks : 0;
  p.few = few;
  p.gate = reinterpret_cast<const __nv_bfloat16*>(gate);
  p.gate_stride = gate_stride;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  p.lse = lse;
  unsigned char* ws = static_cast<unsigned char*>(workspace);
  p.flags = reinterpret_cast<unsigned*>(ws);
  static std::atomic<unsigned> calls{0};
  do p.raised = calls.fetch_add(1, std::memory_order_relaxed) + 1;
  while (p.raised == 0);
  unsigned char* parts = ws + (Q4 ? kFlagBytes + zb::q4::kFewFlagBytes : l.flag_bytes);
  p.acc = reinterpret_cast<float*>(parts);
  p.ml = reinterpret_cast<float*>(parts + l.acc_bytes);
  p.rows_max = l.rows_max;
  p.status = zb::device_status_ptr();
  if (Q4 && few > 0) {
    const zb::q4::FewCall call{p.kv, p.q, q_stride, Hq, p.scale_log2, causal, window, p.sinks, few, only_few, p.gate,
                               gate_stride, p.out, out_stride, lse, ws + kFlagBytes};
    const int rc = zb::q4::launch_few(call, stream);
    if (rc != zb::kOk || only_few) return rc;
  }
  if constexpr (!Q4)
    if (p.sinks == 0) return hd <= 64 ? launch_chunk<64, false, false>(p, l, stream) : launch_chunk<128, false, false>(p, l, stream);
  return hd <= 64 ? launch_chunk<64, Q4, true>(p, l, stream) : launch_chunk<128, Q4, true>(p, l, stream);
}

}  // namespace

ZB_API int64_t zb_gqa_chunk_workspace_bytes(int B, int N, int Hq, int Hkv, int hd, int64_t max_keys) {
  const Launch l = plan(B, N, Hq, Hkv, hd, max_keys);
  return l.flag_bytes + l.acc_bytes + l.ml_bytes;
}

ZB_API int zb_gqa_chunk_sinks(const uint16_t* q, int64_t q_stride, const uint16_t* k_cache, const uint16_t* v_cache,
                              int64_t page_stride, int64_t slot_stride, int64_t head_stride, int64_t num_pages,
                              int page_size, const int32_t* page_table, int64_t table_stride, int max_pages,
                              const int32_t* cache_seqlens, const int32_t* cu_seqlens_q, int B, int N, int Hq, int Hkv,
                              int hd, float softmax_scale, int causal, int window, int sinks, const uint16_t* gate,
                              int64_t gate_stride, uint16_t* out, int64_t out_stride, float* lse, void* workspace,
                              int64_t workspace_bytes, cudaStream_t stream) {
  ChunkParams p;
  p.kv = zb::PagedBatch{reinterpret_cast<__nv_bfloat16*>(const_cast<uint16_t*>(k_cache)),
                        reinterpret_cast<__nv_bfloat16*>(const_cast<uint16_t*>(v_cache)), page_stride, slot_stride,
                        head_stride, num_pages, page_size, page_table, table_stride, max_pages, cache_seqlens,
                        cu_seqlens_q, B, N, Hkv, hd};
  if (int rc = zb::check_paged(p.kv, "gqa_chunk")) return rc;
  return chunk<false>(p, "gqa_chunk", q, q_stride, Hq, softmax_scale, causal, window, sinks, 0, gate, gate_stride, out,
                      out_stride, lse, workspace, workspace_bytes, stream);
}

ZB_API int zb_gqa_chunk(const uint16_t* q, int64_t q_stride, const uint16_t* k_cache, const uint16_t* v_cache,
                        int64_t page_stride, int64_t slot_stride, int64_t head_stride, int64_t num_pages, int page_size,
                        const int32_t* page_table, int64_t table_stride, int max_pages, const int32_t* cache_seqlens,
                        const int32_t* cu_seqlens_q, int B, int N, int Hq, int Hkv, int hd, float softmax_scale,
                        int causal, int window, const uint16_t* gate, int64_t gate_stride, uint16_t* out,
                        int64_t out_stride, float* lse, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  return zb_gqa_chunk_sinks(q, q_stride, k_cache, v_cache, page_stride, slot_stride, head_stride, num_pages, page_size,
                            page_table, table_stride, max_pages, cache_seqlens, cu_seqlens_q, B, N, Hq, Hkv, hd,
                            softmax_scale, causal, window, 0, gate, gate_stride, out, out_stride, lse, workspace,
                            workspace_bytes, stream);
}

ZB_API int64_t zb_gqa_chunk_q4_workspace_bytes(int B, int N, int Hq, int Hkv, int hd, int64_t max_keys, int max_new) {
  const Launch l = plan(B, N, Hq, Hkv, hd, max_keys);
  if (l.ctas == 0) return 0;
  max_new = max_new > 0 ? std::min(max_new, N) : N;
  const int few = zb::q4::few_rows(hd, Hq / Hkv, max_new);
  return q4_workspace_bytes(l, B, N, Hkv, hd, max_keys, few, few > 0 && (int64_t)max_new * (Hq / Hkv) <= few);
}

ZB_API int zb_gqa_chunk_q4(const uint16_t* q, int64_t q_stride, const uint8_t* kv_cache, int64_t page_stride,
                           int64_t head_stride, int64_t num_pages, int page_size, const int32_t* page_table,
                           int64_t table_stride, int max_pages, const int32_t* cache_seqlens, const int32_t* cu_seqlens_q,
                           int B, int N, int Hq, int Hkv, int hd, float softmax_scale, int causal, int window, int sinks,
                           int max_new, const uint16_t* gate, int64_t gate_stride, uint16_t* out, int64_t out_stride,
                           float* lse, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  ChunkParams p;
  p.kv = zb::PagedBatch{reinterpret_cast<__nv_bfloat16*>(const_cast<uint8_t*>(kv_cache)), nullptr, page_stride, 0,
                        head_stride, num_pages, page_size, page_table, table_stride, max_pages, cache_seqlens,
                        cu_seqlens_q, B, N, Hkv, hd};
  if (int rc = zb::q4::check_cache(p.kv, "gqa_chunk_q4")) return rc;
  ZB_REQUIRE(max_new >= 0, "gqa_chunk_q4: max_new %d must not be negative", max_new);
  return chunk<true>(p, "gqa_chunk_q4", q, q_stride, Hq, softmax_scale, causal, window, sinks,
                     max_new > 0 ? std::min(max_new, N) : N, gate, gate_stride, out, out_stride, lse, workspace,
                     workspace_bytes, stream);
}
