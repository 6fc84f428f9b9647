// A ragged batch over a paged KV cache, as the append and the chunk attention see it.
//
// Token t of the batch's N new tokens belongs to request b when cu[b] <= t < cu[b + 1] (cu has B + 1 entries and does
// not decrease); request b has keys[b] keys, its new tokens among them as the last ones, so token t stands at key
// position keys[b] - (cu[b + 1] - t). Position j of request b lies in row j % page_size of page
// table[b * table_stride + j / page_size]; a page outside [0, num_pages) or past the table's columns holds no keys.
#pragma once

#include "common.cuh"

namespace zb {

struct PagedBatch {
  __nv_bfloat16* k;  // page p, row r, KV head h at p * page_stride + r * slot_stride + h * head_stride
  __nv_bfloat16* v;
  int64_t page_stride, slot_stride, head_stride;
  int64_t num_pages;
  int page_size;
  const int32_t* table;
  int64_t table_stride;
  int max_pages;
  const int32_t* keys;  // [B]
  const int32_t* cu;    // [B + 1]
  int B, N, Hkv, hd;
};

// Checks what every entry point over a paged batch asks of it; `who` names the entry point.
inline int check_paged(const PagedBatch& p, const char* who) {
  ZB_REQUIRE(p.B >= 0 && p.N >= 0 && p.Hkv > 0 && p.num_pages >= 0 && p.max_pages >= 0, "%s: negative sizes", who);
  if (p.hd < 8 || p.hd > 128 || p.hd % 8 != 0)
    return fail(kUnsupported, "%s: head dim %d (a multiple of 8 up to 128)", who, p.hd);
  ZB_REQUIRE(p.page_size >= 1 && (int64_t)p.page_size * p.max_pages <= (int64_t)1 << 26,
             "%s: page size %d x %d table columns (at most 2^26 keys)", who, p.page_size, p.max_pages);
  ZB_REQUIRE(p.page_stride % 8 == 0 && p.slot_stride % 8 == 0 && p.head_stride % 8 == 0 && p.page_stride >= 0 &&
                 p.slot_stride >= 0 && p.head_stride >= 0,
             "%s: cache strides (page %lld, row %lld, head %lld) must be multiples of 8", who, (long long)p.page_stride,
             (long long)p.slot_stride, (long long)p.head_stride);
  ZB_REQUIRE(p.table_stride >= p.max_pages || p.B <= 1, "%s: table stride %lld < %d columns", who,
             (long long)p.table_stride, p.max_pages);
  if (p.B == 0 || p.N == 0) return kOk;
  ZB_REQUIRE(p.cu && p.keys && (p.table || p.max_pages == 0) && ((p.k && p.v) || p.num_pages == 0), "%s: null pointer",
             who);
  ZB_REQUIRE((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) % 16 == 0,
             "%s: the K and V caches must be 16-byte aligned", who);
  return kOk;
}

// The request of token t, found by the whole warp: 32 probes of cu at a time cut the range by 32 per round. Returns
// -1 for a token of no request (before cu[0] or from cu[B] on).
__device__ __forceinline__ int request_of(const int32_t* cu, int B, int t, int lane) {
  int lo = 0, hi = B + 1;  // the count of entries <= t lies in [lo, hi]
  while (hi - lo > 0) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + (lane + 1) * step - 1;  // the last entry of the lane's piece
    const bool below = i < hi && cu[i] <= t;
    const int pieces = __popc(__ballot_sync(0xffffffffu, below));
    const int next = lo + pieces * step;
    hi = min(hi, next + step - 1);
    lo = min(next, hi);
    if (step == 1) break;
  }
  return lo - 1 < B ? lo - 1 : -1;
}

}  // namespace zb
