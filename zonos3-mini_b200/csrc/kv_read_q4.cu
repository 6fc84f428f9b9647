// Keys and values of a ragged batch read back from a KV cache of 4 bits (kv_q4.cuh), as rows of bf16.
//
// Row t of request b (paged.cuh) is its key position keys[b] - (cu[b + 1] - t), as for the tokens that the append writes: the
// last cu[b + 1] - cu[b] keys of every request. k_out[t, h] and v_out[t, h] get m + s c of head h's groups, rounded once; rows
// of no request, and keys whose page is outside the cache or past the table, get zeros.
//
// Bound by HBM: 1.25 hd bytes in and 4 hd out per key and KV head. A warp takes a few tokens; its lanes find their pages
// together, then hold a word of codes each (8 elements of one group), so that a row's codes are read in order and its 16-byte
// pieces leave in whole lines. The pair of a word is read beside it.
//
// Measured (B200): 65536 keys of 4 KV heads of 128 (176 MB) 34 us, 5.2 TB/s, 0.79 of a copy's 6.55. Short runs keep the lines that
// neighbouring warps write close together in time: 4 tokens a warp 39.7, 8 42.0, 16 47.3; with stores that do not stay in the L2
// 34.1 and 37.4. Four words a lane in flight: two 50, eight 47. 800 keys of a ragged batch 5 us.
#include <algorithm>

#include "kv_q4.cuh"

namespace {

constexpr int kWarps = 4, kRun = 4, kTogether = 4;

struct ReadParams {
  zb::PagedBatch kv;  // a cache of 4 bits
  __nv_bfloat16* k_out;  // [N, Hkv, hd], row stride k_stride
  __nv_bfloat16* v_out;
  int64_t k_stride, v_stride;
  int run;  // tokens of a warp
};

template <int GROUPS>
__global__ void __launch_bounds__(kWarps * 32) kv_read_q4_kernel(const __grid_constant__ ReadParams p) {
  zb::pdl_enter();
  constexpr int kHd = GROUPS * zb::q4::kGroup, kWords = 4 * GROUPS, kRows = 32 / kWords;  // rows (heads' keys or values) of a pass
  const int lane = threadIdx.x % 32;
  const int64_t t0 = ((int64_t)blockIdx.x * kWarps + threadIdx.x / 32) * p.run;
  if (t0 >= p.kv.N) return;
  const int tokens = (int)min((int64_t)p.run, p.kv.N - t0);
  // lane i: where token t0 + i's rows lie
  int64_t block = -1;
  int in = 0;
  {
    int b = zb::request_of(p.kv.cu, p.kv.B, (int)t0, lane);
    const int t = (int)t0 + lane;
    if (b < 0) b = 0;  // before the first request, or behind the last one
    if (b < p.kv.B && p.kv.cu[b + 1] <= t) {
      if (p.kv.cu[p.kv.B] <= t) b = p.kv.B;  // nothing to look for, through whatever requests without rows
      while (b < p.kv.B && p.kv.cu[b + 1] <= t) ++b;
    }
    if (lane < tokens && b < p.kv.B && p.kv.cu[b] <= t) {
      const int64_t pos = (int64_t)p.kv.keys[b] - ((int64_t)p.kv.cu[b + 1] - t);
      if (pos >= 0 && pos / p.kv.page_size < p.kv.max_pages) {
        const int page = p.kv.table[(int64_t)b * p.kv.table_stride + pos / p.kv.page_size];
        const int row = (int)(pos % p.kv.page_size);
        if (page >= 0 && page < p.kv.num_pages)
          block = (int64_t)page * p.kv.page_stride + (int64_t)(row / zb::q4::kBlock) * zb::q4::block_bytes(kHd);
        in = row % zb::q4::kBlock;
      }
    }
  }
  const int word = lane % kWords, sub = lane / kWords, group = word % GROUPS, part = word / GROUPS;
  const bool takes = sub < kRows;
  const int heads = p.kv.Hkv;
  const unsigned char* cache = reinterpret_cast<const unsigned char*>(p.kv.k);
  // rows r of the run's tokens (a key's heads, then a value's) together: what depends on r alone is formed once for them
#pragma unroll 1
  for (int r = sub; r - sub < 2 * heads; r += kRows) {
    const bool mine = takes && r < 2 * heads, value = r >= heads;
    const int h = value ? r - heads : r;
    const unsigned char* from = cache + (int64_t)h * p.kv.head_stride + (value ? 8 : 0) * kHd + 4 * word;
    const int to_pairs = (value ? 10 : 16) * kHd + 4 * (group - word);
    const int64_t stride = value ? p.v_stride : p.k_stride;
    __nv_bfloat16* to = (value ? p.v_out : p.k_out) + t0 * stride + (int64_t)h * kHd + 32 * group + 8 * part;
#pragma unroll 1
    for (int i = 0; i < tokens; i += kTogether, to += kTogether * stride) {
      uint32_t words[kTogether], pairs[kTogether];
#pragma unroll
      for (int k = 0; k < kTogether; ++k) {
        const int64_t at = __shfl_sync(0xffffffffu, block, min(i + k, 31));
        const int row_in = __shfl_sync(0xffffffffu, in, min(i + k, 31));
        words[k] = pairs[k] = 0;
        if (mine && i + k < tokens && at >= 0) {
          words[k] = __ldcs(reinterpret_cast<const uint32_t*>(from + at + row_in * (kHd / 2)));
          pairs[k] = __ldcs(reinterpret_cast<const uint32_t*>(from + at + to_pairs + row_in * 4 * GROUPS));
        }
      }
#pragma unroll
      for (int k = 0; k < kTogether; ++k)
        if (mine && i + k < tokens)
          __stcs(reinterpret_cast<uint4*>(to + k * stride),
                 zb::q4::read_word(words[k], zb::q4::pair_is_none(pairs[k]) ? 0u : pairs[k]));
    }
  }
}

}  // namespace

ZB_API int zb_kv_read_q4(const uint8_t* kv_cache, int64_t page_stride, int64_t head_stride, int64_t num_pages, int page_size,
                         const int32_t* page_table, int64_t table_stride, int max_pages, const int32_t* cache_seqlens,
                         const int32_t* cu_seqlens, int B, int N, int Hkv, int hd, uint16_t* k_out, int64_t k_stride,
                         uint16_t* v_out, int64_t v_stride, cudaStream_t stream) {
  ReadParams p;
  p.kv = zb::PagedBatch{reinterpret_cast<__nv_bfloat16*>(const_cast<uint8_t*>(kv_cache)), nullptr, page_stride, 0,
                        head_stride, num_pages, page_size, page_table, table_stride, max_pages, cache_seqlens,
                        cu_seqlens, B, N, Hkv, hd};
  if (int rc = zb::q4::check_cache(p.kv, "kv_read_q4")) return rc;
  ZB_REQUIRE(k_stride >= (int64_t)Hkv * hd && k_stride % 8 == 0 && v_stride >= (int64_t)Hkv * hd && v_stride % 8 == 0,
             "kv_read_q4: strides (k %lld, v %lld)", (long long)k_stride, (long long)v_stride);
  if (N == 0) return zb::kOk;
  ZB_REQUIRE(B > 0, "kv_read_q4: %d rows of no request", N);
  ZB_REQUIRE(k_out && v_out, "kv_read_q4: null pointer");
  ZB_REQUIRE_ALIGNED(k_out, 16, "kv_read_q4 k_out");
  ZB_REQUIRE_ALIGNED(v_out, 16, "kv_read_q4 v_out");
  p.k_out = reinterpret_cast<__nv_bfloat16*>(k_out);
  p.v_out = reinterpret_cast<__nv_bfloat16*>(v_out);
  p.k_stride = k_stride;
  p.v_stride = v_stride;
  // runs of tokens share the search for their request; shorter ones while there are warps to fill
  p.run = std::max(1, std::min<int>(kRun, N / (zb::sm_count() * 32)));
  const int64_t warps = ((int64_t)N + p.run - 1) / p.run;
  const dim3 grid((unsigned)((warps + kWarps - 1) / kWarps)), block(kWarps * 32);
  cudaError_t err = cudaSuccess;
  switch (hd / zb::q4::kGroup) {
    case 1: err = zb::launch(kv_read_q4_kernel<1>, grid, block, 0, stream, 1, p); break;
    case 2: err = zb::launch(kv_read_q4_kernel<2>, grid, block, 0, stream, 1, p); break;
    case 3: err = zb::launch(kv_read_q4_kernel<3>, grid, block, 0, stream, 1, p); break;
    default: err = zb::launch(kv_read_q4_kernel<4>, grid, block, 0, stream, 1, p); break;
  }
  ZB_CUDA(err);
  return zb::check_launch("kv_read_q4");
}
