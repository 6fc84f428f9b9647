// Attention of every request's new tokens over its pages of a KV cache.
//
// Token t of request b at key position p (paged.cuh) sees the keys j <= p (causal; every key of the request otherwise)
// with j > p - window when there is a window, and whose page is in the cache. With s_j = scale q . k_j over them,
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  m = max_j s_j,  lse = m + log sum_j e^(s_j - m);
// a token that sees no key, or belongs to no request, gives 0 (lse -inf). Query head h reads KV head h / (Hq / Hkv).
// The layer's output gate multiplies head h's row by sigmoid(gate[t, h]) before the one rounding to bf16.
//
// A warp per (token, query head): groups of lanes, 8 elements each, take the keys in turn with their own running
// maximum, sum and accumulator, joined at the end. All in fp32.
#include "paged.cuh"

namespace {

constexpr int kWarps = 4;

struct ChunkParams {
  zb::PagedBatch kv;
  const __nv_bfloat16* q;  // [N, Hq, hd], row stride q_stride
  int64_t q_stride;
  int Hq;
  float scale_log2;  // softmax scale * log2(e)
  int causal, window;
  const __nv_bfloat16* gate;  // [N, Hq] or null
  int64_t gate_stride;
  __nv_bfloat16* out;  // [N, Hq, hd]
  int64_t out_stride;
  float* lse;  // [N, Hq] or null
};

template <int GL>
__global__ void __launch_bounds__(kWarps * 32) gqa_chunk_kernel(const __grid_constant__ ChunkParams p) {
  zb::pdl_enter();
  constexpr int kKeys = 32 / GL;
  const int64_t unit = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  const int lane = threadIdx.x % 32, gl = lane % GL, kl = lane / GL;
  if (unit >= (int64_t)p.kv.N * p.Hq) return;
  const int t = (int)(unit / p.Hq), h = (int)(unit % p.Hq), kvh = h / (p.Hq / p.kv.Hkv);
  const int hd = p.kv.hd;
  const bool carries = gl * 8 < hd;
  const int b = zb::request_of(p.kv.cu, p.kv.B, t, lane);
  float m = -INFINITY, l = 0.f, acc[8] = {};
  if (b >= 0) {
    const int64_t keys = p.kv.keys[b], pos = keys - ((int64_t)p.kv.cu[b + 1] - t);
    const int64_t capacity = (int64_t)p.kv.max_pages * p.kv.page_size;
    int64_t end = p.causal ? pos + 1 : keys, begin = p.window > 0 ? pos + 1 - p.window : 0;
    if (end > keys) end = keys;
    if (end > capacity) end = capacity;
    if (begin < 0) begin = 0;
    float q[8] = {};
    if (carries) zb::ld_bf16x8(p.q + (int64_t)t * p.q_stride + (int64_t)h * hd + gl * 8, q);
    for (int64_t j0 = begin; j0 < end; j0 += kKeys) {
      const int64_t j = j0 + kl;
      bool sees = j < end;
      int page = -1;
      if (sees) page = p.kv.table[(int64_t)b * p.kv.table_stride + j / p.kv.page_size];
      sees = page >= 0 && page < p.kv.num_pages;
      float k[8] = {}, v[8] = {};
      if (sees && carries) {
        const int64_t at = (int64_t)page * p.kv.page_stride + (int64_t)(j % p.kv.page_size) * p.kv.slot_stride +
                           (int64_t)kvh * p.kv.head_stride + gl * 8;
        zb::ld_bf16x8(p.kv.k + at, k);
        zb::ld_bf16x8(p.kv.v + at, v);
      }
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(q[i], k[i], s);
#pragma unroll
      for (int o = GL / 2; o > 0; o /= 2) s += __shfl_xor_sync(0xffffffffu, s, o);
      if (!sees) continue;
      s *= p.scale_log2;
      const float m_new = fmaxf(m, s), corr = exp2f(m - m_new), e = exp2f(s - m_new);
      l = l * corr + e;
      m = m_new;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] = acc[i] * corr + e * v[i];
    }
  }
#pragma unroll
  for (int o = GL; o < 32; o *= 2) {  // join the key groups
    const float m2 = __shfl_xor_sync(0xffffffffu, m, o), l2 = __shfl_xor_sync(0xffffffffu, l, o);
    const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
    const float c1 = exp2f(m - base), c2 = exp2f(m2 - base);
    l = l * c1 + l2 * c2;
    m = top;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = acc[i] * c1 + __shfl_xor_sync(0xffffffffu, acc[i], o) * c2;
  }
  float f = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;  // a NaN sum stays one
  if (p.gate) f *= 1.f / (1.f + expf(-__bfloat162float(p.gate[(int64_t)t * p.gate_stride + h])));
  if (kl == 0 && carries) {
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = acc[i] * f;
    *reinterpret_cast<uint4*>(p.out + (int64_t)t * p.out_stride + (int64_t)h * hd + gl * 8) = zb::pack_bf16x8(y);
  }
  if (p.lse && lane == 0)
    p.lse[(int64_t)t * p.Hq + h] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

}  // namespace

ZB_API int64_t zb_gqa_chunk_workspace_bytes(int B, int N, int Hq, int Hkv, int hd, int64_t max_keys) {
  return 0;
}

ZB_API int zb_gqa_chunk(const uint16_t* q, int64_t q_stride, const uint16_t* k_cache, const uint16_t* v_cache,
                        int64_t page_stride, int64_t slot_stride, int64_t head_stride, int64_t num_pages, int page_size,
                        const int32_t* page_table, int64_t table_stride, int max_pages, const int32_t* cache_seqlens,
                        const int32_t* cu_seqlens_q, int B, int N, int Hq, int Hkv, int hd, float softmax_scale,
                        int causal, int window, const uint16_t* gate, int64_t gate_stride, uint16_t* out,
                        int64_t out_stride, float* lse, void* workspace, int64_t workspace_bytes, cudaStream_t stream) {
  ChunkParams p;
  p.kv = zb::PagedBatch{reinterpret_cast<__nv_bfloat16*>(const_cast<uint16_t*>(k_cache)),
                        reinterpret_cast<__nv_bfloat16*>(const_cast<uint16_t*>(v_cache)), page_stride, slot_stride,
                        head_stride, num_pages, page_size, page_table, table_stride, max_pages, cache_seqlens,
                        cu_seqlens_q, B, N, Hkv, hd};
  if (int rc = zb::check_paged(p.kv, "gqa_chunk")) return rc;
  ZB_REQUIRE(Hq > 0 && Hq % Hkv == 0, "gqa_chunk: %d query heads do not group over %d KV heads", Hq, Hkv);
  ZB_REQUIRE(softmax_scale > 0.f && softmax_scale < INFINITY, "gqa_chunk: softmax_scale %g must be positive",
             (double)softmax_scale);
  ZB_REQUIRE(window >= 0 && (causal || window == 0), "gqa_chunk: window %d (>= 0, and only with causal)", window);
  ZB_REQUIRE(q_stride >= (int64_t)Hq * hd && q_stride % 8 == 0 && out_stride >= (int64_t)Hq * hd && out_stride % 8 == 0 &&
                 (!gate || gate_stride >= Hq),
             "gqa_chunk: strides (q %lld, out %lld, gate %lld)", (long long)q_stride, (long long)out_stride,
             (long long)gate_stride);
  if (N == 0) return zb::kOk;
  ZB_REQUIRE(B > 0, "gqa_chunk: %d tokens of no request", N);
  ZB_REQUIRE(q && out, "gqa_chunk: null pointer");
  ZB_REQUIRE_ALIGNED(q, 16, "gqa_chunk q");
  ZB_REQUIRE_ALIGNED(out, 16, "gqa_chunk out");
  p.q = reinterpret_cast<const __nv_bfloat16*>(q);
  p.q_stride = q_stride;
  p.Hq = Hq;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.causal = causal;
  p.window = window;
  p.gate = reinterpret_cast<const __nv_bfloat16*>(gate);
  p.gate_stride = gate_stride;
  p.out = reinterpret_cast<__nv_bfloat16*>(out);
  p.out_stride = out_stride;
  p.lse = lse;
  const dim3 grid((unsigned)(((int64_t)N * Hq + kWarps - 1) / kWarps)), block(kWarps * 32);
  const int lanes = hd / 8;
  cudaError_t err = lanes <= 4   ? zb::launch(gqa_chunk_kernel<4>, grid, block, 0, stream, 1, p)
                    : lanes <= 8 ? zb::launch(gqa_chunk_kernel<8>, grid, block, 0, stream, 1, p)
                                 : zb::launch(gqa_chunk_kernel<16>, grid, block, 0, stream, 1, p);
  ZB_CUDA(err);
  return zb::check_launch("gqa_chunk");
}
