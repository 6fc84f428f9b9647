// New tokens' keys and values into a paged cache, with the q / k normalisation and the rotary embedding on the way.
//
// Per token and head row x of hd elements of the fused projection (q | k | v):
//   q, k:  x <- x / sqrt(mean(x^2) + eps)                       (when normalize)
//   q:     x <- x |temp_h|                                      (when temp is given)
//   q, k:  pair j of the first `rotary` elements turns by position * theta^(-2j / rotary); the pair is (2j, 2j + 1)
//          (interleaved) or (j, j + rotary / 2)
// q goes to q_out, k and v to the token's row of its request's pages. Everything is fp32 with one rounding to bf16 at
// the end. The angle is formed as a fraction of a turn in 64-bit fixed point (position times the frequency's fraction,
// whole turns dropping out of the top), so that it is as good at position 10^6 as at 10: in fp32 the product would lose
// a bit of the angle with every doubling of the position. Its sine and cosine are the fast ones, within 2^-20 on
// [-pi, pi]; the result keeps 8 bits.
//
// Each element is read once and written once, so the kernel is bound by HBM; a call of a few tokens is bound by its
// latency: the token's request and page come from dependent loads (cu, keys, page table), which run while the
// projection row's loads are in flight. A warp takes a token (or a share of its heads when there are few tokens): a
// group of lanes, 8 elements each, holds a head, so a warp moves 512 bytes an instruction and turns its lanes' pairs by
// sines and cosines that it computes once for all heads.
//
// Measured (B200): 16210 tokens of 16 query and 4 KV heads of 128 (199 MB) 45 us, 4.4 TB/s, 0.68 of a copy's 6.46: the
// schedulers issue in 65 % of the cycles, a norm, a turn and a rounding for every element, where a copy would issue in few.
// Four warps a block and four passes of heads in flight is the best of 2-8 by 1-8; several tokens to a warp (64-66 us) and
// a token over several warps (66-75) are slower there. 256 single tokens 5.5 us, one 3.4.
#include <cmath>

#include "paged.cuh"

namespace {

constexpr int kWarps = 4;
constexpr int kMaxPairs = 64;

struct AppendParams {
  zb::PagedBatch kv;
  const __nv_bfloat16* proj;  // [N, Hq * hd | Hkv * hd | Hkv * hd | ...], row stride proj_stride
  int64_t proj_stride;
  const __nv_bfloat16* temp;  // [Hq] or null
  const int32_t* positions;   // [N] rotary positions, or null: the key positions
  __nv_bfloat16* q_out;       // [N, Hq, hd], row stride q_stride
  int64_t q_stride;
  float eps;
  int normalize, interleaved, rotary, Hq;
  int shares;              // warps of a token
  float inv_hd;
  uint64_t turns[kMaxPairs];  // the fraction of theta^(-2j / rotary) / (2 pi), times 2^64
};

// 8 consecutive elements from an address aligned to ALIGN bytes.
template <int ALIGN>
__device__ __forceinline__ uint4 load8(const __nv_bfloat16* p) {
  if constexpr (ALIGN == 16) {
    return __ldcs(reinterpret_cast<const uint4*>(p));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (ALIGN == 4) {
        w[i] = reinterpret_cast<const uint32_t*>(p)[i];
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + 2 * i;
        w[i] = (uint32_t)h[0] | ((uint32_t)h[1] << 16);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ void widen(const uint4& r, float (&x)[8]) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

// GL lanes hold a head (hd / 8 of them carry elements).
template <int GL, int ALIGN>
__global__ void __launch_bounds__(kWarps * 32) gqa_append_kernel(const __grid_constant__ AppendParams p) {
  zb::pdl_enter();
  constexpr int kHeads = 32 / GL;  // heads of a pass
  constexpr int kBatch = 4;        // passes whose loads are in flight together
  const int64_t unit = (int64_t)blockIdx.x * kWarps + threadIdx.x / 32;
  const int lane = threadIdx.x % 32, gl = lane % GL;
  const int t = (int)(unit / p.shares), share = (int)(unit % p.shares);
  if (t >= p.kv.N) return;
  const int hd = p.kv.hd, heads = p.Hq + 2 * p.kv.Hkv;
  const bool carries = gl * 8 < hd;
  const int first = share * kHeads + lane / GL, step = p.shares * kHeads;
  const __nv_bfloat16* row = p.proj + (int64_t)t * p.proj_stride + gl * 8;

  uint4 raw[kBatch];
  auto fetch = [&](int h0) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i * step;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (carries && h < heads) raw[i] = load8<ALIGN>(row + (int64_t)h * hd);
    }
  };
  fetch(first);

  const int b = zb::request_of(p.kv.cu, p.kv.B, t, lane);
  int64_t slot = -1;  // offset of the token's cache row
  int at = 0;
  if (b >= 0) {
    const int pos = (int)((int64_t)p.kv.keys[b] - ((int64_t)p.kv.cu[b + 1] - t));
    at = pos;
    if (pos >= 0 && pos / p.kv.page_size < p.kv.max_pages) {
      const int page = p.kv.table[(int64_t)b * p.kv.table_stride + pos / p.kv.page_size];
      if (page >= 0 && page < p.kv.num_pages)
        slot = (int64_t)page * p.kv.page_stride + (int64_t)(pos % p.kv.page_size) * p.kv.slot_stride;
    }
  }
  if (p.positions) at = p.positions[t];
  // the lane's rotation: interleaved, pairs gl * 4 ..; halves, the 8 pairs its elements belong to
  float cs[8], sn[8];
  const int half = p.rotary / 2;
  const bool turned = gl * 8 < p.rotary && b >= 0;
  const bool upper = !p.interleaved && gl * 8 >= half;  // the lane holds second elements of its pairs
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    cs[i] = 1.f;
    sn[i] = 0.f;
    const int e = gl * 8 + i;
    const int pair = p.interleaved ? e / 2 : (upper ? e - half : e);
    if ((p.interleaved && i % 2) || !turned) continue;
    const int turn = (int)(((uint64_t)(int64_t)at * p.turns[pair]) >> 32);  // of 2^32
    __sincosf((float)turn * 1.4629180792671596e-9f, &sn[i], &cs[i]);          // 2 pi / 2^32
  }

  for (int h0 = first; h0 < heads + lane / GL; h0 += kBatch * step) {  // every lane of the warp takes the same turns
    if (h0 != first) fetch(h0);
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int h = h0 + i * step;
      if (h - lane / GL >= heads) break;  // warp-uniform
      const bool is_v = h >= p.Hq + p.kv.Hkv, is_q = h < p.Hq;
      if (h - lane / GL >= p.Hq + p.kv.Hkv) {  // values only, for the whole warp: a copy
        if (carries && h < heads && slot >= 0)
          *reinterpret_cast<uint4*>(p.kv.v + slot + (int64_t)(h - p.Hq - p.kv.Hkv) * p.kv.head_stride + gl * 8) = raw[i];
        continue;
      }
      float x[8], factor = 1.f;
      widen(raw[i], x);
      if (p.normalize) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], ss);
#pragma unroll
        for (int o = GL / 2; o > 0; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        factor = rsqrtf(fmaf(ss, p.inv_hd, p.eps));
      }
      if (is_q && p.temp) factor *= fabsf(__bfloat162float(p.temp[h]));
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] *= factor;
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          if (!turned) break;
          const float a = x[j], c = x[j + 1];
          x[j] = a * cs[j] - c * sn[j];
          x[j + 1] = a * sn[j] + c * cs[j];
        }
      } else {
        const int partner = lane + (upper ? -(half / 8) : half / 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float other = __shfl_sync(0xffffffffu, x[j], turned ? partner : lane);
          if (turned) x[j] = upper ? other * sn[j] + x[j] * cs[j] : x[j] * cs[j] - other * sn[j];
        }
      }
      if (!carries || h >= heads) continue;
      const uint4 packed = is_v ? raw[i] : zb::pack_bf16x8(x);
      if (is_q) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(p.q_out + (int64_t)t * p.q_stride + (int64_t)h * hd + gl * 8) = b >= 0 ? packed : zero;
      } else if (slot >= 0) {
        __nv_bfloat16* cache = is_v ? p.kv.v : p.kv.k;
        const int g = h - p.Hq - (is_v ? p.kv.Hkv : 0);
        *reinterpret_cast<uint4*>(cache + slot + (int64_t)g * p.kv.head_stride + gl * 8) = packed;
      }
    }
  }
}

template <int GL>
cudaError_t launch_append(const AppendParams& p, int align, cudaStream_t stream) {
  const int64_t units = (int64_t)p.kv.N * p.shares;
  const dim3 grid((unsigned)((units + kWarps - 1) / kWarps)), block(kWarps * 32);
  if (align >= 16) return zb::launch(gqa_append_kernel<GL, 16>, grid, block, 0, stream, 1, p);
  if (align >= 4) return zb::launch(gqa_append_kernel<GL, 4>, grid, block, 0, stream, 1, p);
  return zb::launch(gqa_append_kernel<GL, 2>, grid, block, 0, stream, 1, p);
}

}  // namespace

ZB_API int zb_gqa_append(const uint16_t* proj, int64_t proj_stride, const uint16_t* temp, const int32_t* positions,
                         float eps, int normalize, double rope_theta, int rotary_dim, int interleaved, uint16_t* q_out,
                         int64_t q_stride, uint16_t* k_cache, uint16_t* v_cache, int64_t page_stride,
                         int64_t slot_stride, int64_t head_stride, int64_t num_pages, int page_size,
                         const int32_t* page_table, int64_t table_stride, int max_pages, const int32_t* cache_seqlens,
                         const int32_t* cu_seqlens_q, int B, int N, int Hq, int Hkv, int hd, cudaStream_t stream) {
  AppendParams p;
  p.kv = zb::PagedBatch{reinterpret_cast<__nv_bfloat16*>(k_cache), reinterpret_cast<__nv_bfloat16*>(v_cache),
                        page_stride, slot_stride, head_stride, num_pages, page_size, page_table, table_stride,
                        max_pages, cache_seqlens, cu_seqlens_q, B, N, Hkv, hd};
  if (int rc = zb::check_paged(p.kv, "gqa_append")) return rc;
  ZB_REQUIRE(Hq > 0, "gqa_append: %d query heads", Hq);
  ZB_REQUIRE(rotary_dim >= 0 && rotary_dim <= hd && rotary_dim % (interleaved ? 8 : 16) == 0,
             "gqa_append: rotary_dim %d (at most %d, a multiple of %d)", rotary_dim, hd, interleaved ? 8 : 16);
  ZB_REQUIRE(rope_theta > 0 && eps >= 0.f, "gqa_append: rope_theta %g > 0, eps %g >= 0", rope_theta, (double)eps);
  ZB_REQUIRE(proj_stride >= (int64_t)(Hq + 2 * Hkv) * hd || N <= 1, "gqa_append: proj_stride %lld < %lld",
             (long long)proj_stride, (long long)(Hq + 2 * Hkv) * hd);
  ZB_REQUIRE(q_stride >= (int64_t)Hq * hd && q_stride % 8 == 0, "gqa_append: q_stride %lld", (long long)q_stride);
  if (N == 0) return zb::kOk;
  ZB_REQUIRE(B > 0, "gqa_append: %d tokens of no request", N);
  ZB_REQUIRE(proj && q_out, "gqa_append: null pointer");
  ZB_REQUIRE_ALIGNED(q_out, 16, "gqa_append q_out");
  ZB_REQUIRE_ALIGNED(proj, 2, "gqa_append proj");
  p.proj = reinterpret_cast<const __nv_bfloat16*>(proj);
  p.proj_stride = proj_stride;
  p.temp = reinterpret_cast<const __nv_bfloat16*>(temp);
  p.positions = positions;
  p.q_out = reinterpret_cast<__nv_bfloat16*>(q_out);
  p.q_stride = q_stride;
  p.eps = eps;
  p.normalize = normalize;
  p.interleaved = interleaved;
  p.rotary = rotary_dim;
  p.Hq = Hq;
  p.inv_hd = 1.f / (float)hd;
  // the pairs' frequencies in turns a position, kept per thread for the next call with the same theta and width
  thread_local double theta = 0;
  thread_local uint64_t turns[kMaxPairs];
  thread_local int width = 0;
  if (theta != rope_theta || width != rotary_dim) {
    for (int j = 0; j < rotary_dim / 2; ++j) {
      const double turn = std::pow(rope_theta, -2.0 * j / rotary_dim) / 6.283185307179586476925;
      turns[j] = (uint64_t)std::ldexp(turn - std::floor(turn), 64);
    }
    theta = rope_theta;
    width = rotary_dim;
  }
  for (int j = 0; j < rotary_dim / 2; ++j) p.turns[j] = turns[j];
  const int lanes = hd / 8, group = lanes <= 1 ? 1 : lanes <= 2 ? 2 : lanes <= 4 ? 4 : lanes <= 8 ? 8 : 16;
  const int passes = (Hq + 2 * Hkv + 32 / group - 1) / (32 / group);
  // A warp a token fills the GPU from a few thousand tokens on; fewer tokens are shared by up to a warp a pass.
  const int64_t want = ((int64_t)zb::sm_count() * 32 + N - 1) / N;
  p.shares = (int)(want < 1 ? 1 : want > passes ? passes : want);
  const uintptr_t spread = reinterpret_cast<uintptr_t>(proj) | (uintptr_t)(N > 1 ? proj_stride * 2 : 0);
  const int align = spread % 16 == 0 ? 16 : spread % 4 == 0 ? 4 : 2;
  cudaError_t err = cudaSuccess;
  switch (group) {
    case 1: err = launch_append<1>(p, align, stream); break;
    case 2: err = launch_append<2>(p, align, stream); break;
    case 4: err = launch_append<4>(p, align, stream); break;
    case 8: err = launch_append<8>(p, align, stream); break;
    default: err = launch_append<16>(p, align, stream); break;
  }
  ZB_CUDA(err);
  return zb::check_launch("gqa_append");
}
