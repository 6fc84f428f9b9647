// A paged KV cache in 4 bits: its layout, and the arithmetic of its groups.
//
// 32 consecutive elements of a token's key or value of one KV head are a group; it is kept as 4-bit codes c and a pair (s, m)
// of bf16, and stands for x = m + s c. From x (bf16; NaN counts as 0, and what is beyond +-2^63 as that):
//   m = min x,  s = bf16((max x - min x) / 15) (0 where that is below 2^-100),  c = floor((x - m) / s + 1/2), 0 .. 15 (0 where s = 0)
// with the difference and the quotient in s rounded to fp32 before, and c exact.
// m is one of the elements, so storing it rounds nothing; s is rounded before it divides, so c allows for it. A pair with a
// magnitude of 2^64 or more, or a NaN, is never written and stands for zeros: rows that no token wrote hold anything, and 0 x
// inf would be NaN in a matrix product that counts them with weight 0; and sums of 2^26 values, times weights of up to 2^15, stay
// in fp32's range.
//
// 16 consecutive keys of a head are a block of 20 hd bytes, a page of a head is page_size / 16 blocks one after the other:
//   [0, 8 hd) codes of the keys, 16 rows of hd / 2 bytes; [8 hd, 16 hd) codes of the values;
//   [16 hd, 18 hd) pairs of the keys, 16 rows of hd / 32 (s in the lower half of a 32-bit word); [18 hd, 20 hd) of the values.
// So one bulk copy of 20 hd bytes (2560 at hd 128) brings the keys and values of 16 tokens of a head. A row's codes are
// 32-bit words: word t * (hd / 32) + g holds elements e = 0 .. 7 of dims 32 g + 8 t + e, element e in bits 4 (e / 2 + 4 (e % 2))
// and up. (w >> 4 i) & 0x000f000f is then the pair of elements 2 i, 2 i + 1, as matrix fragments hold them; a word lies in one
// group; and the words of a t are consecutive, which are what one lane of a fragment of 16 keys needs of a row.
#pragma once

#include <cuda_fp16.h>

#include "paged.cuh"

namespace zb {
namespace q4 {

constexpr int kBlock = 16;   // keys of a block
constexpr int kGroup = 32;   // elements of a group
constexpr float kLargest = 0x1p63f, kSmallestStep = 0x1p-100f;

__host__ __device__ constexpr int block_bytes(int hd) { return 20 * hd; }

// The cache as a PagedBatch: `k` is its first byte, strides are in bytes, `v` and slot_stride are not used.
inline int check_cache(const PagedBatch& p, const char* who) {
  ZB_REQUIRE(p.B >= 0 && p.N >= 0 && p.Hkv > 0 && p.num_pages >= 0 && p.max_pages >= 0, "%s: negative sizes", who);
  if (p.hd < kGroup || p.hd > 128 || p.hd % kGroup != 0)
    return fail(kUnsupported, "%s: head dim %d (32, 64, 96 or 128)", who, p.hd);
  ZB_REQUIRE(p.page_size >= kBlock && p.page_size % kBlock == 0 && (int64_t)p.page_size * p.max_pages <= (int64_t)1 << 26,
             "%s: page size %d (a multiple of 16) x %d table columns (at most 2^26 keys)", who, p.page_size, p.max_pages);
  ZB_REQUIRE(p.page_stride % 16 == 0 && p.head_stride % 16 == 0 && p.page_stride >= 0 && p.head_stride >= 0,
             "%s: cache strides (page %lld, head %lld bytes) must be multiples of 16", who, (long long)p.page_stride,
             (long long)p.head_stride);
  ZB_REQUIRE(p.table_stride >= p.max_pages || p.B <= 1, "%s: table stride %lld < %d columns", who,
             (long long)p.table_stride, p.max_pages);
  if (p.B == 0 || p.N == 0) return kOk;
  ZB_REQUIRE(p.cu && p.keys && (p.table || p.max_pages == 0) && (p.k || p.num_pages == 0), "%s: null pointer", who);
  ZB_REQUIRE(reinterpret_cast<uintptr_t>(p.k) % 16 == 0, "%s: the cache must be 16-byte aligned", who);
  return kOk;
}

// Whether a pair stands for zeros by the rule above: a number that is not finite or has a magnitude of 2^64 or more has an exponent
// field of 191 or more, and with 0x8000 - 0x5f80 added carries into its sign (which `none_bits` leaves, among other bits).
__device__ __forceinline__ uint32_t none_bits(uint32_t pair) { return (pair & 0x7fff7fffu) + 0x20802080u; }
__device__ __forceinline__ bool pair_is_none(uint32_t pair) { return (none_bits(pair) & 0x80008000u) != 0; }

__device__ __forceinline__ __nv_bfloat162 as_bf162(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
__device__ __forceinline__ uint32_t as_word(__nv_bfloat162 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// (x & mask) | bits, in one instruction: of two constants the compiler makes two.
__device__ __forceinline__ uint32_t masked_or(uint32_t x, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(x), "r"(mask), "r"(bits));
  return d;
}
// 128 + c of codes 2 i, 2 i + 1 of a word, as bf16: 128 has its last bit at 1, so a code is the lower bits of the significand.
template <int I>
__device__ __forceinline__ uint32_t codes_128(uint32_t word) {
  return masked_or(word >> (4 * I), 0x000f000fu, 0x43004300u);
}
// m + s c of two codes, rounded once: s2, m2 hold s and m twice (or those of two tokens).
__device__ __forceinline__ uint32_t stands_for(uint32_t c128, uint32_t s2, uint32_t m2) {
  return as_word(__hfma2(__hsub2(as_bf162(c128), as_bf162(0x43004300u)), as_bf162(s2), as_bf162(m2)));
}
// The 8 elements of a word of codes, as bf16.
__device__ __forceinline__ uint4 read_word(uint32_t word, uint32_t pair) {
  const uint32_t s2 = __byte_perm(pair, 0, 0x1010), m2 = __byte_perm(pair, 0, 0x3232);
  return make_uint4(stands_for(codes_128<0>(word), s2, m2), stands_for(codes_128<1>(word), s2, m2),
                    stands_for(codes_128<2>(word), s2, m2), stands_for(codes_128<3>(word), s2, m2));
}

// Whether fp16 holds what a pair stands for as well as bf16 and better: |m| is below 2^14 and s below 2^10 (a sign bit of `over`
// else), and s is 2^-14 or more, so that fp16's smallest step is little beside it, or the pair is 0 (`holds`).
__device__ __forceinline__ void fp16_holds(uint32_t pair, uint32_t& over, bool& holds) {
  const uint32_t a = pair & 0x7fff7fffu;
  over |= a + (((0x8000u - 0x4680u) << 16) | (0x8000u - 0x4480u));
  holds &= pair << 16 >= 0x3880u << 16 || a == 0;
}
// A pair in fp16, s and m twice; and the 8 elements of a word of codes, m + s c rounded once.
struct HalfPair {
  uint32_t s2, m2;
  __device__ __forceinline__ explicit HalfPair(uint32_t pair) {
    const float s = __uint_as_float(pair << 16), m = __uint_as_float(pair & 0xffff0000u);
    asm("cvt.rn.f16x2.f32 %0, %1, %1;" : "=r"(s2) : "f"(s));
    asm("cvt.rn.f16x2.f32 %0, %1, %1;" : "=r"(m2) : "f"(m));
  }
  template <int I>
  __device__ __forceinline__ uint32_t two(uint32_t word) const {
    // 1024 + c, or 64 + c from 4 bits higher in the significand
    const uint32_t zero = I % 2 ? 0x54005400u : 0x64006400u;
    const uint32_t c = masked_or(I >= 2 ? word >> 8 : word, I % 2 ? 0x00f000f0u : 0x000f000fu, zero);
    const __half2 v = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&c), *reinterpret_cast<const __half2*>(&zero)),
                              *reinterpret_cast<const __half2*>(&s2), *reinterpret_cast<const __half2*>(&m2));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  __device__ __forceinline__ uint4 read_word(uint32_t word) const {
    return make_uint4(two<0>(word), two<1>(word), two<2>(word), two<3>(word));
  }
};

// 8 bf16 elements of a group whose other elements are on the lanes' neighbours (4 lanes of a group, lane % 4 = t): their
// word of codes and the group's pair. Every lane of the warp takes part.
__device__ __forceinline__ uint32_t write_word(uint4 x, uint32_t& pair) {
  uint32_t w[4] = {x.x, x.y, x.z, x.w};
  // the smallest element and the negated largest, as a pair of bf16; a NaN anywhere comes out as NaN
  auto bounds = [&]() {
    const __nv_bfloat162 lo = __hmin2_nan(__hmin2_nan(as_bf162(w[0]), as_bf162(w[1])), __hmin2_nan(as_bf162(w[2]), as_bf162(w[3])));
    const __nv_bfloat162 hi = __hmax2_nan(__hmax2_nan(as_bf162(w[0]), as_bf162(w[1])), __hmax2_nan(as_bf162(w[2]), as_bf162(w[3])));
    const uint32_t l = as_word(lo), h = as_word(hi) ^ 0x80008000u;
    __nv_bfloat162 b = __hmin2_nan(as_bf162(__byte_perm(l, h, 0x5410)), as_bf162(__byte_perm(l, h, 0x7632)));
#pragma unroll
    for (int o = 1; o < 4; o *= 2) b = __hmin2_nan(b, as_bf162(__shfl_xor_sync(0xffffffffu, as_word(b), o)));
    return as_word(b);
  };
  uint32_t b = bounds();
  float low = __uint_as_float(b << 16), high = -__uint_as_float(b & 0xffff0000u);
  if (__any_sync(0xffffffffu, !(low >= -kLargest && high <= kLargest))) {  // elements that 4 bits do not keep
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t fixed = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float v = __uint_as_float(e ? w[i] & 0xffff0000u : w[i] << 16);
        const float kept = v != v ? 0.f : fminf(fmaxf(v, -kLargest), kLargest);  // exact in bf16
        fixed |= e ? __float_as_uint(kept) : __float_as_uint(kept) >> 16;
      }
      w[i] = fixed;
    }
    b = bounds();
    low = __uint_as_float(b << 16);
    high = -__uint_as_float(b & 0xffff0000u);
  }
  float s = bf16_round(__fdiv_rn(high - low, 15.f));
  if (s < kSmallestStep) s = 0.f;
  pair = (__float_as_uint(s) >> 16) | (__float_as_uint(low) & 0xffff0000u);
  // floor(d / s + 1/2) is d r rounded to an integer, or one more: r is below 1 / s by more than its and the product's roundings,
  // and what is left of d after that many steps, which fp32 holds exactly, tells which.
  // d is rounded down where fp32 does not hold it: a border, (c + 1/2) s, has few bits, so what is below it stays below.
  // It is not above 15, as s is within 2^-8 of a fifteenth of the largest d. With s = 0 all codes are 0.
  const float r = s > 0.f ? __frcp_rn(s) * (1.f - 0x1p-20f) : 0.f, half = s > 0.f ? 0.5f * s : INFINITY;
  constexpr float kMagic = 12582912.f;  // 1.5 x 2^23: a sum with it has the nearest integer in its lower bits
  constexpr uint32_t kMagicBits = 0x4b400000u;
  uint32_t word = 0u - kMagicBits * 0x11111111u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float d = __fsub_rd(__uint_as_float(e ? w[i] & 0xffff0000u : w[i] << 16), low);
      float c = fmaf(d, r, kMagic);
      if (fmaf(kMagic - c, s, d) >= half) c += 1.f;
      word += __float_as_uint(c) << (4 * (i + 4 * e));
    }
  }
  return word;
}

}  // namespace q4
}  // namespace zb
