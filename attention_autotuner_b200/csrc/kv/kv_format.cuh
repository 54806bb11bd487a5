// The packed form of a quantised KV cache: what kv_write.cuh writes and reads back and kv_attn.cuh attends over.
//
// A position of a head holds d values of K and d of V. Each of the two is kept as d whole numbers n of BITS (4 or 8) bits and two
// 16-bit numbers, scale and zero, of the cache's type: value = zero + scale n, with
//     zero = min x,  scale = round16((max x - min x) / N),  n = min(rint((x - zero) / scale), N),  N = 2^BITS - 1
// (differences and quotients in fp32, correctly rounded; half to even). scale = 0: n = 0. A range that is not finite in fp32
// (an infinity, a NaN): scale = zero = NaN, n = 0.
//
// Memory: [page][head][page_size / 16 blocks]; a block is 16 positions of one head in one piece, so that one bulk copy brings it:
//     16 d BITS / 8 bytes of K | as many of V | 16 x 8 bytes {K scale, K zero, V scale, V zero}
// Inside, the numbers lie as the lanes of a warp hold them in mma.sync m16n8k16 A fragments (lane = 4 g + t, g < 8, t < 4):
//   K (S^T = K Q^T, rows = positions): lane owns positions g and g + 8, the t-th quarter of the channels. Which channels form a
//     k-step is free (it is the contraction index), so that a lane's share is a run of channels;
//   V (O^T = V^T P^T, rows = channels): lane owns positions 2t, 2t + 1, 2t + 8, 2t + 9, the g-th eighth of the channels;
//   16-byte units of a lane are 512 bytes apart, so that a warp reads a unit of all lanes without bank conflicts and in one
//     coalesced piece; the 8-byte quads of positions g and g + 8 are neighbours.
// No byte holds numbers of two positions: a position is written without reading what is there.
// V of odd positions is stored as N - n: the sums of the products of values about the middle of their ranges then stay near zero, where
// the accumulators of the tensor cores, which drop the bits that do not fit, lose the least (kv_attn.cuh).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "../ptx.cuh"

namespace ab200 {

constexpr int kKvBlockTokens = 16;

template <int BITS_, int D_>
struct KvBlock {
  static constexpr int BITS = BITS_, D = D_;
  static_assert(BITS == 4 || BITS == 8, "bits");
  static_assert(D == 64 || D == 128 || D == 256, "head dimension");
  static constexpr int ROW = D * BITS / 8;  // bytes of the numbers of one position, K or V
  static constexpr int CODE = kKvBlockTokens * ROW;
  static constexpr int META = 2 * CODE;  // offset of the scales and zeros
  static constexpr int BYTES = META + kKvBlockTokens * 8;
  static_assert(BYTES % 16 == 0, "bulk copies");
  static constexpr int KCHUNK = ROW / 4, VCHUNK = ROW / 8;

  // offset of byte x of a lane's share
  __host__ __device__ static constexpr int lane_byte(int lane, int x) { return ((x >> 4) * 32 + lane) * 16 + (x & 15); }
  // offsets inside a block of the byte with channels byte * 8 / BITS ... of position tok (0..15)
  __host__ __device__ static constexpr int k_byte(int tok, int byte) {
    return lane_byte((tok & 7) * 4 + byte / KCHUNK, (tok >> 3) * KCHUNK + byte % KCHUNK);
  }
  __host__ __device__ static constexpr int v_byte(int tok, int byte) {
    return CODE + lane_byte((byte / VCHUNK) * 4 + ((tok & 7) >> 1), ((tok & 1) | ((tok >> 3) << 1)) * VCHUNK + byte % VCHUNK);
  }
  __host__ __device__ static constexpr int meta_byte(int tok) { return META + ((tok & 7) * 2 + (tok >> 3)) * 8; }
};

inline int kv_block_bytes(int bits, int d) { return 2 * kKvBlockTokens * d * bits / 8 + kKvBlockTokens * 8; }

// What every kernel knows of a cache and of the sequences in it.
struct KvCacheView {
  uint8_t* data;
  const int* table;          // [B][table_stride]: page of positions [i page_size, (i + 1) page_size)
  long long head_bytes;      // one head of one page
  int table_stride, table_width;
  int num_pages, heads, page_shift;  // page_size = 1 << page_shift
  int first;                         // the call's number of the first sequence that this launch works on
};

// What a kernel found in the tables that it was given (the host cannot see them). The kernels leave such positions out: not
// written, read back as zeros, not attended to. Sticky like the status words of ptx.cuh, with the fourth word of the same mirror.
enum KvBad : int { kKvBadPage = 1, kKvBadLength = 2 };
__device__ int g_kv_bad = 0;
__device__ __noinline__ void kv_report(int what, int sequence) {
  if (atomicCAS(&g_kv_bad, 0, what) == 0) {
    volatile int* mirror = g_status_mirror;
    if (mirror != nullptr) mirror[3] = what | (sequence << 8);
  }
}

// Page of a position, or -1 (reported) if the table has none that exists. pos >= 0.
__device__ __forceinline__ int kv_page(const KvCacheView& c, int b, int pos) {
  const int i = pos >> c.page_shift;
  if (i >= c.table_width) {
    kv_report(kKvBadLength, c.first + b);
    return -1;
  }
  const int page = c.table[static_cast<long long>(b) * c.table_stride + i];
  if (page < 0 || page >= c.num_pages) {
    kv_report(kKvBadPage, c.first + b);
    return -1;
  }
  return page;
}
// The block that holds position pos of a head on that page.
__device__ __forceinline__ uint8_t* kv_block(const KvCacheView& c, int page, int head, int pos, int block_bytes) {
  const int in_page = (pos & ((1 << c.page_shift) - 1)) / kKvBlockTokens;
  return c.data + (static_cast<long long>(page) * c.heads + head) * c.head_bytes + static_cast<long long>(in_page) * block_bytes;
}

// The two 16-bit types by one name.
template <bool BF16>
struct Kv16;
template <>
struct Kv16<false> {
  __device__ static __forceinline__ float lo(uint32_t u) { return __half2float(__ushort_as_half(u & 0xffffu)); }
  __device__ static __forceinline__ float hi(uint32_t u) { return __half2float(__ushort_as_half(u >> 16)); }
  __device__ static __forceinline__ uint32_t round(float x) { return __half_as_ushort(__float2half_rn(x)); }
  __device__ static __forceinline__ uint32_t round2(float lo, float hi) {  // beyond the range: infinity, as a conversion in PyTorch
    const __half2 r = __floats2half2_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(r);
  }
  __device__ static __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(reinterpret_cast<__half2&>(a), reinterpret_cast<__half2&>(b), reinterpret_cast<__half2&>(c));
    return reinterpret_cast<const uint32_t&>(r);
  }
  __device__ static __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(reinterpret_cast<__half2&>(a), reinterpret_cast<__half2&>(b));
    return reinterpret_cast<const uint32_t&>(r);
  }
  __device__ static __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
    const __half2 r = __hmin2_nan(reinterpret_cast<__half2&>(a), reinterpret_cast<__half2&>(b));
    return reinterpret_cast<const uint32_t&>(r);
  }
  __device__ static __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2_nan(reinterpret_cast<__half2&>(a), reinterpret_cast<__half2&>(b));
    return reinterpret_cast<const uint32_t&>(r);
  }
};
template <>
struct Kv16<true> {
  __device__ static __forceinline__ float lo(uint32_t u) { return __uint_as_float(u << 16); }
  __device__ static __forceinline__ float hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
  __device__ static __forceinline__ uint32_t round(float x) { return __bfloat16_as_ushort(__float2bfloat16_rn(x)); }
  __device__ static __forceinline__ uint32_t round2(float lo, float hi) {
    const __nv_bfloat162 r = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(r);
  }
  __device__ static __forceinline__ uint32_t fma2(uint32_t a, uint32_t b, uint32_t c) {
    const __nv_bfloat162 r = __hfma2(reinterpret_cast<__nv_bfloat162&>(a), reinterpret_cast<__nv_bfloat162&>(b), reinterpret_cast<__nv_bfloat162&>(c));
    return reinterpret_cast<const uint32_t&>(r);
  }
  __device__ static __forceinline__ uint32_t sub2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(reinterpret_cast<__nv_bfloat162&>(a), reinterpret_cast<__nv_bfloat162&>(b));
    return reinterpret_cast<const uint32_t&>(r);
  }
  __device__ static __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmin2_nan(reinterpret_cast<__nv_bfloat162&>(a), reinterpret_cast<__nv_bfloat162&>(b));
    return reinterpret_cast<const uint32_t&>(r);
  }
  __device__ static __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2_nan(reinterpret_cast<__nv_bfloat162&>(a), reinterpret_cast<__nv_bfloat162&>(b));
    return reinterpret_cast<const uint32_t&>(r);
  }
};

}  // namespace ab200
