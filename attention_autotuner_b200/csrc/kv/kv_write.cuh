// Quantising K and V of new positions into the pages of a cache (the form: kv_format.cuh), and reading positions back.
//
// What bounds both: memory. Writing reads 4 d bytes per position and head and writes 2 (d BITS / 8 + 4); reading back the other
// way round. A lane owns eight channels (16 bytes of K and of V): d / 8 lanes hold a position, so that the 16-bit side moves in
// whole rows, minimum and maximum take log2(d / 8) shuffles of a packed pair, and a lane's numbers are one or two words that lie
// in one piece of a block. A warp owns the (up to) 16 positions of one block of one head: everything it touches of the packed
// side is one piece of a page.
#pragma once

#include <limits.h>

#include "kv_format.cuh"

namespace ab200 {

// How many positions from `start` on to work on: 0 to L, and no further than the table's row reaches. Anything else is reported.
__device__ __forceinline__ int kv_count(const KvCacheView& c, int count, int start, int L, int b) {
  if (count == 0) return 0;
  const int room = static_cast<int>(static_cast<long long>(c.table_width) << c.page_shift);  // below 2^31 - 31, the host checks
  if (count > 0 && count <= L && start >= 0 && start <= room - count) return count;
  if (threadIdx.x == 0) kv_report(kKvBadLength, b);
  return start < 0 || start >= room ? 0 : min(min(max(count, 0), L), room - start);
}

struct KvWriteParams {
  KvCacheView cache;
  const void* k;
  const void* v;
  long long k_stride[3], v_stride[3];  // elements: batch, head, position; channels are dense
  const int* start;   // [B] position of the first new one
  const int* count;   // [B] how many of the L are there, or nullptr: all
  int B, L, blocks;   // blocks: of a sequence that L positions can touch
};

// Eight consecutive channels -> eight numbers of BITS bits. a: x - zero >= 0 in fp32, s: the scale in fp32.
template <int BITS>
__device__ __forceinline__ void kv_quantise8(const float* a, float s, uint32_t* out) {
  constexpr float N = static_cast<float>((1 << BITS) - 1);
  // rint(a / s) by a product: q is off a / s by less than 1e-4 (N times three half steps of fp32), so that its rounding can
  // only differ next to a half; there the quotient itself decides. (A quotient for each: 20 instructions against 4.)
  const float inv = 1.0f / s;
  float n[8];
  bool near_half = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = a[i] * inv;
    n[i] = rintf(q);
    near_half |= !(fabsf(q - n[i]) <= 0.4999f);  // true for a q that is not a number as well
  }
  if (near_half) {
#pragma unroll
    for (int i = 0; i < 8; ++i) n[i] = rintf(__fdiv_rn(a[i], s));
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) n[i] = fminf(n[i], N);
  if constexpr (BITS == 4) {
    // four numbers by sums below 2^16, exact in fp32; + 2^23 puts them into the low bits
    uint32_t half[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      half[h] = __float_as_uint(fmaf(n[4 * h + 3], 4096.f, fmaf(n[4 * h + 2], 256.f, fmaf(n[4 * h + 1], 16.f, n[4 * h]))) + 8388608.f);
    out[0] = __byte_perm(half[0], half[1], 0x5410);
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t lo = __float_as_uint(fmaf(n[4 * h + 1], 256.f, n[4 * h]) + 8388608.f);
      const uint32_t hi = __float_as_uint(fmaf(n[4 * h + 3], 256.f, n[4 * h + 2]) + 8388608.f);
      out[h] = __byte_perm(lo, hi, 0x5410);
    }
  }
}

// One row of K or V, eight channels per lane, LANES lanes per row: its numbers, and scale | zero << 16.
template <int BITS, bool BF16, int LANES>
__device__ __forceinline__ uint32_t kv_quantise_row(const uint4& x, uint32_t* out) {
  using T = Kv16<BF16>;
  const uint32_t u[4] = {x.x, x.y, x.z, x.w};
  constexpr uint32_t SIGNS = 0x80008000u;
  uint32_t lo = T::min2_nan(T::min2_nan(u[0], u[1]), T::min2_nan(u[2], u[3]));
  uint32_t hi = T::min2_nan(T::min2_nan(u[0] ^ SIGNS, u[1] ^ SIGNS), T::min2_nan(u[2] ^ SIGNS, u[3] ^ SIGNS));  // of -x
  uint32_t both = T::min2_nan(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));  // min x | min -x << 16
#pragma unroll
  for (int m = 1; m < LANES; m <<= 1) both = T::min2_nan(both, __shfl_xor_sync(0xffffffffu, both, m));
  const float zero = T::lo(both), range = -T::hi(both) - zero;
  const float N = static_cast<float>((1 << BITS) - 1);
  const uint32_t s16 = T::round(__fdiv_rn(range, N));
  const float s = T::lo(s16);
  if (!(fabsf(range) < INFINITY) || s == 0.f) {  // a row without a finite range, or without one that the type can hold
    out[0] = 0;
    if constexpr (BITS == 8) out[1] = 0;
    return s == 0.f ? (both << 16) : 0x7fff7fffu;  // scale 0; or both NaN
  }
  float a[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    a[2 * i] = T::lo(u[i]) - zero;
    a[2 * i + 1] = T::hi(u[i]) - zero;
  }
  kv_quantise8<BITS>(a, s, out);
  return s16 | (both << 16);
}

template <int BITS>
__device__ __forceinline__ void kv_store_words(uint8_t* to, const uint32_t* w) {
  if constexpr (BITS == 4) *reinterpret_cast<uint32_t*>(to) = w[0];
  else *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
}

// grid (ceil(blocks / warps per CTA), heads, B)
template <int BITS, int D, bool BF16>
__global__ void __launch_bounds__(128) kv_write_kernel(const __grid_constant__ KvWriteParams p) {
  using Blk = KvBlock<BITS, D>;
  constexpr int LANES = D / 8, PER = 32 / LANES;  // lanes per position, positions per instruction
  constexpr int BATCH = 4;                        // positions in flight per lane
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, h = blockIdx.y;
  const int start = p.start[b];
  int count = p.count != nullptr ? p.count[b] : p.L;
  count = kv_count(p.cache, count, start, p.L, b);
  const int off = (blockIdx.x * 4 + warp) * kKvBlockTokens - start % kKvBlockTokens;  // of this warp's block, from start on
  if (count <= max(off, 0)) return;
  const int pos0 = start + off, first = max(-off, 0), last = min(count - off, kKvBlockTokens);
  const int page = kv_page(p.cache, b, pos0);
  if (page < 0) return;
  uint8_t* blk = kv_block(p.cache, page, h, pos0, Blk::BYTES);
  const int sub = lane / LANES, ch = (lane % LANES) * 8;
  const uint16_t* k = static_cast<const uint16_t*>(p.k) + b * p.k_stride[0] + h * p.k_stride[1] + off * p.k_stride[2] + ch;
  const uint16_t* v = static_cast<const uint16_t*>(p.v) + b * p.v_stride[0] + h * p.v_stride[1] + off * p.v_stride[2] + ch;
#pragma unroll 1
  for (int base = first / PER * PER; base < last; base += BATCH * PER) {
    uint4 kx[BATCH], vx[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int tok = base + i * PER + sub;
      const bool mine = tok >= first && tok < last;
      kx[i] = mine ? __ldcs(reinterpret_cast<const uint4*>(k + tok * p.k_stride[2])) : make_uint4(0, 0, 0, 0);
      vx[i] = mine ? __ldcs(reinterpret_cast<const uint4*>(v + tok * p.v_stride[2])) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (base + i * PER >= last) break;  // the same for all lanes
      const int tok = base + i * PER + sub;
      uint32_t kw[2], vw[2];
      const uint32_t km = kv_quantise_row<BITS, BF16, LANES>(kx[i], kw);
      const uint32_t vm = kv_quantise_row<BITS, BF16, LANES>(vx[i], vw);
      if (tok >= first && tok < last) {
        kv_store_words<BITS>(blk + Blk::k_byte(tok, ch * BITS / 8), kw);
        kv_store_words<BITS>(blk + Blk::v_byte(tok, ch * BITS / 8), vw);
        if (ch == 0) *reinterpret_cast<uint2*>(blk + Blk::meta_byte(tok)) = make_uint2(km, vm);
      }
    }
  }
}

struct KvReadParams {
  KvCacheView cache;
  void* k;  // [B, heads, L, D], dense
  void* v;
  const int* start;
  const int* count;  // or nullptr: L
  int B, L;
};

// Eight numbers -> eight values of the cache's type.
template <int BITS, bool BF16>
__device__ __forceinline__ uint4 kv_values8(const uint8_t* from, uint32_t meta) {
  using T = Kv16<BF16>;
  const float s = T::lo(meta), z = T::hi(meta);
  uint32_t w[2];
  if constexpr (BITS == 4) w[0] = __ldg(reinterpret_cast<const uint32_t*>(from));
  else {
    const uint2 x = __ldg(reinterpret_cast<const uint2*>(from));
    w[0] = x.x;
    w[1] = x.y;
  }
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t n = BITS == 4 ? (w[0] >> (4 * i)) & 15u : (w[i >> 2] >> (8 * (i & 3))) & 255u;
    f[i] = fmaf(__uint_as_float(0x4b000000u | n) - 8388608.f, s, z);  // the product is exact: 8 by 11 bits
  }
  return make_uint4(T::round2(f[0], f[1]), T::round2(f[2], f[3]), T::round2(f[4], f[5]), T::round2(f[6], f[7]));
}

// grid (ceil(L / (16 * warps per CTA)), heads, B): a warp owns 16 rows of the output
template <int BITS, int D, bool BF16>
__global__ void __launch_bounds__(128) kv_read_kernel(const __grid_constant__ KvReadParams p) {
  using Blk = KvBlock<BITS, D>;
  constexpr int LANES = D / 8, PER = 32 / LANES;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, h = blockIdx.y;
  const int row0 = (blockIdx.x * 4 + warp) * kKvBlockTokens;
  if (row0 >= p.L) return;
  const int start = p.start != nullptr ? p.start[b] : 0;
  int count = p.count != nullptr ? p.count[b] : p.L;
  count = kv_count(p.cache, count, start, p.L, b);
  const int sub = lane / LANES, ch = (lane % LANES) * 8;
  const long long out0 = ((static_cast<long long>(b) * p.cache.heads + h) * p.L) * D + ch;
#pragma unroll 4
  for (int i = 0; i < kKvBlockTokens; i += PER) {
    const int row = row0 + i + sub;
    if (row >= p.L) break;
    uint4 kx = make_uint4(0, 0, 0, 0), vx = kx;
    if (row < count) {
      const int pos = start + row, tok = pos & (kKvBlockTokens - 1);
      const int page = kv_page(p.cache, b, pos);
      if (page >= 0) {
        const uint8_t* blk = kv_block(p.cache, page, h, pos, Blk::BYTES);
        const uint2 m = __ldg(reinterpret_cast<const uint2*>(blk + Blk::meta_byte(tok)));
        kx = kv_values8<BITS, BF16>(blk + Blk::k_byte(tok, ch * BITS / 8), m.x);
        vx = kv_values8<BITS, BF16>(blk + Blk::v_byte(tok, ch * BITS / 8), m.y);
      }
    }
    const long long o = out0 + static_cast<long long>(row) * D;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.k) + o) = kx;
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.v) + o) = vx;
  }
}

}  // namespace ab200
