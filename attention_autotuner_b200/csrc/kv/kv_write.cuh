// Quantising K and V of new positions into the pages of a cache (the form: kv_format.cuh), and reading positions back.
//
// What bounds both: memory. Writing reads 4 d bytes per position and head and writes 2 (d BITS / 8 + 4); reading back the other
// way round. A lane owns eight channels of either half of a row (16 bytes twice, each load of a warp in whole rows); d / 16 lanes
// hold a position, so that what is done once per row (minimum and maximum by shuffles of a packed pair, two quotients) is
// shared by 16 channels. A warp owns the 16 positions of one block of one head. It puts them together in shared memory and stores
// them with one bulk copy if they are all new; a block that is written in part is stored position by position.
//
// Next to the memory it is the issue slots that count: at the copy bandwidth an SM has 14 instructions of a lane for each number
// written, 17 for each read. Hence packed fp32 arithmetic for the numbers (kv_quantise) and the packed fma of the type for the values
// (kv_values8).
//
// Measured (B200, us of the device; at the copy bandwidth): 16 heads x 16384 positions, d = 128, 8 bits, bf16 written 38 (31; the ALUs are 62% busy, a
// bf16 row needs its largest numbers put right), read 32 (31); 4 x 16 heads of up to 2999, 4 bits, bf16 read 19.1 (16.3); 64 x 8 heads,
// one position each, written and read 5.0. With a quotient for every number next to a half, where bf16 has one in 200: 78 written.
#pragma once

#include <limits.h>

#include "kv_format.cuh"

namespace ab200 {

// How many positions from `start` on to work on: 0 to L, and no further than the table's row reaches. Anything else is reported.
__device__ __forceinline__ int kv_count(const KvCacheView& c, int count, int start, int L, int b) {
  if (count == 0) return 0;
  const int room = static_cast<int>(static_cast<long long>(c.table_width) << c.page_shift);  // below 2^31 - 31, the host checks
  if (count > 0 && count <= L && start >= 0 && start <= room - count) return count;
  if (threadIdx.x == 0) kv_report(kKvBadLength, c.first + b);
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

// Numbers of 16 channels of a row, u: as 16-bit pairs; zero, s, range: of the row, in fp32, range and s finite, s > 0.
// What is rounded to a whole number is the fp32 quotient (x - zero) / s itself, halves included (of bf16 numbers one in 200 is one):
// q = a inv, then one Newton step q + (a - q s) inv, which gives the quotient rounded to nearest if inv is the reciprocal rounded to
// nearest and s is not all ones (P. Markstein, IBM J. Res. Dev. 34, 1990); s has 11 bits at most. Two numbers per instruction.
template <int BITS, bool BF16>
__device__ __forceinline__ void kv_quantise(const uint32_t* u, float zero, float s, float range, uint32_t (*out)[2]) {
  using T = Kv16<BF16>;
  constexpr float N = static_cast<float>((1 << BITS) - 1);
  constexpr float ROUND = 12582912.f;  // 1.5 * 2^23: a sum with it is rounded to whole numbers, half to even, in its low bits
  uint32_t n[16];
  if (s >= 7.9e-31f && range <= 1.3e30f) {  // 2^-100, 2^100: nothing below leaves the range of fp32
    const float inv = __frcp_rn(s);
    const uint64_t inv2 = f2_pack(inv, inv), minus_s2 = f2_pack(-s, -s), minus_zero2 = f2_pack(-zero, -zero), round2 = f2_pack(ROUND, ROUND);
    uint64_t q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t a = fadd2(f2_pack(T::lo(u[i]), T::hi(u[i])), minus_zero2);
      const uint64_t q0 = fmul2(a, inv2);
      q[i] = ffma2(ffma2(q0, minus_s2, a), inv2, q0);
    }
    // a scale that was rounded down, by up to half a step of its type, can make the largest number N + 1: of 8 bits and bf16 it
    // often does and is put right below, else only a subnormal scale is that coarse
    if ((BITS == 4 || !BF16) && range * inv > N + 0.25f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float x, y;
        f2_unpack(q[i], x, y);
        q[i] = f2_pack(fminf(x, N), fminf(y, N));
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float x, y;
      f2_unpack(fadd2(q[i], round2), x, y);
      n[2 * i] = __float_as_uint(x);
      n[2 * i + 1] = __float_as_uint(y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      n[i] = __float_as_uint(fminf(__fdiv_rn((i & 1 ? T::hi(u[i >> 1]) : T::lo(u[i >> 1])) - zero, s), N) + ROUND);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t* m = n + 8 * h;
    if constexpr (BITS == 4) {
      uint32_t w = m[7];
#pragma unroll
      for (int i = 6; i >= 0; --i) w = (w << 4) + m[i];
      out[h][0] = w - 0x3f400000u;  // the bits of ROUND, 0x4b400000, shifted by 0, 4, ... and added
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        out[h][i] = BF16 ? __byte_perm(__vminu2(__byte_perm(m[4 * i], m[4 * i + 1], 0x5410), 0x00ff00ffu),
                                       __vminu2(__byte_perm(m[4 * i + 2], m[4 * i + 3], 0x5410), 0x00ff00ffu), 0x6420)
                         : __byte_perm(__byte_perm(m[4 * i], m[4 * i + 1], 0x0040), __byte_perm(m[4 * i + 2], m[4 * i + 3], 0x0040), 0x5410);
    }
  }
}

// One row of K or V, eight channels of either half per lane, LANES lanes per row: its numbers, and scale | zero << 16.
template <int BITS, bool BF16, int LANES>
__device__ __forceinline__ uint32_t kv_quantise_row(const uint4* x, uint32_t (*out)[2]) {
  using T = Kv16<BF16>;
  const uint32_t u[8] = {x[0].x, x[0].y, x[0].z, x[0].w, x[1].x, x[1].y, x[1].z, x[1].w};
  constexpr uint32_t SIGNS = 0x80008000u;
  uint32_t lo = u[0], hi = u[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = T::min2_nan(lo, u[i]);
    hi = T::max2_nan(hi, u[i]);
  }
  hi ^= SIGNS;
  uint32_t both = T::min2_nan(__byte_perm(lo, hi, 0x5410), __byte_perm(lo, hi, 0x7632));  // min x | min -x << 16
#pragma unroll
  for (int m = 1; m < LANES; m <<= 1) both = T::min2_nan(both, __shfl_xor_sync(0xffffffffu, both, m));
  const float zero = T::lo(both), range = -T::hi(both) - zero;
  const uint32_t s16 = T::round(__fdiv_rn(range, static_cast<float>((1 << BITS) - 1)));
  const float s = T::lo(s16);
  if (!(fabsf(range) < INFINITY) || s == 0.f) {  // a row without a finite range, or without one that the type can hold
#pragma unroll
    for (int h = 0; h < 2; ++h) out[h][0] = out[h][1] = 0;
    return s == 0.f ? (both << 16) : 0x7fff7fffu;  // scale 0; or both NaN
  }
  kv_quantise<BITS, BF16>(u, zero, s, range, out);
  return s16 | (both << 16);
}

// Untiled bulk copy shared -> global memory; both addresses 16-byte aligned, bytes a multiple of 16.
__device__ __forceinline__ void kv_bulk_store(void* gmem, const void* smem_src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(gmem), "r"(smem_u32(smem_src)), "r"(bytes) : "memory");
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
  constexpr int LANES = D / 16, PER = 32 / LANES;  // lanes per position, positions per instruction
  __shared__ __align__(128) uint8_t stage[4][Blk::BYTES];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, h = blockIdx.y;
  pdl_grid_dependency_wait();  // launched as a programmatic dependent: what is in front has completed from here on
  const int start = p.start[b];
  const int count = kv_count(p.cache, p.count != nullptr ? p.count[b] : p.L, start, p.L, b);
  const int off = (blockIdx.x * 4 + warp) * kKvBlockTokens - start % kKvBlockTokens;  // of this warp's block, from start on
  if (count <= max(off, 0)) return;
  const int pos0 = start + off, first = max(-off, 0), last = min(count - off, kKvBlockTokens);
  const int sub = lane / LANES, ch = (lane % LANES) * 8;
  const uint16_t* k = static_cast<const uint16_t*>(p.k) + b * p.k_stride[0] + h * p.k_stride[1] + off * p.k_stride[2] + ch;
  const uint16_t* v = static_cast<const uint16_t*>(p.v) + b * p.v_stride[0] + h * p.v_stride[1] + off * p.v_stride[2] + ch;
  auto load = [&](int tok, uint4* kx, uint4* vx) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kx[i] = vx[i] = make_uint4(0, 0, 0, 0);
      if (tok >= first && tok < last) {
        kx[i] = __ldcs(reinterpret_cast<const uint4*>(k + tok * p.k_stride[2] + i * (D / 2)));
        vx[i] = __ldcs(reinterpret_cast<const uint4*>(v + tok * p.v_stride[2] + i * (D / 2)));
      }
    }
  };
  const bool whole = first == 0 && last == kKvBlockTokens;
  const int base0 = first / PER * PER;
  uint4 kx[2], vx[2], kn[2], vn[2];
  load(base0 + sub, kx, vx);
  const int page = kv_page(p.cache, b, pos0);  // beside the first loads
  if (page < 0) return;
  uint8_t* blk = kv_block(p.cache, page, h, pos0, Blk::BYTES);
  uint8_t* to = whole ? stage[warp] : blk;
#pragma unroll 1
  for (int base = base0; base < last; base += PER) {
    const int tok = base + sub;
    load(tok + PER, kn, vn);
    uint32_t kw[2][2], vw[2][2];
    const uint32_t km = kv_quantise_row<BITS, BF16, LANES>(kx, kw);
    const uint32_t vm = kv_quantise_row<BITS, BF16, LANES>(vx, vw);
    const uint32_t flip = tok & 1 ? ~0u : 0u;  // V of odd positions: 2^BITS - 1 - n
    if (tok >= first && tok < last) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        vw[i][0] ^= flip;
        vw[i][1] ^= flip;
        kv_store_words<BITS>(to + Blk::k_byte(tok, (ch + i * (D / 2)) * BITS / 8), kw[i]);
        kv_store_words<BITS>(to + Blk::v_byte(tok, (ch + i * (D / 2)) * BITS / 8), vw[i]);
      }
      if (ch == 0) *reinterpret_cast<uint2*>(to + Blk::meta_byte(tok)) = make_uint2(km, vm);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      kx[i] = kn[i];
      vx[i] = vn[i];
    }
  }
  if (whole) {
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {
      kv_bulk_store(blk, stage[warp], Blk::BYTES);
      tma_store_commit();
      tma_store_wait0();  // it depends on no other thread, and the buffer must outlive it
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

// Eight numbers -> eight values of the cache's type, each rounded once. meta: scale | zero << 16.
template <int BITS, bool BF16>
__device__ __forceinline__ uint4 kv_values8(const uint32_t* w, uint32_t meta) {
  using T = Kv16<BF16>;
  // n in the mantissa of 1024 (bf16: 128; with 8 bits 2^23 in fp32, since a bf16 has seven bits behind the leading one), an exact
  // difference, and one packed fma
  constexpr uint32_t BASE = BF16 ? 0x43004300u : 0x64006400u;
  const uint32_t s2 = __byte_perm(meta, meta, 0x1010), z2 = __byte_perm(meta, meta, 0x3232);
  uint32_t n[4];
  if constexpr (BITS == 8 && BF16) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t f[2];
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f[j] = __float_as_uint(__uint_as_float(__byte_perm(w[i >> 1], 0x4b000000u, 0x7440 + 2 * (i & 1) + j)) - 8388608.f);
      n[i] = __byte_perm(f[0], f[1], 0x7632);  // the upper halves: n has eight bits
    }
  } else {
    if constexpr (BITS == 4) {
      // nibbles 0 and 4, 1 and 5, ...; put back in order below
#pragma unroll
      for (int i = 0; i < 4; ++i) n[i] = ((w[0] >> (4 * i)) & 0x000f000fu) | BASE;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) n[i] = __byte_perm(w[i >> 1], BASE, i & 1 ? 0x7372 : 0x7170);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = T::sub2(n[i], BASE);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) n[i] = T::fma2(n[i], s2, z2);
  if constexpr (BITS == 8) return make_uint4(n[0], n[1], n[2], n[3]);
  return make_uint4(__byte_perm(n[0], n[1], 0x5410), __byte_perm(n[2], n[3], 0x5410), __byte_perm(n[0], n[1], 0x7632),
                    __byte_perm(n[2], n[3], 0x7632));
}
template <int BITS>
__device__ __forceinline__ void kv_load_words(const uint8_t* from, uint32_t* w) {
  if constexpr (BITS == 4) w[0] = *reinterpret_cast<const uint32_t*>(from);
  else {
    const uint2 x = *reinterpret_cast<const uint2*>(from);
    w[0] = x.x;
    w[1] = x.y;
  }
}

enum KvReadTag : int { kTagKvRead = 103 };

// grid (ceil(blocks / warps per CTA), heads, B): a warp owns the positions of a block of the cache, which one bulk copy brings
template <int BITS, int D, bool BF16>
__global__ void __launch_bounds__(128) kv_read_kernel(const __grid_constant__ KvReadParams p) {
  using Blk = KvBlock<BITS, D>;
  constexpr int LANES = D / 16, PER = 32 / LANES;
  __shared__ __align__(128) uint8_t stage[4][Blk::BYTES];
  __shared__ uint64_t full[4];
  __shared__ CtaAbort abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, h = blockIdx.y;
  if (lane == 0) mbar_init(&full[warp], 1);
  abort_flag.flag = 0;  // every thread the same; another warp sets it only for a wait that ran out, a second later
  fence_mbar_init();
  __syncwarp();
  pdl_grid_dependency_wait();
  int start = p.start != nullptr ? p.start[b] : 0;
  const int count = kv_count(p.cache, p.count != nullptr ? p.count[b] : p.L, start, p.L, b);
  if (count == 0) start = 0;  // whatever it was
  const int off = (blockIdx.x * 4 + warp) * kKvBlockTokens - start % kKvBlockTokens;  // of this warp's block, from start on
  if (off >= p.L) return;
  bool there = false;  // the same for the warp
  if (off < count) {
    const int page = kv_page(p.cache, b, start + off);
    there = page >= 0;
    if (there && lane == 0) {
      mbar_expect_tx(&full[warp], Blk::BYTES);
      bulk_load_1d(stage[warp], kv_block(p.cache, page, h, start + off, Blk::BYTES), Blk::BYTES, &full[warp]);
    }
    __syncwarp();
    if (there && !mbar_wait_warp(&full[warp], 0, &abort_flag, kTagKvRead)) {
      if (lane == 0) mbar_wait_drain(&full[warp], 0, 2000000ull);
      return;
    }
  }
  const uint8_t* blk = stage[warp];
  const int sub = lane / LANES, ch = (lane % LANES) * 8;
  const long long out0 = ((static_cast<long long>(b) * p.cache.heads + h) * p.L + off) * D + ch;
#pragma unroll 2
  for (int base = 0; base < kKvBlockTokens; base += PER) {
    const int tok = base + sub, row = off + tok;
    if (row < 0 || row >= p.L) continue;
    uint4 k[2], v[2];
    if (there && row < count) {
      const uint2 meta = *reinterpret_cast<const uint2*>(blk + Blk::meta_byte(tok));
      const uint32_t flip = tok & 1 ? ~0u : 0u;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t kw[2], vw[2] = {0, 0};
        kv_load_words<BITS>(blk + Blk::k_byte(tok, (ch + i * (D / 2)) * BITS / 8), kw);
        kv_load_words<BITS>(blk + Blk::v_byte(tok, (ch + i * (D / 2)) * BITS / 8), vw);
        vw[0] ^= flip;
        vw[1] ^= flip;
        k[i] = kv_values8<BITS, BF16>(kw, meta.x);
        v[i] = kv_values8<BITS, BF16>(vw, meta.y);
      }
    } else {
      k[0] = k[1] = v[0] = v[1] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long o = out0 + static_cast<long long>(tok) * D + i * (D / 2);
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.k) + o) = k[i];
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.v) + o) = v[i];
    }
  }
}

}  // namespace ab200
