// Attention of a few query rows over a quantised, paged KV cache (the form: kv_format.cuh).
//
//   s_j = (ks_j (q . kn_j) + kz_j sum q) * scale,  p = softmax(s),  o = sum_j p_j vs_j vn_j + sum_j p_j vz_j
// The numbers kn, vn go into the tensor cores as they are; scales and zeros are applied in fp32, to a score and to a probability,
// so that no value of the cache is ever rounded.
//
// What bounds it: reading the cache once, 136 bytes per position and head of K and V at 4 bits and d = 128. At the copy bandwidth
// (6.55 TB/s) an SM takes in a block of 16 positions every 94 cycles, in which its four schedulers issue 376 instructions; a block
// costs a warp about 279 (72 to unpack K, 64 to transpose and unpack V, 16 products, 50 for the softmax, the rest to fetch). So:
//   * every warp works alone, on units of 16 or 32 positions that it fetches itself, 16 bytes a lane at a time, into a ring of its
//     own: no warp waits for another until the last unit of a head is done;
//   * S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16 with positions, then channels, as the 16 rows: eight query rows fill the
//     eight columns (a tcgen05 tile would pad them to 128), and the packed side is an A operand that a lane unpacks in
//     registers, without shared memory in between: a nibble masked out of a word is an fp16 subnormal, n 2^-24 or n 2^-20, and
//     goes into the product as that, or times a power of two where the tensor cores would lose bits of it;
//   * with up to four rows the other four columns repeat them, and each lane takes half of its scores through the softmax;
//   * the reference of the exponentials follows the running maximum only when a score is more than 2^4 above it, and the power of
//     two by which a row's probabilities times scales of V are brought into fp16 range falls when one of them leaves it and rises
//     with the reference (of the products: a large value that has no weight, none any more, or none in this row, costs the others
//     nothing); both are looked at with one vote per unit;
//   * work is dealt out in equal runs over all CTAs, across heads and sequences of whatever lengths (the lengths are on the
//     device, a captured launch sees new ones). A head that lies in one run is finished by its CTA; the others leave
//     maximum, sum and fp32 accumulator in scratch memory, and kv_attn_join_kernel, launched as a programmatic dependent, adds
//     them in order. Nothing is added with atomics: the same call has the same bits.
// The accumulators of the tensor cores drop the bits that do not fit, always the same way. V of odd positions counts from the other end
// (kv_format.cuh), so that both signs occur and the sums stay near zero where a channel's values lie about the middle of their rows'
// ranges: 131072 positions in fp16 are then 2.1e-4 from 64 bits, all of it the rounding of the output, where numbers from 0 were 7e-3
// off. For values at one end of the range, accumulators run over 1024 positions of a warp (HELD) and not over a sequence. A
// probability times its scale goes through the tensor cores in two pieces, its fp16 value and what that leaves: one piece alone is off by
// as much as rounding the output to fp16, and turns one output in a few hundred to the other side of a rounding to bf16. Up to four rows
// the second piece costs no product; beyond, it takes two bf16 rows of eight heads from 22.5 to 24.1 us, four from 32.9 to 37.5.
//
// Measured (B200, us of the device, calls one after another in a captured graph; at the copy bandwidth): 8 sequences of 131072 positions, 32
// heads over 8, d = 128, 4 bits, fp16 210 (174), 5.4 TB/s, in bursts of a few ms, and 232 to 248 when the power limit sets the clock; 2 of
// 16384, 16 heads, 8 bits, bf16 28.4 (21); 32 of up to 8192, 32 over 8, 4 bits, bf16 23.6 (10.8); 16 of up to 4096, four queries, 8 bits,
// fp16 15.2 (3.1); one of 50001, 8 heads over one, d = 256 14.9 (2.0); 2 of 512, 4 heads, d = 64 6.8.
// What is left of the short ones: 3 us until the first unit has come (lengths, table, unit: three trips to memory behind one
// another), 1 us to add the warps' results, 3 us for the second kernel; of the middle ones as well that SMs with the same share
// of the bytes finish up to 25% apart. Tried and not kept, each against the kernel of its time: units by bulk copies and mbarriers (one
// lane's work holds up its warp: 214 -> 220), three units in the ring (the SMs finish further apart, 28.6 -> 30.2 for 8 bits), four CTAs
// per SM (spills, 227), CTAs of one or two warps (the partial results of more runs: 22.2 -> 24.4, 23.2), twice the runs (28.5 -> 35.2).
#pragma once

#include "../fast_div.cuh"
#include "kv_format.cuh"

namespace ab200 {

constexpr int kKvMaxBatch = 4096;  // prefix sums of the work in shared memory

template <int BITS_, int D_, int ROWS_, bool BF16_>
struct KvAttnConfig {
  using Blk = KvBlock<BITS_, D_>;
  static constexpr int BITS = BITS_, D = D_, ROWS = ROWS_;  // 4, 8 or 16 query rows
  static constexpr int NT = (ROWS + 7) / 8;                 // tiles of eight columns
  // Up to four rows stand twice in the eight columns. Then a lane has the scores of positions g and g + 8 that the lane with t ^ 2
  // has as well, and each takes one of the two through the softmax: half the work of a warp there. The probabilities of
  // positions 8 to 15 come to lie in the other four columns, and so does their part of O^T, until the columns are added at the end.
  static constexpr bool HALF = ROWS == 4;
  static constexpr int R = HALF ? 1 : 2;  // of positions g and g + 8, those a lane works on
  static constexpr bool BF16 = BF16_;
  // The sums of V are kept times this until they are divided: below the largest fp32 number for every finite bf16 value, up to half a
  // million positions. bf16 values lose bits below 2^-117 for it.
  static constexpr float VDOWN = BF16 ? 1.f / 16777216.f : 1.f, VUP = 1.f / VDOWN;
  static constexpr int NWARPS = 4, NTHREADS = 32 * NWARPS;
  static constexpr int UNIT_BLOCKS = Blk::BYTES <= 2176 ? 2 : 1;  // a unit of work, and of the ring
  static constexpr int UNIT = UNIT_BLOCKS * kKvBlockTokens;       // positions
  static constexpr int UNIT_BYTES = UNIT_BLOCKS * Blk::BYTES;
  static constexpr int NSTAGE = UNIT_BYTES <= 2304 ? 4 : 2;
  // Units of a warp until its accumulators are added to fp32 sums in shared memory and begin anew. The tensor cores drop the bits that
  // do not fit, always the same way. A channel of V 40 above the others, which puts those at one end of their numbers, 65536 positions
  // in one CTA, fp16: up to 4.6e-4 of sum p |v| beyond the rounding of the output, after 1024 positions 6.1e-5, after 512 3.5e-5;
  // 8 of 131072 take 208, 210 and 213 us.
  static constexpr int HELD = 1024 / UNIT;
  static constexpr int RING_BYTES = NWARPS * NSTAGE * UNIT_BYTES;
  static constexpr int PART_STRIDE = D + 4;  // floats of a row: the rows of a warp's store fall on other banks
  static constexpr int STAT_BYTES = 3 * NWARPS * ROWS * 4;  // reference, sum, sum of p vz
  static constexpr int Q_BYTES = 8 * NT * (D * 2 + 16);  // fragments, and what kv_store_q says of a row
  static constexpr int Q_PASSES = (ROWS * D / 8 + NTHREADS - 1) / NTHREADS;
  // 168 or 255 registers. d = 64 with 16 rows spills up to 104 bytes at 168; with two CTAs per SM and no spills a draft of four (16 of up to
  // 4096, 8 bits) takes 12.7 us instead of 12.9, four of a ragged batch (4 bits, bf16) 26.0 instead of 26.4, four of 131072 positions in 8 bits
  // 134.7 instead of 129.4.
  static constexpr int MIN_CTAS = NT * D <= 128 ? 3 : 2;
  static constexpr int part_bytes(int rows) { return NWARPS * (rows < ROWS ? rows : ROWS) * PART_STRIDE * 4; }
  static int smem_bytes(int rows, int B) { return RING_BYTES + Q_BYTES + STAT_BYTES + part_bytes(rows) + (B + 1) * 8; }
};

struct KvAttnParams {
  KvCacheView cache;
  const int* lengths;  // [B]
  const void* q;       // [B, group * heads, Lq, D]: the rows of a head of the cache are rows = group * Lq neighbours
  void* o;
  float* lse;          // or nullptr
  float* ws;           // 2 slots per CTA
  int B, Lq, rows, row_blocks, causal;
  int whole;           // runs begin where heads begin: nothing to add afterwards
  FastDiv by_grid;     // of the attention kernel, for both
  float scale_log2;
};

// Work: sequence b has n = units(b) of Cfg::UNIT positions for each (head, row block), and a head costs kKvHeadCost units more
// (queries in, partial results out). The CTAs' runs are equal shares of that cost. Measured with 4 / 8 / 12 / 16 / 24 units: 64 sequences
// of 100 to 4000 positions, 8 heads, d = 128, 4 bits 27.8 / 25.2 / 24.3 / 24.9 / 26.7 us (units of 32 positions); 32 of 64 to 4096,
// four queries, 8 bits 35.7 / 31.7 / 27.4 / 25.7 / 25.7 (units of 16).
template <int UNIT>
constexpr int kKvHeadCost = UNIT == 32 ? 12 : 16;
// a / b for quotients far below 2^22: the product with the reciprocal is off by less than one.
__device__ __forceinline__ int kv_div(int a, int b) {
  const int q = static_cast<int>(__int2float_rn(a) * __frcp_rn(__int2float_rn(b))), r = a - q * b;
  return q + (r >= b ? 1 : 0) - (r < 0 ? 1 : 0);
}
constexpr int kKvMinCost = 8;     // of a run: two units for each warp
constexpr int kKvMaxRuns = 2048;  // CTAs of a launch
struct KvRange {  // the first `more` runs are one longer than `each`
  int ctas, each, more;
  __device__ __forceinline__ int first(int cta) const { return cta * each + min(cta, more); }
  __device__ __forceinline__ int owner(int at) const {
    const int split = more * (each + 1);
    return at < split ? kv_div(at, each + 1) : more + kv_div(at - split, each);
  }
};
__device__ __forceinline__ KvRange kv_range(int total, int grid, FastDiv by_grid) {  // total > 0
  KvRange r;
  if (total >= grid * kKvMinCost) {
    r.ctas = grid;
    r.each = fast_div(total, by_grid);
  } else {
    r.ctas = max(total / kKvMinCost, 1);
    r.each = kv_div(total, r.ctas);
  }
  r.more = total - r.each * r.ctas;
  return r;
}
// The length of a sequence as far as its table row reaches; anything else is reported once.
__device__ __forceinline__ int kv_length(const KvAttnParams& p, int b, bool report) {
  const int n = p.lengths[b];
  const long long room = static_cast<long long>(p.cache.table_width) << p.cache.page_shift;
  if (n >= 0 && n <= room) return n;
  if (report) kv_report(kKvBadLength, p.cache.first + b);
  return n < 0 ? 0 : static_cast<int>(room);
}
template <int UNIT>
__device__ __forceinline__ int kv_units(int length) { return (length + UNIT - 1) / UNIT; }

// d = a b + c
__device__ __forceinline__ void kv_mma(float* d, const uint32_t* a, const uint32_t* b, const float* c) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
// 16 bytes from global to shared memory; both addresses multiples of 16.
__device__ __forceinline__ void kv_copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ uint32_t kv_transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Whole numbers as fp16 bit patterns: n in the low bits of a half is the subnormal n 2^-24, a nibble four bits higher n 2^-20. The
// tensor cores take a subnormal as that, but line it up as if its leading bit were set, and drop what lies below the same place as for a
// number with that bit. Of an odd channel of V (4 bits), or of the numbers of V in 8 bits, whose sums have grown past that place, nothing
// is lost that an output shows; the even channels of V (4 bits) and all numbers of K are multiplied up to n 2^-14 first.
constexpr float kKvLoUnit = 16777216.f, kKvHiUnit = 1048576.f, kKvUnit = 16384.f;  // 2^24, 2^20, 2^14
__device__ __forceinline__ uint32_t kv_nibble_lo(uint32_t x) { return x & 0x000f000fu; }  // nibbles 0 and 4
__device__ __forceinline__ uint32_t kv_nibble_hi(uint32_t x) { return x & 0x00f000f0u; }  // nibbles 1 and 5, times 16
__device__ __forceinline__ uint32_t kv_times(uint32_t x, uint32_t up) {
  const __half2 r = __hmul2(reinterpret_cast<__half2&>(x), reinterpret_cast<__half2&>(up));
  return reinterpret_cast<const uint32_t&>(r);
}
__device__ __forceinline__ uint32_t kv_from_lo(uint32_t x) { return kv_times(x, 0x64006400u); }  // 2^10
__device__ __forceinline__ uint32_t kv_from_hi(uint32_t x) { return kv_times(x, 0x54005400u); }  // 2^6
__device__ __forceinline__ uint32_t kv_bytes(uint32_t x, uint32_t sel) { return __byte_perm(x, 0, sel); }

// Over the lanes that work on the same rows: those of one t, with HALF of t and t ^ 2.
template <bool HALF>
__device__ __forceinline__ float kv_max_rows(float x) {
#pragma unroll
  for (int m = HALF ? 2 : 4; m < 32; m <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, m));
  return x;
}
template <bool HALF>
__device__ __forceinline__ float kv_sum_rows(float x) {
#pragma unroll
  for (int m = HALF ? 2 : 4; m < 32; m <<= 1) x += __shfl_xor_sync(0xffffffffu, x, m);
  return x;
}

// Weight of a partial result with reference m and sum l in a row whose largest reference is M. A partial result without a key has
// m = -inf and l = 0; one whose scores are all NaN has m = -inf and l = NaN and must not get lost.
__device__ __forceinline__ float kv_weight(float m, float l, float M) {
  if (m == -INFINITY) return l == 0.f ? 0.f : 1.f;
  return ex2_approx(m - M);
}

// 2^-x of a whole number x from 0; 0 beyond 126, and of NaN (from -inf to -inf).
__device__ __forceinline__ float kv_fall(float x) {
  return __uint_as_float(static_cast<uint32_t>(127 - static_cast<int>(fminf(x, 127.f))) << 23);
}
// 1 / x of a power of two from 2^-126 to 2^126.
__device__ __forceinline__ float kv_inverse(float x) { return __uint_as_float((254u << 23) - __float_as_uint(x)); }

// The state of a warp for one (sequence, head, row block).
template <class Cfg>
struct KvAttnState {
  static constexpr int NT = Cfg::NT, D = Cfg::D;
  uint32_t qb[D / 16][NT][2];  // B fragments of Q
  float sq[NT][2], cq[NT][2];  // of the lane's two columns: sum of q, and what turns a product into a score, both in exp2 units
  int lim[NT][2];              // keys that the row of the column may see
  float m[NT][2], l[NT][2], z[NT][2];
  float acc[D / 16][NT][4];
  float vflip;                 // 0, or 2^bits - 1 for a lane whose positions are odd: their numbers of V are stored as that minus n
  float wup[NT][2];            // what brings a column's probabilities times scales of V into fp16: a power of two, minus at odd positions
};

// The query rows row0 ... of a head, a thread eight channels: fetched early, stored as the fragments of all warps.
template <class Cfg>
__device__ __forceinline__ void kv_load_q(uint4* x, const KvAttnParams& p, long long q_row0, int row0) {
  constexpr int D = Cfg::D;
#pragma unroll
  for (int i = 0; i < Cfg::Q_PASSES; ++i) {
    const int e = (i * Cfg::NTHREADS + static_cast<int>(threadIdx.x)) * 8, row = row0 + e / D;
    x[i] = e < Cfg::ROWS * D && row < p.rows
               ? __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + (q_row0 + row) * D + e % D))
               : make_uint4(0, 0, 0, 0);
  }
}
template <class Cfg>
__device__ __forceinline__ void kv_store_q(const uint4* x, uint8_t* qs, const KvAttnParams& p, int row0, int len) {
  constexpr int D = Cfg::D, CH = D / 4;
  using T = Kv16<Cfg::BF16>;
#pragma unroll
  for (int i = 0; i < Cfg::Q_PASSES; ++i) {
    const int e = (i * Cfg::NTHREADS + static_cast<int>(threadIdx.x)) * 8, row = e / D, ch = e % D;
    const uint32_t u[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
    float f[8], top = 0.f, sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[2 * j] = T::lo(u[j]);
      f[2 * j + 1] = T::hi(u[j]);
      top = fmax3(top, fabsf(f[2 * j]), fabsf(f[2 * j + 1]));
      sum += f[2 * j] + f[2 * j + 1];
    }
#pragma unroll
    for (int m = 1; m < D / 8; m <<= 1) {
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
      sum += __shfl_xor_sync(0xffffffffu, sum, m);
    }
    // q as fp16 times a power of two that puts the row's largest below 2^14: exact, but for channels less than 2^-23 of the largest
    const int ex = top > 0.f ? max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -100) : 13;
    const float up = __uint_as_float(static_cast<uint32_t>(127 + 13 - ex) << 23);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] *= up;
    uint4 w;
    if constexpr (Cfg::BITS == 4) {  // the pairs in which nibbles come out of a word
      w = make_uint4(Kv16<false>::round2(f[0], f[4]), Kv16<false>::round2(f[1], f[5]), Kv16<false>::round2(f[2], f[6]),
                     Kv16<false>::round2(f[3], f[7]));
    } else {
      w = make_uint4(Kv16<false>::round2(f[0], f[1]), Kv16<false>::round2(f[2], f[3]), Kv16<false>::round2(f[4], f[5]),
                     Kv16<false>::round2(f[6], f[7]));
    }
    if (e < Cfg::ROWS * D) {
      // [row / 8][eight channels of a quarter][lane]
      uint4* to = reinterpret_cast<uint4*>(qs) + ((row >> 3) * (D / 32) + ch % CH / 8) * 32 + (row & 7) * 4 + ch / CH;
      to[0] = w;
      if constexpr (Cfg::HALF) to[16] = w;  // column row + 4
      if (ch == 0) {
        const int lim = p.causal ? len - p.Lq + 1 + (row0 + row) % p.Lq : len;
        // the middle one also undoes the 2^-14 of the numbers
        reinterpret_cast<float4*>(qs + 8 * Cfg::NT * D * 2)[row] =
            make_float4(sum * p.scale_log2, p.scale_log2 * kKvUnit * __uint_as_float(static_cast<uint32_t>(min(127 - 13 + ex, 254)) << 23),
                        __int_as_float(lim), 0.f);
      }
    }
  }
}
template <class Cfg>
__device__ __forceinline__ void kv_begin(KvAttnState<Cfg>& st, const uint8_t* qs, int lane) {
  constexpr int NT = Cfg::NT, D = Cfg::D;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint4 w = reinterpret_cast<const uint4*>(qs)[(nt * (D / 32) + j) * 32 + lane];
      st.qb[2 * j][nt][0] = w.x;
      st.qb[2 * j][nt][1] = w.y;
      st.qb[2 * j + 1][nt][0] = w.z;
      st.qb[2 * j + 1][nt][1] = w.w;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 r = reinterpret_cast<const float4*>(qs + 8 * Cfg::NT * D * 2)[nt * 8 + 2 * (lane & (Cfg::HALF ? 1 : 3)) + i];
      st.sq[nt][i] = r.x;
      st.cq[nt][i] = r.y;
      st.lim[nt][i] = __float_as_int(r.z);
      st.m[nt][i] = -INFINITY;
      st.l[nt][i] = st.z[nt][i] = 0.f;
      st.wup[nt][i] = st.vflip != 0.f ? -8.507059e37f : 8.507059e37f;  // 2^126: the first scale that is not zero brings it down
    }
  }
}

// NB blocks of 16 positions at blk, the first of them position pos0. EDGE: some of them are past the length or hidden from some
// row, or (missing, a bit per block) are in no page.
template <class Cfg, int NB, bool EDGE>
__device__ __forceinline__ void kv_attn_blocks(KvAttnState<Cfg>& st, const uint8_t* blk, int pos0, int len, int missing, int lane) {
  constexpr int NT = Cfg::NT, D = Cfg::D, BITS = Cfg::BITS;
  using Blk = typename Cfg::Blk;
  using T = Kv16<Cfg::BF16>;
  constexpr int KW = Blk::KCHUNK / 4;  // words of a position in a lane's share of K
  constexpr int VW = Blk::VCHUNK / 4;  // of V
  constexpr int LANE_UNITS = 2 * Blk::KCHUNK / 16;
  const int g = lane >> 2;

  constexpr int R = Cfg::R;
  const int own = Cfg::HALF ? (lane & 2) * 4 : 0;  // the first position of this lane is g + own

  float y[NB][NT][2 * R];              // scores, in exp2 units
  float vs[NB][R], vz[NB][R];  // of the lane's positions; vz: what V stands for with its numbers 0
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const uint8_t* at = blk + nb * Blk::BYTES;
    float ks[R], kz[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      uint2 meta = *reinterpret_cast<const uint2*>(at + Blk::META + g * 16 + own + 8 * r);
      if constexpr (EDGE) {  // what lies behind the length is whatever was in the page
        if (((missing >> nb) & 1) || pos0 + nb * 16 + g + own + 8 * r >= len) meta = make_uint2(0, 0);
      }
      ks[r] = T::lo(meta.x);
      kz[r] = T::hi(meta.x);
      vs[nb][r] = T::lo(meta.y);
      vz[nb][r] = fmaf(st.vflip, vs[nb][r], T::hi(meta.y)) * Cfg::VDOWN;
    }
    uint32_t w[LANE_UNITS * 4];
#pragma unroll
    for (int u = 0; u < LANE_UNITS; ++u)
      *reinterpret_cast<uint4*>(w + 4 * u) = *reinterpret_cast<const uint4*>(at + (u * 32 + lane) * 16);
    float sum[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[nt][i] = 0.f;
#pragma unroll
    for (int x = 0; x < KW; ++x) {
      const uint32_t a = w[x], c = w[KW + x];  // positions g and g + 8
      auto product = [&](int k, const uint32_t* f) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) kv_mma(sum[nt], f, st.qb[k][nt], sum[nt]);
      };
      if constexpr (BITS == 4) {
        const uint32_t a8 = a >> 8, c8 = c >> 8;
        const uint32_t f0[4] = {kv_from_lo(kv_nibble_lo(a)), kv_from_lo(kv_nibble_lo(c)), kv_from_hi(kv_nibble_hi(a)), kv_from_hi(kv_nibble_hi(c))};
        product(2 * x, f0);
        const uint32_t f1[4] = {kv_from_lo(kv_nibble_lo(a8)), kv_from_lo(kv_nibble_lo(c8)), kv_from_hi(kv_nibble_hi(a8)),
                                kv_from_hi(kv_nibble_hi(c8))};
        product(2 * x + 1, f1);
      } else {
        const uint32_t f0[4] = {kv_from_lo(kv_bytes(a, 0x4140)), kv_from_lo(kv_bytes(c, 0x4140)), kv_from_lo(kv_bytes(a, 0x4342)),
                                kv_from_lo(kv_bytes(c, 0x4342))};
        product(x, f0);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2 * R; ++i)
        y[nb][nt][i] = fmaf(ks[i >> 1] * st.cq[nt][i & 1], Cfg::HALF && own ? sum[nt][i + 2] : sum[nt][i], kz[i >> 1] * st.sq[nt][i & 1]);
  }

  // probabilities against the present references, and weights of the numbers of V
  float e[NB][NT][2 * R], x[NB][NT][2 * R], wt[NB][NT][2 * R];
  bool hidden[NB][NT][2 * R];
  auto probabilities = [&] {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2 * R; ++i) {
          const int r = i >> 1, c = i & 1;  // position g + own + 8 r, the lane's column c
          e[nb][nt][i] = y[nb][nt][i] - st.m[nt][c];  // of the very number that the reference comes from: below 0 whatever its size
          if constexpr (EDGE) {
            hidden[nb][nt][i] = ((missing >> nb) & 1) || pos0 + nb * 16 + g + own + 8 * r >= st.lim[nt][c];
            if (hidden[nb][nt][i]) e[nb][nt][i] = -INFINITY;
          }
          x[nb][nt][i] = ex2_approx(e[nb][nt][i]);
          wt[nb][nt][i] = EDGE && hidden[nb][nt][i] ? 0.f : x[nb][nt][i] * vs[nb][r] * st.wup[nt][c];
        }
  };
  probabilities();
  float etop = -INFINITY, wtop = 0.f;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        etop = fmax3(etop, e[nb][nt][2 * r], e[nb][nt][2 * r + 1]);
        wtop = fmax3(wtop, fabsf(wt[nb][nt][2 * r]), fabsf(wt[nb][nt][2 * r + 1]));
      }
  if (__any_sync(0xffffffffu, etop > 4.f || wtop > 16384.f)) {
    // per column: the largest score, and the largest score plus logarithm of a scale of V, from the scores themselves
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = -INFINITY, wide = -INFINITY;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (!EDGE || !hidden[nb][nt][2 * r + c]) top = fmaxf(top, y[nb][nt][2 * r + c]);
        // The reference is a whole number, so that what it moves by is taken out of the sums exactly.
        const float mn = fmaxf(st.m[nt][c], ceilf(kv_max_rows<Cfg::HALF>(top)));
        // of the largest weight; a logarithm added to a score would be lost where a step of fp32 is above it
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int r = 0; r < R; ++r)
            if (!EDGE || !hidden[nb][nt][2 * r + c]) wide = fmaxf(wide, y[nb][nt][2 * r + c] - mn + __log2f(vs[nb][r]));
        wide = kv_max_rows<Cfg::HALF>(wide);
        const int drop = static_cast<int>(fminf(mn - st.m[nt][c], 252.f));  // 252 from -inf too, and where nothing was seen yet
        const float f = kv_fall(mn - st.m[nt][c]);
        st.m[nt][c] = mn;
        st.l[nt][c] *= f;
        st.z[nt][c] *= f;
        // What was added before has lost 1 / f of its weight, and the range of the weights may rise by as much. A weight above 2^8
        // is brought there or just below it: what it is needed for reaches 2^-32 of that, and the next ones have room to grow.
        const float was = fabsf(st.wup[nt][c]);
        const int risen = min(static_cast<int>(__float_as_uint(was) >> 23) + drop, 253);
        const uint32_t up = static_cast<uint32_t>(min(risen, 135 - static_cast<int>(ceilf(fmaxf(wide, -200.f))))) << 23;
        st.wup[nt][c] = st.vflip != 0.f ? -__uint_as_float(up) : __uint_as_float(up);
        const float g2 = f * __uint_as_float(up) * kv_inverse(was);
#pragma unroll
        for (int u = 0; u < D / 16; ++u) {
          st.acc[u][nt][c] *= g2;
          st.acc[u][nt][2 + c] *= g2;
        }
      }
    probabilities();
  }

  uint32_t pb[NB][NT][2], pl[NB][NT][2];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float* w2 = &wt[nb][nt][2 * r];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int i = 2 * r + c;
          st.l[nt][c] += x[nb][nt][i];
          if (!EDGE || !hidden[nb][nt][i]) st.z[nt][c] = fmaf(x[nb][nt][i], vz[nb][r], st.z[nt][c]);
        }
        hi[r] = Kv16<false>::round2(w2[0], w2[1]);
        lo[r] = Kv16<false>::round2(w2[0] - Kv16<false>::lo(hi[r]), w2[1] - Kv16<false>::hi(hi[r]));
      }
      if constexpr (Cfg::HALF) {
        // Transposed, lanes of columns 0 to 3 have positions 0 to 7, those of columns 4 to 7 positions 8 to 15; the other places of
        // the fragment take the second pieces, which columns 4 to 7 and 0 to 3 then hold: all columns of a row are added at the end.
        const uint32_t most = kv_transpose8x8(hi[0]);
        const uint32_t rest = __shfl_xor_sync(0xffffffffu, kv_transpose8x8(lo[0]), 16);
        pb[nb][nt][0] = lane < 16 ? most : rest;
        pb[nb][nt][1] = lane < 16 ? rest : most;
      } else {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          pb[nb][nt][r] = kv_transpose8x8(hi[r]);
          pl[nb][nt][r] = kv_transpose8x8(lo[r]);
        }
      }
    }
  uint32_t w[NB][LANE_UNITS * 4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int u = 0; u < LANE_UNITS; ++u)
      *reinterpret_cast<uint4*>(w[nb] + 4 * u) = *reinterpret_cast<const uint4*>(blk + nb * Blk::BYTES + Blk::CODE + (u * 32 + lane) * 16);
  constexpr int TILES = BITS == 4 ? 4 : 2;  // of 16 channels in a word of each of eight lanes
#pragma unroll
  for (int v = 0; v < VW; ++v) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      // positions 2t, 2t + 1 | 2t + 8, 2t + 9: their halves side by side, then pairs of one channel
      const uint32_t a = w[nb][v], b = w[nb][VW + v], c = w[nb][2 * VW + v], d = w[nb][3 * VW + v];
      uint32_t ab[2] = {__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632)};
      uint32_t cd[2] = {__byte_perm(c, d, 0x5410), __byte_perm(c, d, 0x7632)};
#pragma unroll
      for (int i = 0; i < TILES; ++i) {
        uint32_t f[4];
        if constexpr (BITS == 4) {
          const uint32_t p0 = i & 1 ? ab[i >> 1] >> 8 : ab[i >> 1], p1 = i & 1 ? cd[i >> 1] >> 8 : cd[i >> 1];
          f[0] = kv_from_lo(kv_nibble_lo(p0));
          f[1] = kv_nibble_hi(p0);
          f[2] = kv_from_lo(kv_nibble_lo(p1));
          f[3] = kv_nibble_hi(p1);
        } else {
          f[0] = kv_bytes(ab[i], 0x4240);
          f[1] = kv_bytes(ab[i], 0x4341);
          f[2] = kv_bytes(cd[i], 0x4240);
          f[3] = kv_bytes(cd[i], 0x4341);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float* acc = st.acc[TILES * v + i][nt];
          kv_mma(acc, f, pb[nb][nt], acc);
          if constexpr (!Cfg::HALF) kv_mma(acc, f, pl[nb][nt], acc);
        }
      }
    }
  }
}

template <class Cfg>
__global__ void __launch_bounds__(Cfg::NTHREADS, Cfg::MIN_CTAS) kv_attn_kernel(const __grid_constant__ KvAttnParams p) {
  using Blk = typename Cfg::Blk;
  constexpr int NT = Cfg::NT, D = Cfg::D, NW = Cfg::NWARPS, ROWS = Cfg::ROWS, NSTAGE = Cfg::NSTAGE, PS = Cfg::PART_STRIDE;
  using T = Kv16<Cfg::BF16>;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* qs = smem + Cfg::RING_BYTES;                                         // kv_store_q
  float* stat = reinterpret_cast<float*>(qs + Cfg::Q_BYTES);                    // [3][NW][ROWS]
  __shared__ int scan[2][NW];
  const int part_rows = min(ROWS, p.rows);
  float* part = reinterpret_cast<float*>(qs + Cfg::Q_BYTES + Cfg::STAT_BYTES);  // [NW][part_rows][PS]
  int* pre = reinterpret_cast<int*>(part + NW * part_rows * PS);  // [B + 1]: units of the sequences before, for one head and row block
  int* costs = pre + p.B + 1;                                     // [B + 1]: the same with the heads' cost

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const int per_seq = p.cache.heads * p.row_blocks;

  pdl_grid_dependency_wait();  // launched as a programmatic dependent: what is in front has completed from here on
  // only now may the join kernel start, which reads the lengths before it waits for this one
  pdl_launch_dependents();
  int run = 0, run_cost = 0;
  for (int b0 = 0; b0 < p.B; b0 += Cfg::NTHREADS) {
    const int b = b0 + threadIdx.x;
    const int n = b < p.B ? kv_units<Cfg::UNIT>(kv_length(p, b, blockIdx.x == 0)) : 0;
    int x = n;
#pragma unroll
    for (int m = 1; m < 32; m <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, m);
      if (lane >= m) x += y;
    }
    const uint32_t some = __ballot_sync(0xffffffffu, n > 0);
    if (lane == 31) {
      scan[0][warp] = x;
      scan[1][warp] = __popc(some);
    }
    __syncthreads();
    int before = run, heads = 0;
    run_cost -= run;  // of the heads alone
    int before_cost = run_cost;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) {
        before += scan[0][w];
        before_cost += kKvHeadCost<Cfg::UNIT> * scan[1][w];
      }
      run += scan[0][w];
      heads += scan[1][w];
    }
    run_cost += kKvHeadCost<Cfg::UNIT> * heads + run;
    if (b < p.B) {
      pre[b] = before + x - n;
      costs[b] = before + x - n + before_cost + kKvHeadCost<Cfg::UNIT> * __popc(some & ((1u << lane) - 1u));
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    pre[p.B] = run;
    costs[p.B] = run_cost;
  }
  // sequences without a position: zeros
  for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
    if (kv_length(p, b, false) != 0) continue;
    const long long n = static_cast<long long>(p.cache.heads) * p.rows;
    for (long long i = threadIdx.x; i < n * (D / 8); i += Cfg::NTHREADS)
      reinterpret_cast<uint4*>(p.o)[b * n * (D / 8) + i] = make_uint4(0, 0, 0, 0);
    if (p.lse != nullptr)
      for (long long i = threadIdx.x; i < n; i += Cfg::NTHREADS) p.lse[b * n + i] = -INFINITY;
  }
  const int total = run_cost * per_seq;  // the host has seen to it that all of this fits
  __syncthreads();
  if (total == 0) return;
  const KvRange range = kv_range(total, gridDim.x, p.by_grid);
  if (blockIdx.x >= range.ctas) return;

  // the last b with prefix[b] * per_seq <= at: the sequence, one that has units, of a place below the whole
  auto find = [&](const int* prefix, int at) {  // the same for the whole warp: 32 places at once
    int lo = 0;
    for (int step = p.B <= 32 ? 1 : p.B <= 1024 ? 32 : 1024;; step >>= 5) {
      const int i = lo + lane * step;
      const uint32_t below = __ballot_sync(0xffffffffu, i < p.B && prefix[i] * per_seq <= at);
      lo += (__popc(below) - 1) * step;  // prefix[lo] is: the lanes below are the first ones
      if (step == 1) return lo;
    }
  };
  auto find_lane = [&](int at) {
    int lo = 0, hi = p.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] * per_seq <= at) lo = mid;
      else hi = mid;
    }
    return lo;
  };
  // a place in the order of costs, where a head's own cost comes before its units: what it falls on, and the units in front of it
  struct Place {
    int b, n, item, in_head, units;
  };
  auto place = [&](int cost) {
    Place x;
    x.b = find(costs, min(cost, total - 1));
    x.n = pre[x.b + 1] - pre[x.b];
    const int rem = min(cost, total - 1) - costs[x.b] * per_seq;
    x.item = kv_div(rem, x.n + kKvHeadCost<Cfg::UNIT>);
    x.in_head = rem - x.item * (x.n + kKvHeadCost<Cfg::UNIT>);
    const int units = p.whole ? (x.in_head > 0 ? x.n : 0) : max(x.in_head - kKvHeadCost<Cfg::UNIT>, 0);
    x.units = cost < total ? pre[x.b] * per_seq + x.item * x.n + units : run * per_seq;
    return x;
  };
  const Place begin = place(range.first(blockIdx.x)), end = place(range.first(blockIdx.x + 1));
  const int t0 = begin.units, mine = end.units - t0;
  if (mine == 0) return;

  // a head's share of the run
  struct Part {
    int b, head, n, from, to, row0, len;  // units [from, to) of n
    long long q_row0;
  };
  auto part_of = [&](int b, int n, int item, int from, int left) {
    Part x;
    x.b = b;
    x.n = n;
    x.head = p.row_blocks == 1 ? item : item / p.row_blocks;
    x.from = from;
    x.to = min(n, from + left);
    x.row0 = (item - x.head * p.row_blocks) * ROWS;
    x.len = kv_length(p, b, false);
    x.q_row0 = (static_cast<long long>(b) * p.cache.heads + x.head) * p.rows;
    return x;
  };
  auto part_at = [&](int done) {  // what comes after so many units of the run
    const int at = t0 + done, b = find(pre, at), n = pre[b + 1] - pre[b], rem = at - pre[b] * per_seq, item = kv_div(rem, n);
    return part_of(b, n, item, rem - item * n, mine - done);
  };
  Part cur = p.whole ? part_at(0) : part_of(begin.b, begin.n, begin.item, max(begin.in_head - kKvHeadCost<Cfg::UNIT>, 0), mine);
  uint4 qx[Cfg::Q_PASSES];
  kv_load_q<Cfg>(qx, p, cur.q_row0, cur.row0);

  // ---------------------------------------------------------------------------------- fetching: unit k of this warp is t0 + warp + NW k
  uint8_t* ring = smem + warp * NSTAGE * Cfg::UNIT_BYTES;
  const int nunits = mine > warp ? (mine - warp + NW - 1) / NW : 0;
  unsigned long long src0 = 0, src1 = 0;  // lane i: blocks of unit (k / 32) * 32 + i, 0: none there
  auto look_up = [&](int k0) {
    src0 = src1 = 0;
    const int k = k0 + lane;
    if (k < nunits) {
      int unit = warp + NW * k, b, head, pos;
      if (k0 == 0 && unit < cur.to - cur.from) {  // in the run's first head, as most of the first ones are
        b = cur.b;
        head = cur.head;
        pos = (cur.from + unit) * Cfg::UNIT;
      } else {
        unit += t0;
        b = find_lane(unit);
        const int n = pre[b + 1] - pre[b], rem = unit - pre[b] * per_seq, item = kv_div(rem, n);
        pos = (rem - item * n) * Cfg::UNIT;
        head = p.row_blocks == 1 ? item : item / p.row_blocks;
      }
      const int len = kv_length(p, b, false);
      const int pg0 = kv_page(p.cache, b, pos);
      if (pg0 >= 0) src0 = reinterpret_cast<unsigned long long>(kv_block(p.cache, pg0, head, pos, Blk::BYTES));
      if (Cfg::UNIT_BLOCKS > 1 && pos + kKvBlockTokens < len) {
        const int pg1 = p.cache.page_shift > 4 ? pg0 : kv_page(p.cache, b, pos + kKvBlockTokens);
        if (pg1 >= 0) src1 = reinterpret_cast<unsigned long long>(kv_block(p.cache, pg1, head, pos + kKvBlockTokens, Blk::BYTES));
      }
    }
  };
  // Every lane brings 16 bytes at a time; one group of copies per unit, empty ones behind the last.
  int fetched = 0, missing = 0;  // missing: of the units in the ring, a bit for each block that is in no page
  auto fetch = [&](int slot) {  // converged warp
    if (fetched < nunits) {
      if ((fetched & 31) == 0) look_up(fetched);
      constexpr int FULL = Blk::BYTES / 512, REST = Blk::BYTES % 512 / 16;  // whole turns of the warp for a block, lanes of one more
      unsigned long long a[2];
      a[0] = __shfl_sync(0xffffffffu, src0, fetched & 31);
      a[1] = Cfg::UNIT_BLOCKS > 1 ? __shfl_sync(0xffffffffu, src1, fetched & 31) : 0ull;
      const uint32_t to = smem_u32(ring + slot * Cfg::UNIT_BYTES) + lane * 16;
      missing &= ~(3 << (2 * slot));
#pragma unroll
      for (int i = 0; i < Cfg::UNIT_BLOCKS; ++i) {
        if (a[i] == 0) {
          missing |= 1 << (2 * slot + i);
          continue;
        }
        const uint8_t* from = reinterpret_cast<const uint8_t*>(a[i]) + lane * 16;
#pragma unroll
        for (int j = 0; j < FULL; ++j) kv_copy16(to + i * Blk::BYTES + j * 512, from + j * 512);
        if (REST > 0 && lane < REST) kv_copy16(to + i * Blk::BYTES + FULL * 512, from + FULL * 512);
      }
      ++fetched;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < NSTAGE; ++i) fetch(i);
  kv_store_q<Cfg>(qx, qs, p, cur.row0, cur.len);
  __syncthreads();

  // ---------------------------------------------------------------------------------- the run, head by head
  int k = 0, slot = 0;  // units of this warp that are done; where the next one is
  KvAttnState<Cfg> st;
  st.vflip = (lane >> 2) & 1 ? static_cast<float>((1 << Cfg::BITS) - 1) : 0.f;
  for (int done = 0;;) {  // units of the run before this head
    kv_begin<Cfg>(st, qs, lane);
    const int clear = p.causal ? cur.len - p.Lq + 1 : cur.len;  // positions below this are seen by every row
    const int todo = done + (cur.to - cur.from);
    const int kend = todo > warp ? (todo - warp + NW - 1) / NW : 0;
    int pos = (cur.from + warp + NW * k - done) * Cfg::UNIT;
    const int g = lane >> 2, t = lane & 3;
    const int nrows = min(ROWS, p.rows - cur.row0);
    // what the numbers were taken for: odd channels of 4 bits times 16
    constexpr float EVEN = (Cfg::BITS == 4 ? kKvUnit : kKvLoUnit) * Cfg::VDOWN, ODD = (Cfg::BITS == 4 ? kKvHiUnit : kKvLoUnit) * Cfg::VDOWN;
    for (bool first = true;; first = false) {
#pragma unroll
      for (int u = 0; u < D / 16; ++u)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int i = 0; i < 4; ++i) st.acc[u][nt][i] = 0.f;
      for (const int kstop = min(kend, k + Cfg::HELD); k < kstop; ++k, pos += NW * Cfg::UNIT) {
        asm volatile("cp.async.wait_group %0;" ::"n"(NSTAGE - 1) : "memory");
        __syncwarp();
        const uint8_t* blk = ring + slot * Cfg::UNIT_BYTES;
        const int gone = (missing >> (2 * slot)) & 3;
        if (gone == 0 && pos + Cfg::UNIT <= clear) {
          kv_attn_blocks<Cfg, Cfg::UNIT_BLOCKS, false>(st, blk, pos, cur.len, 0, lane);
        } else {
#pragma unroll 1
          for (int i = 0; i < Cfg::UNIT_BLOCKS && pos + i * kKvBlockTokens < cur.len; ++i)
            kv_attn_blocks<Cfg, 1, true>(st, blk + i * Blk::BYTES, pos + i * kKvBlockTokens, cur.len, (gone >> i) & 1, lane);
        }
        __syncwarp();  // every lane has read the slot
        fetch(slot);
        slot = slot + 1 == NSTAGE ? 0 : slot + 1;
      }
      // the accumulators go to the warp's partial result
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int row = nt * 8 + 2 * t + c;
          const float down = kv_inverse(fabsf(st.wup[nt][c]));  // a factor of its own: with EVEN or ODD it may exceed fp32
          if constexpr (Cfg::HALF) {
#pragma unroll
            for (int u = 0; u < D / 16; ++u) {
              st.acc[u][nt][c] += __shfl_xor_sync(0xffffffffu, st.acc[u][nt][c], 2);
              st.acc[u][nt][2 + c] += __shfl_xor_sync(0xffffffffu, st.acc[u][nt][2 + c], 2);
            }
          }
          if (row < nrows) {
            float* dst = part + (warp * part_rows + row) * PS + g * (D / 8);
            const float f = first ? 0.f : kv_fall(st.m[nt][c] - stat[warp * ROWS + row]);  // what is there is for an older reference
#pragma unroll
            for (int u = 0; u < D / 16; u += 2) {
              float4 x = make_float4(st.acc[u][nt][c] * EVEN * down, st.acc[u][nt][2 + c] * ODD * down,
                                     st.acc[u + 1][nt][c] * EVEN * down, st.acc[u + 1][nt][2 + c] * ODD * down);
              if (!first) {
                const float4 y = *reinterpret_cast<const float4*>(dst + 2 * u);
                x = make_float4(fmaf(y.x, f, x.x), fmaf(y.y, f, x.y), fmaf(y.z, f, x.z), fmaf(y.w, f, x.w));
              }
              *reinterpret_cast<float4*>(dst + 2 * u) = x;
            }
          }
        }
      __syncwarp();  // every lane has read the reference
      if (g == 0) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c)
            if (nt * 8 + 2 * t + c < ROWS) stat[warp * ROWS + nt * 8 + 2 * t + c] = st.m[nt][c];
      }
      if (k >= kend) break;
    }
    const bool more = todo < mine;
    Part next;
    if (more) {
      next = part_at(todo);
      kv_load_q<Cfg>(qx, p, next.q_row0, next.row0);
    }

    // the four warps' partial results
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float l = kv_sum_rows<Cfg::HALF>(st.l[nt][c]), z = kv_sum_rows<Cfg::HALF>(st.z[nt][c]);
        const int row = nt * 8 + 2 * t + c;
        if (g == 0 && row < ROWS) {
          stat[(1 * NW + warp) * ROWS + row] = l;
          stat[(2 * NW + warp) * ROWS + row] = z;
        }
      }
    __syncthreads();
    const bool whole = cur.from == 0 && cur.to == cur.n;
    float* slot_o = p.ws + (2ll * blockIdx.x + (done == 0 ? 0 : 1)) * (ROWS * (D + 2));
    float* slot_m = slot_o + ROWS * D;
    for (int i = threadIdx.x; i < nrows * (D / 4); i += Cfg::NTHREADS) {
      const int row = i / (D / 4), c4 = i % (D / 4);
      float M = -INFINITY, L = 0.f, Z = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) M = fmaxf(M, stat[w * ROWS + row]);
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float lw = stat[(NW + w) * ROWS + row];
        const float f = kv_weight(stat[w * ROWS + row], lw, M);
        const float4 y = *reinterpret_cast<const float4*>(part + (w * part_rows + row) * PS + c4 * 4);
        L = fmaf(f, lw, L);
        Z = fmaf(f, stat[(2 * NW + w) * ROWS + row], Z);
        x.x = fmaf(f, y.x, x.x);
        x.y = fmaf(f, y.y, x.y);
        x.z = fmaf(f, y.z, x.z);
        x.w = fmaf(f, y.w, x.w);
      }
      x.x += Z;
      x.y += Z;
      x.z += Z;
      x.w += Z;
      if (whole) {
        const float inv = L == 0.f ? 0.f : 1.f / L * Cfg::VUP;
        const long long row_at = cur.q_row0 + cur.row0 + row;
        reinterpret_cast<uint2*>(p.o)[row_at * (D / 4) + c4] = make_uint2(T::round2(x.x * inv, x.y * inv), T::round2(x.z * inv, x.w * inv));
        if (p.lse != nullptr && c4 == 0) p.lse[row_at] = L == 0.f ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
      } else {
        reinterpret_cast<float4*>(slot_o)[i] = x;
        if (c4 == 0) {
          slot_m[row] = M;
          slot_m[ROWS + row] = L;
        }
      }
    }
    if (!more) break;
    kv_store_q<Cfg>(qx, qs, p, next.row0, next.len);  // every warp has read the fragments before the barrier above
    __syncthreads();
    cur = next;
    done = todo;
  }
}

// Adds the partial results of the heads that lie in more than one run, in the order of the runs. grid (B * heads * row blocks, GY): a
// task is one row and 64 channels of it, and a block takes every GY-th. Up to 64 parts (24 where a block has a single task): a warp a
// task, eight loads of a lane in flight. More (few heads make up the whole batch): the block turns the references of all parts into
// weights, then its warps add them.
template <int D, int ROWS, int UNIT, bool BF16>
__global__ void __launch_bounds__(512) kv_attn_join_kernel(const __grid_constant__ KvAttnParams p, int grid) {
  using T = Kv16<BF16>;
  constexpr float VUP = KvAttnConfig<4, D, ROWS, BF16>::VUP;
  constexpr int STRIDE = ROWS * (D + 2);
  __shared__ float2 weight[kKvMaxRuns];  // of a part: reference, then weight; sum
  __shared__ float red[2][16];
  __shared__ float2 so[16][32];
  __shared__ int before[16], all[16];
  const int NT = blockDim.x, NW = NT >> 5;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_seq = p.cache.heads * p.row_blocks;
  const int b = blockIdx.x / per_seq, item = blockIdx.x % per_seq;
  const int row0 = (item % p.row_blocks) * ROWS, nrows = min(ROWS, p.rows - row0);
  int mine_before = 0, mine_all = 0, heads_before = 0, heads_all = 0;
  for (int i = threadIdx.x; i < p.B; i += NT) {
    const int n = kv_units<UNIT>(kv_length(p, i, false));
    mine_all += n;
    heads_all += n > 0;
    if (i < b) {
      mine_before += n;
      heads_before += n > 0;
    }
  }
  mine_before = __reduce_add_sync(0xffffffffu, mine_before + kKvHeadCost<UNIT> * heads_before);
  mine_all = __reduce_add_sync(0xffffffffu, mine_all + kKvHeadCost<UNIT> * heads_all);
  if (lane == 0) {
    before[warp] = mine_before;
    all[warp] = mine_all;
  }
  __syncthreads();
  int first = 0, total = 0;
  for (int w = 0; w < NW; ++w) {
    first += before[w];
    total += all[w];
  }
  const int n = kv_units<UNIT>(kv_length(p, b, false));
  int c0 = 0, c1 = 0;
  KvRange range{};
  if (n > 0) {
    first = first * per_seq + item * (n + kKvHeadCost<UNIT>);  // in costs
    range = kv_range(total * per_seq, grid, p.by_grid);
    c0 = range.owner(first + kKvHeadCost<UNIT>);
    c1 = range.owner(first + kKvHeadCost<UNIT> + n - 1);
  }
  // nothing is read or written before the kernel in front has completed; every thread waits, so that this one completes after it
  pdl_grid_dependency_wait();
  if (c0 == c1) return;
  const int parts = c1 - c0 + 1;
  // a part is its run's first thing, unless the head begins inside the run
  const float* parts_ws = p.ws + 2ll * c0 * STRIDE;
  const int part0 = range.first(c0) >= first ? 0 : STRIDE;
  auto part_at = [&](int i) { return parts_ws + (i == 0 ? part0 : 2 * STRIDE * i); };
  constexpr int PAIRS = D / 64;
  const int tasks = nrows * PAIRS;
  const long long out0 = (static_cast<long long>(b) * p.cache.heads + item / p.row_blocks) * p.rows + row0;
  auto store = [&](int row, int pair, float2 x, float L) {
    const float inv = L == 0.f ? 0.f : 1.f / L * VUP;
    reinterpret_cast<uint32_t*>(p.o)[(out0 + row) * (D / 2) + pair * 32 + lane] = T::round2(x.x * inv, x.y * inv);
  };
  auto store_lse = [&](int row, float M, float L) {
    if (p.lse != nullptr) p.lse[out0 + row] = L == 0.f ? -INFINITY : (M + __log2f(L)) * 0.6931471805599453f;
  };
  if (parts <= (gridDim.y >= tasks ? 24 : 64)) {
    for (int task = blockIdx.y + gridDim.y * warp; task < tasks; task += gridDim.y * NW) {
      const int row = task / PAIRS, pair = task % PAIRS;
      float m[2], l[2], M = -INFINITY, L = 0.f;
      float2 y[8];
      auto fetch = [&](int i0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (i0 + j < parts) y[j] = reinterpret_cast<const float2*>(part_at(i0 + j) + row * D)[pair * 32 + lane];
      };
      fetch(0);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const bool there = lane + 32 * j < parts;
        const float* at = part_at(there ? lane + 32 * j : 0) + ROWS * D + row;
        m[j] = there ? at[0] : -INFINITY;
        l[j] = there ? at[ROWS] : 0.f;
        M = fmaxf(M, m[j]);
      }
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, k));
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        m[j] = kv_weight(m[j], l[j], M);
        L = fmaf(m[j], l[j], L);
      }
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) L += __shfl_xor_sync(0xffffffffu, L, k);
      float2 x = make_float2(0.f, 0.f);
      for (int i0 = 0; i0 < parts; i0 += 8) {
        if (i0 > 0) fetch(i0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float w = __shfl_sync(0xffffffffu, i0 < 32 ? m[0] : m[1], i0 + j);
          if (i0 + j < parts) {
            x.x = fmaf(w, y[j].x, x.x);
            x.y = fmaf(w, y[j].y, x.y);
          }
        }
      }
      store(row, pair, x, L);
      if (pair == 0 && lane == 0) store_lse(row, M, L);
    }
    return;
  }
  for (int task = blockIdx.y; task < tasks; task += gridDim.y) {
    const int row = task / PAIRS, pair = task % PAIRS;
    float top = -INFINITY;
    for (int i = threadIdx.x; i < parts; i += NT) {
      const float* at = part_at(i) + ROWS * D + row;
      weight[i] = make_float2(at[0], at[ROWS]);  // its own, in a moment
      top = fmaxf(top, weight[i].x);
    }
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
    if (lane == 0) red[0][warp] = top;
    __syncthreads();
    float M = red[0][0];
    for (int w = 1; w < NW; ++w) M = fmaxf(M, red[0][w]);
    float sum = 0.f;
    for (int i = threadIdx.x; i < parts; i += NT) {
      const float2 ml = weight[i];
      const float w = kv_weight(ml.x, ml.y, M);
      weight[i].x = w;
      sum = fmaf(w, ml.y, sum);
    }
#pragma unroll
    for (int k = 1; k < 32; k <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if (lane == 0) red[1][warp] = sum;
    __syncthreads();
    float L = 0.f;
    for (int w = 0; w < NW; ++w) L += red[1][w];
    float2 x = make_float2(0.f, 0.f);
    for (int i0 = warp; i0 < parts; i0 += 8 * NW) {
      float2 y[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j * NW < parts) y[j] = reinterpret_cast<const float2*>(part_at(i0 + j * NW) + row * D)[pair * 32 + lane];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (i0 + j * NW < parts) {
          const float w = weight[i0 + j * NW].x;
          x.x = fmaf(w, y[j].x, x.x);
          x.y = fmaf(w, y[j].y, x.y);
        }
    }
    so[warp][lane] = x;
    __syncthreads();
    if (warp == 0) {
      for (int w = 1; w < NW; ++w) {
        x.x += so[w][lane].x;
        x.y += so[w][lane].y;
      }
      store(row, pair, x, L);
      if (pair == 0 && lane == 0) store_lse(row, M, L);
    }
    __syncthreads();
  }
}

}  // namespace ab200
