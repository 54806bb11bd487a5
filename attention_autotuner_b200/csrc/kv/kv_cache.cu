// libattn_b200_kv.so: the quantised KV cache (declarations in include/attn_b200_kv.h). A library of its own, as every tile
// configuration is: its own status words and error text, and it can be built beside libattn_b200.so.
#include "../../../include/attn_b200_kv.h"

#include <algorithm>
#include <array>
#include <atomic>

#include "../host_common.cuh"
#include "kv_attn.cuh"
#include "kv_write.cuh"

using namespace ab200;

namespace {

// The mirror's fourth word is kv_report's.
int kv_check_prior(const char* what) {
  if (int rc = check_prior_status(what)) return rc;
  volatile int* m = status_mirror();
  if (m == nullptr) return kErrCuda;
  if (m[3] != 0) {
    const int w = m[3];
    return fail(kErrDevice, "%s: an earlier call found %s of sequence %d; it left those positions out. Read and clear the status "
                "(attn_b200_kv_status(1)) before launching again",
                what, (w & 255) == kKvBadPage ? "a page that does not exist in the table" : "a length, start or count out of range", w >> 8);
  }
  return kOk;
}

// The tensors' device is the calling thread's.
int kv_check_device(const void* ptr, const char* what) {
  cudaPointerAttributes at;
  if (cudaPointerGetAttributes(&at, ptr) != cudaSuccess)
    return fail(kErrCuda, "%s: cudaPointerGetAttributes: %s", what, cudaGetErrorString(cudaGetLastError()));
  int cur = -1;
  cudaGetDevice(&cur);
  if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged)
    return fail(kErrInvalidArgument, "%s: tensor pointer is not device memory", what);
  if (at.type == cudaMemoryTypeDevice && cur != at.device)
    return fail(kErrInvalidArgument, "%s: tensors live on device %d but the calling thread's current device is %d", what, at.device, cur);
  return kOk;
}

int kv_view(KvCacheView* c, const attn_b200_kv_cache* cache, const int* table, int table_stride, int table_width, int B, const char* what) {
  if (cache == nullptr || cache->data == nullptr || table == nullptr) return fail(kErrInvalidArgument, "%s: null pointer", what);
  if (cache->bits != 4 && cache->bits != 8) return fail(kErrInvalidArgument, "%s: bits=%d (4 or 8)", what, cache->bits);
  if (cache->head_dim != 64 && cache->head_dim != 128 && cache->head_dim != 256)
    return fail(kErrUnsupported, "%s: head dimension %d (64, 128 or 256)", what, cache->head_dim);
  if (cache->dtype != ATTN_B200_KV_F16 && cache->dtype != ATTN_B200_KV_BF16) return fail(kErrInvalidArgument, "%s: dtype %d", what, cache->dtype);
  const int ps = cache->page_size;
  if (ps < 16 || ps > 65536 || (ps & (ps - 1)) != 0)
    return fail(kErrInvalidArgument, "%s: page_size=%d (a power of two from 16 to 65536)", what, ps);
  if (cache->num_pages <= 0 || cache->heads <= 0 || cache->heads > 65535)
    return fail(kErrInvalidArgument, "%s: %d pages of %d heads", what, cache->num_pages, cache->heads);
  if (!aligned16(cache->data)) return fail(kErrInvalidArgument, "%s: the cache must be 16-byte aligned", what);
  if (B <= 0 || B > 65535) return fail(kErrInvalidArgument, "%s: %d sequences (1 to 65535)", what, B);
  if (table_width <= 0 || table_stride < table_width) return fail(kErrInvalidArgument, "%s: table rows of %d, %d apart", what, table_width, table_stride);
  c->data = static_cast<uint8_t*>(cache->data);
  c->table = table;
  c->table_stride = table_stride;
  c->table_width = table_width;
  c->num_pages = cache->num_pages;
  c->heads = cache->heads;
  c->page_shift = 31 - __builtin_clz(static_cast<unsigned>(ps));
  c->head_bytes = static_cast<long long>(ps / kKvBlockTokens) * kv_block_bytes(cache->bits, cache->head_dim);
  // positions are 32-bit numbers
  if ((static_cast<long long>(table_width) << c->page_shift) > 0x7fffffe0ll)
    return fail(kErrInvalidArgument, "%s: a table row of %d pages of %d positions exceeds 2^31", what, table_width, ps);
  return kOk;
}

template <class F>
int kv_dispatch(const attn_b200_kv_cache* c, F run) {
  auto by_type = [&](auto bits, auto d) {
    return c->dtype == ATTN_B200_KV_BF16 ? run(bits, d, std::true_type{}) : run(bits, d, std::false_type{});
  };
  auto by_dim = [&](auto bits) {
    if (c->head_dim == 64) return by_type(bits, std::integral_constant<int, 64>{});
    if (c->head_dim == 128) return by_type(bits, std::integral_constant<int, 128>{});
    return by_type(bits, std::integral_constant<int, 256>{});
  };
  return c->bits == 4 ? by_dim(std::integral_constant<int, 4>{}) : by_dim(std::integral_constant<int, 8>{});
}

int kv_sms() {
  constexpr int kMaxDevices = 64;
  static int table[kMaxDevices] = {};
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 148;
  if (table[dev] == 0) table[dev] = cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess && n > 0 ? n : 148;
  return table[dev];
}

// Every kernel of the cache is launched as a programmatic dependent: its blocks may start while the kernel in front drains, and they
// wait for its completion before they touch memory.
template <class Kernel, class... Args>
int kv_launch(const char* what, Kernel kernel, dim3 grid, int threads, int smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) return kOk;
  (void)cudaGetLastError();
  return fail(kErrCuda, "%s: launch: %s", what, cudaGetErrorString(e));
}

// Once per device; always the same limit, whatever the batch.
template <class Cfg>
cudaError_t kv_attn_allow_smem() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(&kv_attn_kernel<Cfg>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::smem_bytes(Cfg::ROWS, kKvMaxBatch));
  if (e == cudaSuccess && dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// CTAs of a launch: as many as the GPU holds at once (with the prefix sums of an ordinary batch).
template <class Cfg>
int kv_attn_grid(int rows) {
  static const std::array<int, Cfg::ROWS + 1> per_sm = [] {
    std::array<int, Cfg::ROWS + 1> t{};
    const bool ok = kv_attn_allow_smem<Cfg>() == cudaSuccess;
    for (int r = 1; r <= Cfg::ROWS; ++r) {
      int n = 0;
      if (!ok || cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, &kv_attn_kernel<Cfg>, Cfg::NTHREADS, Cfg::smem_bytes(r, 256)) != cudaSuccess) {
        (void)cudaGetLastError();
        n = 1;
      }
      t[r] = n > 0 ? n : 1;
    }
    return t;
  }();
  return std::min(per_sm[rows < Cfg::ROWS ? rows : Cfg::ROWS] * kv_sms(), kKvMaxRuns);
}

// Heads of few positions are not split, which saves the second kernel: a quarter of a head's units, one after another, then
// take less than the parts' way through memory. With tables of 128 / 256 / 512 / 768 positions, a call split and whole, us:
//   2 x 4 heads, d = 64, 4 bits   5.1  4.4 |  6.2  5.1 |  6.4  6.2 |  6.4  7.3
//   16 x 8 heads, d = 128, 4 bits 6.6  6.1 |  8.1  7.5 |  9.5 10.0 | 11.0 12.7
//   64 x 8 heads, d = 128, 4 bits 11.0 9.6 | 13.3 12.1 | 16.8 17.2 | 20.2 22.1
//   8 x 8 heads, d = 128, 8 bits  5.8  5.4 |  7.4  6.9 |  8.4  9.4 |  8.9 12.0
bool kv_attn_whole(long long positions, int d) { return positions * d <= 512 * 64; }

template <class Cfg>
size_t kv_attn_ws_bytes(int rows, long long positions) {
  if (kv_attn_whole(positions, Cfg::D)) return 0;
  return static_cast<size_t>(2) * kv_attn_grid<Cfg>(rows) * Cfg::ROWS * (Cfg::D + 2) * sizeof(float);
}

template <class Cfg>
int kv_attn_launch(KvAttnParams p, size_t ws_bytes, cudaStream_t stream) {
  p.row_blocks = (p.rows + Cfg::ROWS - 1) / Cfg::ROWS;
  // The kernels count work in 32 bits (and kv_div), for tables as full as they can be: the lengths are on the device. A batch that
  // could hold more goes out in several launches, one after another with the same workspace.
  const long long per_seq = static_cast<long long>(p.cache.heads) * p.row_blocks;
  const long long units = (static_cast<long long>(p.cache.table_width) << p.cache.page_shift) / Cfg::UNIT + 1 + kKvHeadCost<Cfg::UNIT>;
  const long long most = 0x7fffffff / (per_seq * units);
  if (most == 0 || per_seq > 1 << 20)
    return fail(kErrInvalidArgument, "kv_attn: %d heads x %d row blocks with tables of %d pages exceed 2^31 units of work", p.cache.heads,
                p.row_blocks, p.cache.table_width);
  const int grid = kv_attn_grid<Cfg>(p.rows);
  const size_t need = kv_attn_ws_bytes<Cfg>(p.rows, static_cast<long long>(p.cache.table_width) << p.cache.page_shift);
  if (ws_bytes < need || (need > 0 && p.ws == nullptr))
    return fail(kErrInvalidArgument, "kv_attn: %zu bytes of workspace, %zu are needed", p.ws == nullptr ? size_t(0) : ws_bytes, need);
  p.by_grid = make_fast_div(grid);
  p.whole = kv_attn_whole(static_cast<long long>(p.cache.table_width) << p.cache.page_shift, Cfg::D);
  auto kernel = &kv_attn_kernel<Cfg>;
  cudaError_t e = kv_attn_allow_smem<Cfg>();
  if (e != cudaSuccess) return fail(kErrCuda, "kv_attn: cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  const int B = p.B, launches = static_cast<int>((B + most - 1) / most), each = (B + launches - 1) / launches;
  const long long rows = static_cast<long long>(p.cache.heads) * p.rows;  // of a sequence
  for (int b = 0; b < B; b += each) {
    KvAttnParams x = p;
    x.B = std::min(each, B - b);
    x.cache.first = b;
    x.cache.table += static_cast<long long>(b) * p.cache.table_stride;
    x.lengths += b;
    x.q = static_cast<const uint16_t*>(p.q) + b * rows * Cfg::D;
    x.o = static_cast<uint16_t*>(p.o) + b * rows * Cfg::D;
    if (p.lse != nullptr) x.lse += b * rows;
    if (int rc = kv_launch("kv_attn", kernel, dim3(grid, 1, 1), Cfg::NTHREADS, Cfg::smem_bytes(p.rows, x.B), stream, x)) return rc;
    if (p.whole) continue;
    // tasks of a head: a block of its own for each where there are few heads (one may lie in all runs), a warp where there are many
    const long long items = x.B * per_seq;
    const int tasks = std::min(p.rows, Cfg::ROWS) * (Cfg::D / 64);
    const bool few = items * tasks <= 2 * kv_sms();
    if (int rc = kv_launch("kv_attn", &kv_attn_join_kernel<Cfg::D, Cfg::ROWS, Cfg::UNIT, Cfg::BF16>,
                           dim3(static_cast<unsigned>(items), static_cast<unsigned>(few ? tasks : (tasks + 7) / 8), 1), few ? 512 : 256, 0,
                           stream, x, grid))
      return rc;
  }
  return kOk;
}

template <class F>
int kv_attn_dispatch(const attn_b200_kv_cache* cache, int rows, F run) {
  return kv_dispatch(cache, [&](auto bits, auto d, auto bf16) {
    constexpr int BITS = decltype(bits)::value, D = decltype(d)::value;
    constexpr bool BF16 = decltype(bf16)::value;
    // rows per pass over the cache: four, where each lane has half the softmax to do, eight, or 16 where registers allow
    if (rows <= 4) return run(KvAttnConfig<BITS, D, 4, BF16>{});
    if constexpr (D <= 128) {
      if (rows > 8) return run(KvAttnConfig<BITS, D, 16, BF16>{});
    }
    return run(KvAttnConfig<BITS, D, 8, BF16>{});
  });
}

bool kv_attn_sizes_ok(const attn_b200_kv_cache* c, int B, int group, int Lq) {
  return c != nullptr && (c->bits == 4 || c->bits == 8) && (c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256) && B > 0 &&
         B <= kKvMaxBatch && group > 0 && Lq > 0 && Lq <= ATTN_B200_KV_MAX_QUERIES && group <= 0x7fffff / Lq;
}

}  // namespace

extern "C" {

const char* attn_b200_kv_last_error(void) { return error_buffer(); }

int attn_b200_kv_status(int clear) {
  int det = 0, bad = 0;
  const int st = read_device_status(clear, &det);
  if (st != 0) return st;
  if (cudaMemcpyFromSymbol(&bad, g_kv_bad, sizeof(int)) != cudaSuccess)
    return fail(kErrCuda, "cudaMemcpyFromSymbol: %s", cudaGetErrorString(cudaGetLastError())), -1;
  if (bad == 0) return 0;
  if (clear) {
    int zero = 0;
    cudaMemcpyToSymbol(g_kv_bad, &zero, sizeof(int));
    volatile int* m = status_mirror();
    if (m != nullptr) m[3] = 0;
  }
  fail(kErrDevice, "device status: %s", bad == kKvBadPage ? "a page table named a page that does not exist"
                                                          : "a length, start or count was out of range");
  return 2 + bad;
}

int attn_b200_kv_prepare(void) { return status_mirror() == nullptr ? static_cast<int>(kErrCuda) : static_cast<int>(kOk); }

int attn_b200_kv_block_bytes(int bits, int head_dim) {
  if ((bits != 4 && bits != 8) || (head_dim != 64 && head_dim != 128 && head_dim != 256)) return 0;
  return kv_block_bytes(bits, head_dim);
}

int attn_b200_kv_write(const attn_b200_kv_cache* cache, const int* table, int table_stride, int table_width, const int* start,
                       const int* count, const void* k, const long long* k_strides, const void* v, const long long* v_strides, int B,
                       int L, void* stream) {
  KvWriteParams p{};
  if (int rc = kv_view(&p.cache, cache, table, table_stride, table_width, B, "kv_write")) return rc;
  if (k == nullptr || v == nullptr || start == nullptr || k_strides == nullptr || v_strides == nullptr)
    return fail(kErrInvalidArgument, "kv_write: null pointer");
  if (L <= 0 || L > 1 << 30) return fail(kErrInvalidArgument, "kv_write: %d positions", L);
  if (!aligned16(k) || !aligned16(v)) return fail(kErrInvalidArgument, "kv_write: k and v must be 16-byte aligned");
  for (int i = 0; i < 3; ++i) {
    if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0)
      return fail(kErrInvalidArgument, "kv_write: strides of k and v must be multiples of 8 elements");
    p.k_stride[i] = k_strides[i];
    p.v_stride[i] = v_strides[i];
  }
  if (int rc = kv_check_prior("kv_write")) return rc;
  if (int rc = kv_check_device(cache->data, "kv_write")) return rc;
  p.k = k;
  p.v = v;
  p.start = start;
  p.count = count;
  p.B = B;
  p.L = L;
  p.blocks = (L + 2 * kKvBlockTokens - 2) / kKvBlockTokens;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return kv_dispatch(cache, [&](auto bits, auto d, auto bf16) {
    const dim3 grid((p.blocks + 3) / 4, p.cache.heads, B);
    return kv_launch("kv_write", &kv_write_kernel<decltype(bits)::value, decltype(d)::value, decltype(bf16)::value>, grid, 128, 0, st, p);
  });
}

int attn_b200_kv_read(const attn_b200_kv_cache* cache, const int* table, int table_stride, int table_width, const int* start,
                      const int* count, void* k, void* v, int B, int L, void* stream) {
  KvReadParams p{};
  if (int rc = kv_view(&p.cache, cache, table, table_stride, table_width, B, "kv_read")) return rc;
  if (k == nullptr || v == nullptr) return fail(kErrInvalidArgument, "kv_read: null pointer");
  if (L <= 0 || L > 1 << 30) return fail(kErrInvalidArgument, "kv_read: %d positions", L);
  if (!aligned16(k) || !aligned16(v)) return fail(kErrInvalidArgument, "kv_read: k and v must be 16-byte aligned");
  if (int rc = kv_check_prior("kv_read")) return rc;
  if (int rc = kv_check_device(cache->data, "kv_read")) return rc;
  p.k = k;
  p.v = v;
  p.start = start;
  p.count = count;
  p.B = B;
  p.L = L;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return kv_dispatch(cache, [&](auto bits, auto d, auto bf16) {
    const dim3 grid(((L + 2 * kKvBlockTokens - 2) / kKvBlockTokens + 3) / 4, p.cache.heads, B);
    return kv_launch("kv_read", &kv_read_kernel<decltype(bits)::value, decltype(d)::value, decltype(bf16)::value>, grid, 128, 0, st, p);
  });
}

size_t attn_b200_kv_attn_workspace_bytes(const attn_b200_kv_cache* cache, int table_width, int B, int group, int Lq) {
  if (!kv_attn_sizes_ok(cache, B, group, Lq) || table_width <= 0) return 0;
  size_t bytes = 0;
  kv_attn_dispatch(cache, group * Lq, [&](auto cfg) {
    bytes = kv_attn_ws_bytes<decltype(cfg)>(group * Lq, static_cast<long long>(table_width) * cache->page_size);
    return 0;
  });
  return bytes;
}

int attn_b200_kv_attn(const void* q, const attn_b200_kv_cache* cache, const int* table, int table_stride, int table_width,
                      const int* lengths, void* o, float* lse, void* workspace, size_t workspace_bytes, int B, int group, int Lq,
                      float scale, int causal, void* stream) {
  KvAttnParams p{};
  if (int rc = kv_view(&p.cache, cache, table, table_stride, table_width, B, "kv_attn")) return rc;
  if (q == nullptr || o == nullptr || lengths == nullptr) return fail(kErrInvalidArgument, "kv_attn: null pointer");
  if (!kv_attn_sizes_ok(cache, B, group, Lq))
    return fail(kErrInvalidArgument, "kv_attn: %d sequences (at most %d), %d query heads per head of the cache, %d queries (at most %d)", B,
                kKvMaxBatch, group, Lq, ATTN_B200_KV_MAX_QUERIES);
  if (!(scale > 0.f) || !isfinite(scale)) return fail(kErrInvalidArgument, "kv_attn: scale must be positive and finite");
  if (!aligned16(q) || !aligned16(o) || !aligned16(workspace)) return fail(kErrInvalidArgument, "kv_attn: q, o and the workspace must be 16-byte aligned");
  if (int rc = kv_check_prior("kv_attn")) return rc;
  if (int rc = kv_check_device(q, "kv_attn")) return rc;
  p.lengths = lengths;
  p.q = q;
  p.o = o;
  p.lse = lse;
  p.ws = static_cast<float*>(workspace);
  p.B = B;
  p.Lq = Lq;
  p.rows = group * Lq;
  p.causal = causal != 0;
  p.scale_log2 = scale * 1.4426950408889634f;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return kv_attn_dispatch(cache, p.rows, [&](auto cfg) { return kv_attn_launch<decltype(cfg)>(p, workspace_bytes, st); });
}

}  // extern "C"
