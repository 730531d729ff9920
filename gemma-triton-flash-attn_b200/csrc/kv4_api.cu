// Host side of the paged 4-bit KV cache's C ABI (include/gqa_fa_b200.h):
// argument validation, variant choice and launches of the kernels in
// kv4_cache_kernels.cuh and kv4_attn_kernel.cuh.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstring>

#include "../../include/gqa_fa_b200.h"
#include "api_shared.cuh"
#include "kv4_attn_kernel.cuh"
#include "kv4_cache_kernels.cuh"

namespace gqafa {
namespace {

int log2_of(int v) {
  int s = 0;
  while ((1 << s) < v) ++s;
  return s;
}

int check_cache(int heads_kv, int head_dim, int page_size, int dtype) {
  if (heads_kv <= 0) return fail(GQAFA_ERR_INVALID, "heads_kv must be positive, got %d", heads_kv);
  if (dtype != GQAFA_DTYPE_FP16 && dtype != GQAFA_DTYPE_BF16)
    return fail(GQAFA_ERR_INVALID, "dtype code %d is not fp16 (0) or bf16 (1)", dtype);
  if (head_dim != 64 && head_dim != 128 && head_dim != 256 && head_dim != 512)
    return fail(GQAFA_ERR_UNSUPPORTED, "head_dim %d is not implemented on sm_100a (supported: 64, 128, 256, 512)",
                head_dim);
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
    return fail(GQAFA_ERR_UNSUPPORTED, "page_size %d is not implemented (supported: 16, 32, 64, 128, 256)", page_size);
  return GQAFA_OK;
}

int check_pages(const void* pages, long long num_pages, int page_size) {
  if (pages == nullptr) return fail(GQAFA_ERR_INVALID, "pages: null pointer");
  if (reinterpret_cast<uintptr_t>(pages) % 16 != 0)
    return fail(GQAFA_ERR_INVALID, "pages: data pointer must be 16-byte aligned");
  if (num_pages <= 0 || num_pages * page_size > INT_MAX)
    return fail(GQAFA_ERR_INVALID, "num_pages %lld out of range (num_pages * page_size must be in 1..2^31-1)",
                num_pages);
  return GQAFA_OK;
}

int check_ints(const char* name, const void* p) {
  if (p == nullptr) return fail(GQAFA_ERR_INVALID, "%s: null pointer", name);
  if (reinterpret_cast<uintptr_t>(p) % 4 != 0) return fail(GQAFA_ERR_INVALID, "%s must be 4-byte aligned", name);
  return GQAFA_OK;
}

int check_table(const void* table, long long stride, int cols, int page_size) {
  int rc = check_ints("block_table", table);
  if (rc) return rc;
  if (cols <= 0 || static_cast<long long>(cols) * page_size > INT_MAX - 4096)
    return fail(GQAFA_ERR_INVALID, "block_table: %d columns out of range", cols);
  if (stride < 0) return fail(GQAFA_ERR_INVALID, "block_table: negative row stride");
  return GQAFA_OK;
}

// A [B, H, N, D] tensor with 16-byte rows; strides of size-1 dims are ignored.
int check_rows(const char* name, const void* ptr, const long long* st, int B, int H, int N, long long* out) {
  if (ptr == nullptr) return fail(GQAFA_ERR_INVALID, "%s: null pointer", name);
  if (st == nullptr) return fail(GQAFA_ERR_INVALID, "%s: null strides", name);
  if (reinterpret_cast<uintptr_t>(ptr) % 16 != 0)
    return fail(GQAFA_ERR_INVALID, "%s: data pointer must be 16-byte aligned", name);
  if (st[3] != 1) return fail(GQAFA_ERR_INVALID, "%s: last (head_dim) stride must be 1, got %lld", name, st[3]);
  const int size[3] = {B, H, N};
  for (int i = 0; i < 3; ++i) {
    out[i] = size[i] == 1 ? 0 : st[i];
    if ((size[i] > 1 && out[i] <= 0) || out[i] % 8 != 0)
      return fail(GQAFA_ERR_INVALID,
                  "%s: strides must be positive multiples of 8 elements (16 bytes), got (%lld, %lld, %lld, %lld)", name,
                  st[0], st[1], st[2], st[3]);
  }
  return GQAFA_OK;
}

int sm_count() {
  static std::atomic<int> counts[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  int n = counts[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    counts[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

int launch_status(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(GQAFA_ERR_CUDA, "%s launch: %s", what, cudaGetErrorString(e));
  return GQAFA_OK;
}

struct AttendShape {
  int B, Hq, Hkv, N, D, G;
  int row_tiles, ctas, join_blocks;
  bool wide;  // tiles of more blocks (kv4_warp_blocks)
  long long units;
  long long part_ctas;  // room for the parts of this many CTAs: no call within the same lengths has more
  // Dense path (0 requests: not taken): rows of K and V, requests at a time.
  int dense_rows, dense_batch;
};

// Bytes that the dense path holds at a time, 2 GiB of K and V in 16 bits and the
// bits that go with them (a 2048th); it goes over the batch in groups of requests
// beyond that (one at least).
constexpr long long kDenseBytes = (2LL << 30) + (1LL << 20);

// Dense path: K and V [batch][Hkv][rows][D] 16-bit, then the bits of groups that
// are not finite [batch][Hkv][kv4_nan_pitch].
long long dense_bytes(int Hkv, long long rows, int D) {  // of one request
  return Hkv * (4 * rows * D + 2 * kv4_nan_pitch(rows, D));
}

// Many query rows per KV head are bound by the products, not by the cache: then
// the keys and values are written out in 16 bits once (exactly) and the tcgen05
// forward of dense caches runs over them, with the lengths of each request. Its
// CTAs (pairs at head_dim 512) take 128 tokens of one query head over all keys;
// the MMAs above take 8 rows of all heads of a group and split the keys. Both
// times grow with the keys: per key a unit of 8 rows costs the whole GPU 82, 46,
// 29, 21 ps at head_dim 512, 256, 128, 64, a wave of 128-row tiles 20.6, 18.7,
// 16.4, 18.0 ns; a group of `batch` requests is one launch, of one wave at least.
// Measured on both sides of the rule, 2 requests of 7K keys, 32/4
// heads, head_dim 512: 24 tokens 141 us in units and 171 us dense, 48 tokens 240
// and 172 us; 8 requests, 16/4 heads, head_dim 64: 48 tokens 120 and 147 us, 100
// tokens 231 and 148 us; 64 requests of 4000 keys in a table for 131072, one a
// group, 8/8 heads, head_dim 512: 64 tokens 1980 us and 12.9 ms (there the empty part
// of the table costs the dense way more than the rule says: 256 tokens are dense,
// 12.9 ms, where units would take about 8).
bool dense_path(int B, int batch, int Hq, int Hkv, int N, int D, int sms) {
  const long long units = static_cast<long long>(B) * Hkv * ((static_cast<long long>(Hq / Hkv) * N + 7) / 8);
  const long long tiles = static_cast<long long>(batch) * Hq * ((N + 127) / 128) * (D == 512 ? 2 : 1);
  const long long waves = static_cast<long long>((B + batch - 1) / batch) * ((tiles + sms - 1) / sms);
  const int ratio = D == 512 ? 250 : (D == 256 ? 400 : (D == 128 ? 560 : 860));
  return units > ratio * waves;
}

// Units of 8 query rows, and the CTAs of the launch: two per SM, fewer where there
// are fewer tiles. max_len 0: not known (a size call before the table is).
AttendShape attend_shape(int B, int Hq, int Hkv, int N, int D, int max_len, int window, int sms) {
  AttendShape s{};
  s.B = B;
  s.Hq = Hq;
  s.Hkv = Hkv;
  s.N = N;
  s.D = D;
  s.G = Hq / Hkv;
  const long long rows = static_cast<long long>(s.G) * N;
  s.row_tiles = static_cast<int>((rows + 7) / 8);
  long long span = max_len;
  if (window > 0) span = std::min<long long>(span, static_cast<long long>(window) + 8 / s.G + 1);
  s.units = static_cast<long long>(B) * s.row_tiles * Hkv;
  auto tiles_of = [&](bool wide, long long keys) {
    const int tile_tokens = 8 * 16 * kv4_warp_blocks(D, wide);
    return s.units * ((keys + 15 + tile_tokens - 1) / tile_tokens + 1);
  };
  auto tiles = [&](bool wide) { return tiles_of(wide, span); };
  // Short tiles and no window give the most CTAs, and more keys never fewer.
  s.part_ctas = max_len > 0 ? std::min<long long>(2LL * sms, tiles_of(false, max_len)) : 2LL * sms;
  // Short tiles where each gets a CTA of its own: one token over a window of 512,
  // 16/8 heads, 4 requests at head_dim 256 12.6 us against 13.7, at 128 11.6 and
  // 12.8, at 64 10.4 and 11.4. Else long ones, fewer barriers: 8 requests at 256
  // 15.2 us against 16.8, at 128 13.7 and 14.8; 16 requests of 8K to 16K keys, 32/4
  // heads, at 256 65.3 and 69.7, at 128 43.5 and 49.6, at 64 32.8 and 34.3. At 512
  // one block a warp is the best of both: with two, 114.8 us against 105.8. (All
  // before the query's third byte, which added about 2 %.) Few units lose CTAs at
  // the change, but no time: one request of 32/4 heads at 128, 9216 keys in 296 CTAs
  // 12.7 us, 9472 in 80 12.3; 16/2 heads, 18800 keys 13.5, 19000 12.2; at 256 9216
  // keys 13.7, 9472 14.2.
  s.wide = D != 512 && tiles(false) > 2LL * sms;
  s.ctas = static_cast<int>(std::min<long long>(2LL * sms, tiles(s.wide)));
  long long held = max_len;
  if (window > 0) held = std::min<long long>(held, static_cast<long long>(window) + N + 15);
  const long long rows16 = (held + 15) / 16 * 16;
  if (max_len > 0) {
    const int batch =
        static_cast<int>(std::min<long long>(B, std::max<long long>(1, kDenseBytes / dense_bytes(Hkv, rows16, D))));
    if (dense_path(B, batch, Hq, Hkv, N, D, sms)) {
      s.dense_rows = static_cast<int>(rows16);
      s.dense_batch = batch;
    }
  }
  // the join: at most two CTAs per SM, all of them where few units are cut into many parts
  s.join_blocks = 1;
  while (s.join_blocks < 8 * D / 128 && s.join_blocks * s.units <= sms) s.join_blocks *= 2;
  return s;
}

// Parts [2 * ctas][8][D] fp32, their maxima and sums [2 * ctas][8].
long long part_bytes(const AttendShape& s, long long ctas) { return 2 * ctas * 8 * (s.D * 4LL + 8) + 256; }
// Both ways' room, and never less for more keys: a caller's bound may lie above
// the table's capacity, which the launch then takes for it.
long long attend_workspace(const AttendShape& s) {
  long long need = part_bytes(s, s.part_ctas);
  if (s.dense_batch) {
    const long long one = dense_bytes(s.Hkv, s.dense_rows, s.D);
    need = std::max(need, s.dense_batch < s.B ? std::max(one, kDenseBytes) : s.B * one);
  }
  return need;
}

template <class C>
int launch_attend(Kv4Params p, cudaStream_t st) {
  static std::atomic<unsigned long long> attr_done_mask{0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return fail(GQAFA_ERR_CUDA, "cudaGetDevice failed");
  const unsigned long long bit = 1ULL << (dev & 63);
  if (!(attr_done_mask.load() & bit)) {
    const cudaError_t e =
        cudaFuncSetAttribute(kv4_attn_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
    if (e != cudaSuccess) return fail(GQAFA_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    attr_done_mask.fetch_or(bit);
  }
  const long long blocks = static_cast<long long>(p.B) * p.row_tiles * p.Hkv * p.join_blocks;
  if (blocks > INT_MAX) return fail(GQAFA_ERR_INVALID, "grid size %lld out of range", blocks);
  kv4_attn_kernel<C><<<p.ctas, C::THREADS, C::SMEM_BYTES, st>>>(p);
  const int rc = launch_status("4-bit cache attention");
  if (rc) return rc;
  // The join starts while the attention's last CTAs run (programmatic
  // dependent launch): it reads the lengths and then waits for them.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(512);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_combine_kernel<C>, static_cast<const Kv4Params>(p));
  if (e != cudaSuccess) return fail(GQAFA_ERR_CUDA, "4-bit cache join launch: %s", cudaGetErrorString(e));
  return GQAFA_OK;
}

template <bool BF16>
int attend_dim(int D, bool wide, const Kv4Params& p, cudaStream_t st) {
  switch (D) {
    case 64: return wide ? launch_attend<Kv4Cfg<64, BF16, true>>(p, st) : launch_attend<Kv4Cfg<64, BF16, false>>(p, st);
    case 128:
      return wide ? launch_attend<Kv4Cfg<128, BF16, true>>(p, st) : launch_attend<Kv4Cfg<128, BF16, false>>(p, st);
    case 256:
      return wide ? launch_attend<Kv4Cfg<256, BF16, true>>(p, st) : launch_attend<Kv4Cfg<256, BF16, false>>(p, st);
    default: return launch_attend<Kv4Cfg<512, BF16, false>>(p, st);
  }
}

// UNITS: (block, group) pairs a warp reads.
template <bool RAGGED, int UNITS>
int launch_read(Kv4ReadParams p, int head_dim, bool bf16, cudaStream_t st) {
  const int NG = head_dim / KV4_GROUP;
  // n tokens from any start touch at most (n + 15 + 15) / 16 blocks
  const long long items = ((p.n + 30LL) / 16) * NG;
  const long long xblocks = (items + 8 * UNITS - 1) / (8 * UNITS), blocks = xblocks * p.B * p.Hkv;
  if (blocks > INT_MAX) return fail(GQAFA_ERR_INVALID, "grid size %lld out of range", blocks);
  p.xblocks = static_cast<int>(xblocks);
  const dim3 grid(static_cast<unsigned>(blocks), 2);
#define GQAFA_LAUNCH(DIM)                                                \
  if (bf16)                                                              \
    kv4_read_kernel<DIM, true, RAGGED, UNITS><<<grid, 256, 0, st>>>(p);  \
  else                                                                   \
    kv4_read_kernel<DIM, false, RAGGED, UNITS><<<grid, 256, 0, st>>>(p); \
  break
  switch (head_dim) {
    case 64: GQAFA_LAUNCH(64);
    case 128: GQAFA_LAUNCH(128);
    case 256: GQAFA_LAUNCH(256);
    default: GQAFA_LAUNCH(512);
  }
#undef GQAFA_LAUNCH
  return launch_status("read");
}

int launch_spread(const Kv4SpreadParams& p, int head_dim, int batch, cudaStream_t st) {
  const unsigned blocks = static_cast<unsigned>(batch) * p.Hkv;
  switch (head_dim) {
    case 64: kv4_spread_nan_kernel<64><<<blocks, 512, 0, st>>>(p); break;
    case 128: kv4_spread_nan_kernel<128><<<blocks, 512, 0, st>>>(p); break;
    case 256: kv4_spread_nan_kernel<256><<<blocks, 512, 0, st>>>(p); break;
    default: kv4_spread_nan_kernel<512><<<blocks, 512, 0, st>>>(p);
  }
  return launch_status("4-bit cache NaN");
}

int check_attend(int batch, int heads_q, int heads_kv, int seqlen_q, int head_dim, int page_size, int dtype) {
  int rc = check_cache(heads_kv, head_dim, page_size, dtype);
  if (rc) return rc;
  if (batch <= 0 || heads_q <= 0 || seqlen_q <= 0)
    return fail(GQAFA_ERR_INVALID, "sizes must be positive (B=%d H_Q=%d N=%d)", batch, heads_q, seqlen_q);
  if (heads_q % heads_kv != 0)
    return fail(GQAFA_ERR_INVALID, "H_Q (%d) must be a multiple of H_KV (%d)", heads_q, heads_kv);
  if (static_cast<long long>(batch) * heads_q > INT_MAX ||
      static_cast<long long>(batch) * heads_q * seqlen_q > INT_MAX / 2)
    return fail(GQAFA_ERR_INVALID, "B * H_Q * N out of range");
  return GQAFA_OK;
}

}  // namespace
}  // namespace gqafa

using namespace gqafa;

extern "C" long long gqafa_kv4_page_bytes(int heads_kv, int head_dim, int page_size) {
  clear_error();
  if (check_cache(heads_kv, head_dim, page_size, GQAFA_DTYPE_BF16)) return -1;
  return 2LL * heads_kv * (page_size / KV4_TOKENS) * kv4_block_bytes(head_dim);
}

extern "C" int gqafa_kv4_plan(const int* kv_lens, const int* new_lens, const int* block_table, long long table_stride,
                              int* free_pages, const int* free_state, int batch, int cols, int num_free,
                              int page_size, int max_new, int* out_block_table, int* out_kv_lens, int* out_new_lens,
                              int* out_slot_map, int* out_positions, int* out_accepted, int* out_free_state,
                              void* stream) {
  clear_error();
  int rc;
  if ((rc = check_cache(1, 64, page_size, GQAFA_DTYPE_BF16))) return rc;
  if (batch <= 0 || max_new <= 0)
    return fail(GQAFA_ERR_INVALID, "sizes must be positive (B=%d max_new=%d)", batch, max_new);
  if ((rc = check_table(block_table, table_stride, cols, page_size))) return rc;
  if (static_cast<long long>(batch) * cols > INT_MAX)
    return fail(GQAFA_ERR_INVALID, "block_table: %d rows of %d columns out of range", batch, cols);
  if (num_free <= 0 || static_cast<long long>(num_free) * page_size > INT_MAX)
    return fail(GQAFA_ERR_INVALID, "free_pages: %d entries out of range (entries * page_size must be in 1..2^31-1)",
                num_free);
  const void* ints[] = {kv_lens, new_lens, free_pages, free_state, out_block_table, out_kv_lens,
                        out_new_lens, out_slot_map, out_positions, out_accepted, out_free_state};
  const char* names[] = {"kv_lens", "new_lens", "free_pages", "free_state", "out_block_table", "out_kv_lens",
                         "out_new_lens", "out_slot_map", "out_positions", "out_accepted", "out_free_state"};
  for (int i = 0; i < 11; ++i)
    if ((rc = check_ints(names[i], ints[i]))) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = bind_device(st))) return rc;
  Kv4PlanParams p{};
  p.kv_lens = kv_lens;
  p.new_lens = new_lens;
  p.table = block_table;
  p.table_stride = table_stride;
  p.free_pages = free_pages;
  p.free_state = free_state;
  p.B = batch;
  p.cols = cols;
  p.F = num_free;
  p.page = page_size;
  p.page_shift = log2_of(page_size);
  p.max_new = max_new;
  p.out_table = out_block_table;
  p.out_kv_lens = out_kv_lens;
  p.out_new_lens = out_new_lens;
  p.out_slots = out_slot_map;
  p.out_positions = out_positions;
  p.out_accepted = out_accepted;
  p.out_state = out_free_state;
  kv4_plan_kernel<<<batch, 256, 0, st>>>(p);
  return launch_status("plan");
}

extern "C" int gqafa_kv4_append(const void* k, const long long* k_strides, const void* v, const long long* v_strides,
                                const int* slot_map, long long slot_stride, void* pages, long long num_pages,
                                int batch, int heads_kv, int seqlen, int head_dim, int page_size, int dtype,
                                void* stream) {
  clear_error();
  int rc;
  if ((rc = check_cache(heads_kv, head_dim, page_size, dtype))) return rc;
  if (batch <= 0 || seqlen <= 0) return fail(GQAFA_ERR_INVALID, "sizes must be positive (B=%d N=%d)", batch, seqlen);
  const long long units = static_cast<long long>(seqlen) * (head_dim / KV4_GROUP);  // (token, group) pairs
  // the last CTA's pairs run up to 127 past the last one, in 32 bits
  if (heads_kv > 65535 || batch > 65535 || units > INT_MAX - 127)
    return fail(GQAFA_ERR_INVALID, "B (%d), heads_kv (%d) and tokens (%d) out of range (65535, 65535, and 2^31 - 128 "
                "groups of 64 values)", batch, heads_kv, seqlen);
  if ((rc = check_pages(pages, num_pages, page_size))) return rc;
  if ((rc = check_ints("slot_map", slot_map))) return rc;
  if (slot_stride < 0) return fail(GQAFA_ERR_INVALID, "slot_map: negative row stride");
  Kv4AppendParams p{};
  long long s[3];
  const void* src[2] = {k, v};
  const long long* strides[2] = {k_strides, v_strides};
  for (int i = 0; i < 2; ++i) {
    if ((rc = check_rows(i ? "v" : "k", src[i], strides[i], batch, heads_kv, seqlen, s))) return rc;
    p.x[i] = static_cast<const uint16_t*>(src[i]);
    p.sb[i] = s[0];
    p.sh[i] = s[1];
    p.sn[i] = s[2];
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = bind_device(st))) return rc;
  p.slots = slot_map;
  p.slots_stride = slot_stride;
  p.pages = static_cast<uint8_t*>(pages);
  p.B = batch;
  p.N = seqlen;
  p.Hkv = heads_kv;
  p.page_shift = log2_of(page_size);
  p.num_slots = static_cast<int>(num_pages * page_size);
  p.status = status_ptr();
  if (!p.status) return fail(GQAFA_ERR_CUDA, "cannot resolve the device status word");
  const int sms = sm_count();
  if (sms <= 0) return fail(GQAFA_ERR_CUDA, "cannot read the device's multiprocessor count");
  // Few groups: four lanes each, the shorter way through (at head_dim 256, 8 heads:
  // 128 tokens 2.2 us against 2.9, 1024 tokens 3.9 and 4.3). Many: two, fewer
  // instructions a value (4096 tokens 10.1 us against 11.0).
  const bool few = units * heads_kv * batch <= 384LL * sms;
  const int pairs = few ? 64 : 128;  // of a CTA
  const dim3 grid(static_cast<unsigned>((units + pairs - 1) / pairs), heads_kv, batch);
  const bool bf16 = dtype == GQAFA_DTYPE_BF16;
#define GQAFA_LAUNCH(DIM)                                                                      \
  if (few) {                                                                                   \
    bf16 ? kv4_append_kernel<DIM, true, 4><<<grid, 256, 0, st>>>(p)                            \
         : kv4_append_kernel<DIM, false, 4><<<grid, 256, 0, st>>>(p);                          \
  } else {                                                                                     \
    bf16 ? kv4_append_kernel<DIM, true, 2><<<grid, 256, 0, st>>>(p)                            \
         : kv4_append_kernel<DIM, false, 2><<<grid, 256, 0, st>>>(p);                          \
  }                                                                                            \
  break
  switch (head_dim) {
    case 64: GQAFA_LAUNCH(64);
    case 128: GQAFA_LAUNCH(128);
    case 256: GQAFA_LAUNCH(256);
    default: GQAFA_LAUNCH(512);
  }
#undef GQAFA_LAUNCH
  return launch_status("append");
}

extern "C" int gqafa_kv4_read(const void* pages, long long num_pages, const int* block_table, long long table_stride,
                              int cols, const int* kv_lens, const int* starts, void* k, void* v, int batch,
                              int heads_kv, int seqlen, int head_dim, int page_size, int dtype, void* stream) {
  clear_error();
  int rc;
  if ((rc = check_cache(heads_kv, head_dim, page_size, dtype))) return rc;
  if (batch <= 0 || seqlen <= 0) return fail(GQAFA_ERR_INVALID, "sizes must be positive (B=%d n=%d)", batch, seqlen);
  if (static_cast<long long>(batch) * heads_kv > INT_MAX ||
      static_cast<long long>(batch) * heads_kv * seqlen > (1LL << 40))
    return fail(GQAFA_ERR_INVALID, "B * H_KV * n out of range");
  if ((rc = check_pages(pages, num_pages, page_size))) return rc;
  if ((rc = check_table(block_table, table_stride, cols, page_size))) return rc;
  if ((rc = check_ints("kv_lens", kv_lens))) return rc;
  if (starts && (rc = check_ints("starts", starts))) return rc;
  void* out[2] = {k, v};
  for (int i = 0; i < 2; ++i)
    if (out[i] == nullptr || reinterpret_cast<uintptr_t>(out[i]) % 32 != 0)
      return fail(GQAFA_ERR_INVALID, "outputs must be 32-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = bind_device(st))) return rc;
  Kv4ReadParams p{};
  p.pages = static_cast<const uint8_t*>(pages);
  p.table = block_table;
  p.table_stride = table_stride;
  p.kv_lens = kv_lens;
  p.starts = starts;
  p.out[0] = static_cast<uint16_t*>(k);
  p.out[1] = static_cast<uint16_t*>(v);
  p.B = batch;
  p.Hkv = heads_kv;
  p.n = seqlen;
  p.cols = cols;
  p.page_shift = log2_of(page_size);
  p.num_pages = static_cast<int>(num_pages);
  p.status = status_ptr();
  if (!p.status) return fail(GQAFA_ERR_CUDA, "cannot resolve the device status word");
  // Few values: one group a warp, whose code is a quarter as long and comes in
  // sooner (512 tokens, 4 heads, head_dim 512: 3.6 us against 4.6; one token of 64
  // requests: 4.8 and 5.9). Many: more loads in flight per warp (1024 tokens: 5.0
  // us against 5.3, 2048: 7.0 and 8.2).
  const int sms = sm_count();
  if (sms <= 0) return fail(GQAFA_ERR_CUDA, "cannot read the device's multiprocessor count");
  const long long groups = 2LL * batch * heads_kv * seqlen * (head_dim / KV4_GROUP);  // of tokens
  const bool bf16 = dtype == GQAFA_DTYPE_BF16;
  return groups <= 256LL * sms ? launch_read<false, 1>(p, head_dim, bf16, st)
                              : launch_read<false, KV4_READ_UNITS>(p, head_dim, bf16, st);
}

extern "C" long long gqafa_kv4_attend_workspace_size(int batch, int heads_q, int heads_kv, int seqlen_q, int head_dim,
                                                     int max_kv_len, int window) {
  clear_error();
  if (check_attend(batch, heads_q, heads_kv, seqlen_q, head_dim, 16, GQAFA_DTYPE_BF16)) return -1;
  if (max_kv_len < 0 || window < 0) {
    fail(GQAFA_ERR_INVALID, "max_kv_len and window must be >= 0");
    return -1;
  }
  const int sms = sm_count();
  if (sms <= 0) {
    fail(GQAFA_ERR_CUDA, "cannot read the device's multiprocessor count");
    return -1;
  }
  return attend_workspace(attend_shape(batch, heads_q, heads_kv, seqlen_q, head_dim, max_kv_len, window, sms));
}

extern "C" int gqafa_kv4_attend(const void* q, const long long* q_strides, const void* pages, long long num_pages,
                                const int* block_table, long long table_stride, int cols, const int* kv_lens,
                                const int* q_lens, void* o, const long long* o_strides, float* lse, int batch,
                                int heads_q, int heads_kv, int seqlen_q, int head_dim, int page_size, int max_kv_len,
                                float softmax_scale, int causal, int window, int dtype, void* workspace,
                                long long workspace_bytes, void* stream) {
  clear_error();
  int rc;
  if ((rc = check_attend(batch, heads_q, heads_kv, seqlen_q, head_dim, page_size, dtype))) return rc;
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale))
    return fail(GQAFA_ERR_INVALID, "softmax_scale must be positive and finite");
  if (window < 0) return fail(GQAFA_ERR_INVALID, "window must be >= 0");
  if ((rc = check_pages(pages, num_pages, page_size))) return rc;
  if ((rc = check_table(block_table, table_stride, cols, page_size))) return rc;
  if ((rc = check_ints("kv_lens", kv_lens))) return rc;
  if (q_lens && (rc = check_ints("q_lens", q_lens))) return rc;
  if (lse && reinterpret_cast<uintptr_t>(lse) % 4 != 0) return fail(GQAFA_ERR_INVALID, "lse must be 4-byte aligned");
  long long qs[3], os[3];
  if ((rc = check_rows("q", q, q_strides, batch, heads_q, seqlen_q, qs))) return rc;
  if ((rc = check_rows("o", o, o_strides, batch, heads_q, seqlen_q, os))) return rc;
  const long long capacity = static_cast<long long>(cols) * page_size;
  if (max_kv_len < 0) return fail(GQAFA_ERR_INVALID, "max_kv_len must be >= 0");
  if (max_kv_len == 0 || max_kv_len > capacity) max_kv_len = static_cast<int>(capacity);
  const int win = causal && window < capacity ? window : 0;  // a window over all keys cuts none
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if ((rc = bind_device(st))) return rc;
  const int sms = sm_count();
  if (sms <= 0) return fail(GQAFA_ERR_CUDA, "cannot read the device's multiprocessor count");
  AttendShape s = attend_shape(batch, heads_q, heads_kv, seqlen_q, head_dim, max_kv_len, win, sms);
  // A workspace that was sized for other arguments (max_kv_len 0, a window that a
  // call without causal does not use) may hold fewer requests at a time, or none:
  // then the units take the call, and also where groups so small do not pay.
  const long long one = dense_bytes(heads_kv, s.dense_rows, head_dim);
  if (s.dense_batch && workspace_bytes / one < s.dense_batch) {
    s.dense_batch = static_cast<int>(std::max<long long>(0, workspace_bytes / one));
    if (s.dense_batch && workspace_bytes >= part_bytes(s, s.ctas) &&
        !dense_path(batch, s.dense_batch, heads_q, heads_kv, seqlen_q, head_dim, sms))
      s.dense_batch = 0;
  }
  if (!s.dense_batch && s.units * (capacity / 64 + 2) > INT_MAX)
    return fail(GQAFA_ERR_INVALID, "B * H_Q * N times the block table's capacity out of range");
  const long long need = s.dense_batch ? s.dense_batch * one : part_bytes(s, s.ctas);
  if (workspace == nullptr || workspace_bytes < need)
    return fail(GQAFA_ERR_INVALID, "workspace of %lld bytes needed, got %lld", need, workspace_bytes);
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return fail(GQAFA_ERR_INVALID, "workspace must be 256-byte aligned");
  if (s.dense_batch) {
    Kv4ReadParams rd{};
    rd.pages = static_cast<const uint8_t*>(pages);
    rd.Hkv = heads_kv;
    rd.n = s.dense_rows;
    rd.cols = cols;
    rd.table_stride = table_stride;
    rd.page_shift = log2_of(page_size);
    rd.num_pages = static_cast<int>(num_pages);
    rd.q_rows = seqlen_q;
    rd.window = win;
    rd.status = status_ptr();
    if (!rd.status) return fail(GQAFA_ERR_CUDA, "cannot resolve the device status word");
    const bool bf16 = dtype == GQAFA_DTYPE_BF16;
    for (int b = 0; b < batch; b += s.dense_batch) {
      const int nb = std::min(s.dense_batch, batch - b);
      uint16_t* k = static_cast<uint16_t*>(workspace);
      uint16_t* v = k + static_cast<long long>(nb) * heads_kv * s.dense_rows * head_dim;
      rd.B = nb;
      rd.table = block_table + b * table_stride;
      rd.kv_lens = kv_lens + b;
      rd.q_lens = q_lens ? q_lens + b : nullptr;
      rd.out[0] = k;
      rd.out[1] = v;
      if ((rc = launch_read<true, KV4_READ_UNITS>(rd, head_dim, bf16, st))) return rc;
      RaggedForward f{};
      f.q = static_cast<const uint16_t*>(q) + b * qs[0];
      f.q_strides = q_strides;
      f.k = k;
      f.v = v;
      f.o = static_cast<uint16_t*>(o) + b * os[0];
      f.o_strides = o_strides;
      f.lse = lse ? lse + static_cast<long long>(b) * heads_q * seqlen_q : nullptr;
      f.kv_lens = rd.kv_lens;
      f.q_lens = rd.q_lens;
      f.B = nb;
      f.Hq = heads_q;
      f.Hkv = heads_kv;
      f.N = seqlen_q;
      f.Nk = s.dense_rows;
      f.D = head_dim;
      f.kv_cap = static_cast<int>(capacity);
      f.causal = causal ? 1 : 0;
      f.window = win;
      f.scale = softmax_scale;
      f.bf16 = bf16;
      if ((rc = ragged_forward(f, st))) return rc;
      Kv4SpreadParams sp{};
      sp.nans = v + static_cast<long long>(nb) * heads_kv * s.dense_rows * head_dim;
      sp.o = static_cast<uint16_t*>(f.o);
      sp.o_sb = os[0];
      sp.o_sh = os[1];
      sp.o_sn = os[2];
      sp.kv_lens = rd.kv_lens;
      sp.q_lens = rd.q_lens;
      sp.Hkv = heads_kv;
      sp.G = s.G;
      sp.N = seqlen_q;
      sp.n = s.dense_rows;
      sp.capacity = f.kv_cap;
      sp.causal = f.causal;
      sp.window = win;
      if ((rc = launch_spread(sp, head_dim, nb, st))) return rc;
    }
    return GQAFA_OK;
  }
  Kv4Params p{};
  p.tops = kv4_tops(dtype == GQAFA_DTYPE_BF16);
  p.q = static_cast<const uint16_t*>(q);
  p.q_sb = qs[0];
  p.q_sh = qs[1];
  p.q_sn = qs[2];
  p.o = static_cast<uint16_t*>(o);
  p.o_sb = os[0];
  p.o_sh = os[1];
  p.o_sn = os[2];
  p.lse = lse;
  p.pages = static_cast<const uint8_t*>(pages);
  p.table = block_table;
  p.table_stride = table_stride;
  p.kv_lens = kv_lens;
  p.q_lens = q_lens;
  p.B = batch;
  p.Hq = heads_q;
  p.Hkv = heads_kv;
  p.G = s.G;
  p.N = seqlen_q;
  p.cols = cols;
  p.page_shift = log2_of(page_size);
  p.num_pages = static_cast<int>(num_pages);
  p.causal = causal ? 1 : 0;
  p.window = win;
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  p.row_tiles = s.row_tiles;
  p.ctas = s.ctas;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + 2LL * s.ctas * 8 * s.D);
  p.join_blocks = s.join_blocks;
  p.status = status_ptr();
  if (!p.status) return fail(GQAFA_ERR_CUDA, "cannot resolve the device status word");
  p.wait_limit = wait_limit_setting();
  p.no_loads = no_loads_setting();
  return dtype == GQAFA_DTYPE_BF16 ? attend_dim<true>(head_dim, s.wide, p, st)
                                   : attend_dim<false>(head_dim, s.wide, p, st);
}
