// The paged 4-bit KV cache's own kernels: the plan of a step (block tables,
// slots and positions from the requests' lengths), the quantised write of new
// tokens and the read back of cached ones. Formats: kv4_layout.cuh.
#pragma once
#include "attn_kernel.cuh"
#include "kv4_layout.cuh"

namespace gqafa {

// ------------------------------------------------------------------ plan
struct Kv4PlanParams {
  const int* kv_lens;   // [B] tokens already cached
  const int* new_lens;  // [B] tokens of this step; -1: the request is finished
  const int* table;     // [B][cols]
  long long table_stride;
  int* free_pages;        // ring of F page ids
  const int* free_state;  // {head, count}
  int B, cols, F, page, page_shift, max_new;
  int* out_table;  // [B][cols]
  int* out_kv_lens;
  int* out_new_lens;
  int* out_slots;      // [B][max_new]
  int* out_positions;  // [B][max_new]
  int* out_accepted;   // [B]
  int* out_state;      // {head, count}
};

struct Kv4Request {
  int len, add, used, need, back;
  bool gone, fits;
};

__device__ __forceinline__ Kv4Request kv4_request(const Kv4PlanParams& p, int b) {
  Kv4Request r;
  const int capacity = p.cols << p.page_shift;
  r.len = min(max(p.kv_lens[b], 0), capacity);
  r.add = p.new_lens[b];
  r.gone = r.add < 0;
  r.used = (r.len + p.page - 1) >> p.page_shift;
  r.fits = r.add <= p.max_new && r.add <= capacity - r.len;
  r.need = (r.gone || !r.fits) ? 0 : ((r.len + r.add + p.page - 1) >> p.page_shift) - r.used;
  r.back = r.gone ? r.used : 0;
  return r;
}

// One CTA per request. Each CTA scans the page counts of all requests (a few
// hundred integers from L2) instead of waiting for another CTA's prefix, so
// the plan is a single launch without communication: 2.6 us for 8 requests, 3.4
// us for 256 with chunks of up to 512 tokens, the time of a launch and three
// dependent loads (the tables' bytes take 0.3 us). The scans grow with the
// square of the requests; 600 are read in three rounds of loads. Requests take
// free pages in request order; one whose running total passes the free count is
// refused.
__global__ void __launch_bounds__(256) kv4_plan_kernel(const Kv4PlanParams p) {
  __shared__ long long warp_sum[8];
  __shared__ long long mine;  // (pages needed, pages given back) before this request
  const int b = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int head = p.free_state[0] % p.F;
  if (head < 0) head += p.F;
  const int count = min(max(p.free_state[1], 0), p.F);

  // Two running sums in one 64-bit word: needed pages in the high half, pages
  // given back in the low half (both below 2^31: at most every page once).
  long long carry = 0, given_total = 0;
  for (int base = 0; base < p.B; base += 256) {
    const int i = base + threadIdx.x;
    long long v = 0;
    if (i < p.B) {
      const Kv4Request r = kv4_request(p, i);
      v = (static_cast<long long>(r.need) << 32) | static_cast<unsigned>(r.back);
    }
    long long s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    long long before = carry;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    const long long upto = before + s;
    if (i == b) mine = upto - v;
    // pages that requests up to this one really take (only CTA 0 reports it)
    if (i < p.B && (upto >> 32) <= count) given_total = max(given_total, upto >> 32);
    for (int w = 0; w < 8; ++w) carry += warp_sum[w];
    __syncthreads();
  }

  const Kv4Request r = kv4_request(p, b);
  const int first = static_cast<int>(mine >> 32), back0 = static_cast<int>(mine & 0x7fffffff);
  const bool ok = r.gone || (r.fits && (r.need == 0 || first + r.need <= count));
  const int add = (ok && !r.gone) ? r.add : 0;
  const int need = ok ? r.need : 0;
  if (threadIdx.x == 0) {
    p.out_kv_lens[b] = r.gone ? 0 : r.len + add;
    p.out_new_lens[b] = add;
    p.out_accepted[b] = ok ? 1 : 0;
  }
  if (b == 0) {
    // the requests that get pages are a prefix of those that need some
    __shared__ long long best[8];
    long long g = given_total;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) g = max(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (lane == 0) best[warp] = g;
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 8; ++w) g = max(g, best[w]);
      const int returned = min(static_cast<int>(carry & 0x7fffffff), p.F - count);
      p.out_state[0] = static_cast<int>((head + g) % p.F);
      p.out_state[1] = count - static_cast<int>(g) + returned;
    }
  }

  const int* row = p.table + b * p.table_stride;
  auto page_of = [&](int col) -> int {
    if (col < r.used) return row[col];
    const long long at = static_cast<long long>(head) + first + (col - r.used);
    return p.free_pages[at % p.F];
  };
  for (int col = threadIdx.x; col < p.cols; col += 256) {
    int v = -1;
    if (!r.gone && col < r.used + need) v = page_of(col);
    p.out_table[static_cast<long long>(b) * p.cols + col] = v;
    if (r.gone && col < r.used) {
      // behind the live part of the ring, which no CTA of this launch reads
      const long long at = static_cast<long long>(back0) + col;
      if (count + at < p.F) p.free_pages[(head + count + at) % p.F] = row[col];
    }
  }
  for (int i = threadIdx.x; i < p.max_new; i += 256) {
    const long long at = static_cast<long long>(b) * p.max_new + i;
    int slot = -1, pos = -1;
    if (i < add) {
      pos = r.len + i;
      const int page = page_of(pos >> p.page_shift);
      if (page >= 0 && page < p.F) slot = (page << p.page_shift) + (pos & (p.page - 1));
    }
    p.out_slots[at] = slot;
    p.out_positions[at] = pos;
  }
}

// ------------------------------------------------------------------ append
struct Kv4AppendParams {
  const uint16_t* x[2];  // keys, values [B, Hkv, N, D]
  long long sb[2], sh[2], sn[2];
  const int* slots;  // [B][N]
  long long slots_stride;
  uint8_t* pages;
  int B, N, Hkv, page_shift;  // page_shift: log2 of the page's tokens
  int num_slots;
  int* status;
};

template <bool BF16>
__device__ __forceinline__ constexpr float kv4_max_finite() {
  return BF16 ? 3.3895313892515355e38f : 65504.f;
}

// Pairwise maximum and minimum of 16-bit values that keep NaNs.
template <bool BF16>
__device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (BF16)
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (BF16)
    asm("min.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("min.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Quantise this lane's W words (8 values each) of a group whose other words are
// held by the 8 / W - 1 lanes beside it: the words as the cache holds them (keys
// or values) and the group's meta word.
template <bool BF16, int W>
__device__ __forceinline__ void kv4_quantise(const uint4 (&raw)[W], bool keys, uint32_t (&word)[W], uint32_t& meta) {
  uint32_t w[4 * W];
#pragma unroll
  for (int i = 0; i < W; ++i) {
    word[i] = 0;
    w[4 * i] = raw[i].x;
    w[4 * i + 1] = raw[i].y;
    w[4 * i + 2] = raw[i].z;
    w[4 * i + 3] = raw[i].w;
  }
  uint32_t up = w[0], dn = w[0];
#pragma unroll
  for (int i = 1; i < 4 * W; ++i) {
    up = max2_nan<BF16>(up, w[i]);
    dn = min2_nan<BF16>(dn, w[i]);
  }
  // largest x and largest -x, in the halves of one word
  dn ^= 0x80008000u;
  uint32_t top = max2_nan<BF16>(__byte_perm(up, dn, 0x5410), __byte_perm(up, dn, 0x7632));
#pragma unroll
  for (int o = 1; o < 8 / W; o <<= 1) top = max2_nan<BF16>(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float most = kv4_max_finite<BF16>();
  float hi = unpack_lo<BF16>(top), lo = -unpack_hi<BF16>(top);
  if (!(hi <= most && lo >= -most && lo <= most && hi >= -most)) {  // an infinity or a NaN in the group
    meta = KV4_META_NAN;
    return;
  }
  hi = fmaxf(hi, 0.f);
  lo = fminf(lo, 0.f);
  // The smallest 4-bit number that is not below range / 7.5 (of half the
  // values): from a product that is surely not above it, then one exact
  // comparison. 20 low mantissa bits are cleared, rounding up.
  const float range = hi * 0.5f - lo * 0.5f;
  uint32_t sb = (__float_as_uint(range * 0.13333330f) + 0xFFFFFu) & ~0xFFFFFu;
  if (__uint_as_float(sb) * 7.5f < range) sb += 0x100000u;
  const float s = fmaxf(__uint_as_float(sb), BF16 ? 1.1754943508222875e-38f : 4.76837158203125e-7f);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));  // s in [2^-126, 2^126): neither side is flushed
  // floor(x/s + 1/2) by x * (1/s): ties must go up. x/s is a tie or at least
  // 2^-14 away from one (x has at most 11 bits, s 4), and the product is off
  // by less than 2^-18, so a bias of 2^-17 decides every case rightly. Adding
  // 1.5 * 2^23 then rounds to the nearest integer in the low mantissa bits.
  constexpr float EPS = 7.62939453125e-6f, MAGIC = 12582912.f;
  const uint32_t z = __float_as_uint(fmaf(-lo, inv, EPS) + MAGIC) & 15u;
  const float zf = static_cast<float>(z), zb = zf + EPS;
  meta = (__float_as_uint(s) >> 16) | z;
  const bool far = fmaxf(hi, -lo) > most - s;  // a code may pass the largest number
  // hi's code is 16 where both ends of the range are ties: codes grow with x, so no other group has one
  const bool over = fmaf(hi, inv, zb) + MAGIC > MAGIC + 15.f;
#pragma unroll
  for (int u = 0; u < W; ++u) {
    uint32_t c[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t v = w[4 * u + (i >> 1)];
      const float x = (i & 1) ? unpack_hi<BF16>(v) : unpack_lo<BF16>(v);
      c[i] = __float_as_uint(fmaf(x, inv, zb) + MAGIC);
    }
    if (over) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(fminf(__uint_as_float(c[i]), MAGIC + 15.f));
    }
    if (far) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = __uint_as_float(c[i]), v = s * (y - MAGIC - zf);
        c[i] = __float_as_uint(y + ((v > most) ? -1.f : (v < -most) ? 1.f : 0.f));
      }
    }
    // codes are the low bytes of c (0..15 each: the magic number's low byte is
    // 0): nibbles 0, 2, 4, 6 and 1, 3, 5, 7 of the word
    auto bytes = [](uint32_t a, uint32_t b, uint32_t d, uint32_t e) {
      return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(d, e, 0x0040), 0x5410);
    };
    const uint32_t even = keys ? bytes(c[0], c[4], c[1], c[5]) : bytes(c[0], c[2], c[4], c[6]);
    const uint32_t odd = keys ? bytes(c[2], c[6], c[3], c[7]) : bytes(c[1], c[3], c[5], c[7]);
    word[u] = even | (odd << 4);
  }
}

// Key word order (nibble i: dim 2i, nibble 4+i: dim 2i+1) -> value order.
__device__ __forceinline__ uint32_t kv4_key_values(uint32_t c) {
  uint32_t t = (c ^ (c >> 8)) & 0x0000FF00u;
  c ^= t ^ (t << 8);
  t = (c ^ (c >> 4)) & 0x00F000F0u;
  c ^= t ^ (t << 4);
  return c;
}

// LANES neighbouring lanes hold one group of a token, lane t the words 2t, 2t+1
// (and 2t+4, 2t+5 where there are two lanes) of its keys and values: the group's
// extremes are a shuffle reduction over packed pairs, and nothing else is shared.
// The rows are loaded beside the slot, not behind it. blockIdx: 256 / LANES
// (token, group) pairs, head, request.
//
// 16384 tokens of 8 heads at head_dim 256 take 31.2 us with two lanes, 5.4 TB/s;
// the scale's arithmetic and the addresses, once per lane, made it bound by ALU
// instructions before: 36 us with four lanes a group, 65 with eight and divisions.
// (An order in which a warp takes the 16 tokens of a block, for stores of whole
// sectors, waits for the row's first slot: 32.5.) Few tokens take four lanes, see
// the launch.
template <int D, bool BF16, int LANES>
__global__ void __launch_bounds__(256) kv4_append_kernel(const Kv4AppendParams p) {
  constexpr int NG = D / KV4_GROUP;
  constexpr int W = 8 / LANES;
  const int t = threadIdx.x % LANES;
  const int blocks_shift = p.page_shift - 4;
  const int h = blockIdx.y, b = blockIdx.z;
  const unsigned pair = blockIdx.x * (256u / LANES) + threadIdx.x / LANES;
  const int g = pair % NG, n = pair / NG;
  uint4 raw[2][W] = {};
  int slot = -1;
  if (n < p.N) {  // the shuffles need all lanes
    slot = p.slots[b * p.slots_stride + n];
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const uint4* src = reinterpret_cast<const uint4*>(p.x[kind] + b * p.sb[kind] + h * p.sh[kind] + n * p.sn[kind] +
                                                        g * KV4_GROUP + t * 16);
#pragma unroll
      for (int i = 0; i < W; ++i) raw[kind][i] = __ldcs(src + (i & 1) + (i >> 1) * 4);
    }
  }
  if (slot >= p.num_slots || slot < -1) {
    if (t == 0) atomicCAS(p.status, 0, ST_KV4_SLOT);
    slot = -1;
  }
  const int r = slot & 15;
  const int blk = (slot >> 4) & ((1 << blocks_shift) - 1);
  uint8_t* page = p.pages + ((((static_cast<long long>(slot >> p.page_shift) * 2 * p.Hkv) + h) << blocks_shift) + blk) *
                                kv4_block_bytes(D);
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    uint32_t meta;
    uint32_t word[W];
    kv4_quantise<BF16, W>(raw[kind], kind == 0, word, meta);
    if (slot >= 0) {
      uint8_t* dst = page + (kind == 0 ? 0 : (static_cast<long long>(p.Hkv) << blocks_shift) * kv4_block_bytes(D));
      uint8_t* codes = dst + g * KV4_CODE_BYTES;
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        const int j = 2 * t + 2 * i;
        if (kind == 0) {
          *reinterpret_cast<uint2*>(codes + kv4_key_word(r, j)) = make_uint2(word[i], word[i + 1]);
        } else {
          *reinterpret_cast<uint32_t*>(codes + kv4_value_word(r, j)) = word[i];
          *reinterpret_cast<uint32_t*>(codes + kv4_value_word(r, j + 1)) = word[i + 1];
        }
      }
      if (t == 0)
        reinterpret_cast<uint16_t*>(dst + NG * KV4_CODE_BYTES + g * KV4_META_BYTES)[kind == 0 ? kv4_key_meta(r)
                                                                                             : kv4_value_meta(r)] =
            static_cast<uint16_t>(meta);
    }
  }
}

// ------------------------------------------------------------------ read
struct Kv4ReadParams {
  const uint8_t* pages;
  const int* table;  // [B][cols]
  long long table_stride;
  const int* kv_lens;
  const int* starts;  // [B] or null (0)
  uint16_t* out[2];   // keys, values [B, Hkv, n, D] contiguous
  int B, Hkv, n, cols, page_shift, num_pages;
  int xblocks;  // CTAs per request and head
  int* status;
  // For the ragged forward: the keys it reads (ragged_lens), and zeros only up
  // to the end of its last key block.
  int q_rows, window;
  const int* q_lens;
};

// Behind the values that are written out for the ragged forward: a bit for each
// token of a (block, group) whose values are not finite, [B * Hkv][kv4_nan_pitch],
// item (block from the first one on) * NG + group. rows: as many as are written
// out, a multiple of 16.
__host__ __device__ constexpr long long kv4_nan_pitch(long long rows, int head_dim) {
  return (rows / KV4_TOKENS * (head_dim / KV4_GROUP) + 7) / 8 * 8;
}

constexpr int KV4_READ_UNITS = 4;  // groups of a block a warp reads, many of them

// Eight values of a word as 16 bytes of 16-bit values, exactly s * (c - z).
template <bool BF16>
__device__ __forceinline__ uint4 kv4_values(uint32_t codes, uint32_t meta) {
  const float s = __uint_as_float((meta & 0xFFF0u) << 16);
  const float zs = -(static_cast<float>(meta & 15u)) * s;  // at most 8 bits: exact
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float lo = fmaf(static_cast<float>((codes >> (8 * i)) & 15u), s, zs);
    const float hi = fmaf(static_cast<float>((codes >> (8 * i + 4)) & 15u), s, zs);
    w[i] = pack2<BF16>(lo, hi);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// A warp reads UNITS consecutive groups of 16-token blocks (16 bytes a lane and
// group, as stored; all loads in flight together) and writes 16 tokens x 64
// values of each: 128 contiguous bytes per token. blockIdx.x: request, head and
// 8 * UNITS (block, group) pairs; blockIdx.y: keys / values. Rows behind a
// request's last token become zeros. Mostly writes, 79 % of the bytes: 16384 tokens
// of 8 heads at head_dim 256 take 34.8 us, 4.9 TB/s read and written, five ragged
// caches of up to 16384 tokens at head_dim 128 5.3 TB/s, of the copy's 6.6. (Key
// stores of 16 bytes, half a sector each: 42 us. Two or eight groups a warp instead
// of four: 7 and 3 % more over the ragged caches.) Stores that the L2 drops first
// took 72 us there instead of 75. Not gone into: `p.out[kind]` makes every thread
// copy the parameters to local memory first.
//
// For the ragged forward, whose MMAs also multiply masked keys' values by P = 0,
// a value group that is NaN goes out as zeros, and a bit behind them tells
// kv4_spread_nan_kernel to mark the rows that see it.
template <int D, bool BF16, bool RAGGED, int UNITS>
__global__ void __launch_bounds__(256) kv4_read_kernel(const Kv4ReadParams p) {
  constexpr int NG = D / KV4_GROUP;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int kind = blockIdx.y;
  const int bh = blockIdx.x / p.xblocks;
  const int h = bh % p.Hkv, b = bh / p.Hkv;
  const int capacity = p.cols << p.page_shift;
  int len = p.kv_lens[b];
  if (len > capacity) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, ST_KV4_LENGTH);
    len = capacity;
  }
  int start = p.starts ? max(p.starts[b], 0) : 0, n = p.n;
  if constexpr (RAGGED) {
    const RaggedLens r = ragged_lens(p.kv_lens, p.q_lens, b, capacity, p.q_rows, p.window);
    start = r.start;
    if (r.Nk > p.n && threadIdx.x == 0) atomicCAS(p.status, 0, ST_KV4_LENGTH);  // beyond the given bound
    n = min(p.n, (r.Nk + 255) & ~255);
  }
  const int item0 = ((blockIdx.x - bh * p.xblocks) * 8 + warp) * UNITS;
  const int blocks_shift = p.page_shift - 4;
  const long long end = static_cast<long long>(start) + n;
  uint4 codes[UNITS];
  uint2 metas[UNITS];
  uint32_t bad[UNITS];  // tokens whose values in this group are not finite
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const int g = (item0 + k) % NG;
    const long long pos0 = (static_cast<long long>(start) / 16 + (item0 + k) / NG) * 16;  // first token of the block
    codes[k] = make_uint4(0, 0, 0, 0);
    metas[k] = make_uint2(0, 0);
    bad[k] = 0;
    if (pos0 >= len || pos0 >= end) continue;
    const int blk = static_cast<int>(pos0 >> 4);
    const int page = __ldg(p.table + b * p.table_stride + (blk >> blocks_shift));
    if (page < 0 || page >= p.num_pages) {
      if (lane == 0) atomicCAS(p.status, 0, ST_KV4_PAGE);
      continue;
    }
    const uint8_t* src = p.pages + ((((static_cast<long long>(page) * 2 + kind) * p.Hkv + h) << blocks_shift) +
                                    (blk & ((1 << blocks_shift) - 1))) *
                                       kv4_block_bytes(D);
    codes[k] = __ldg(reinterpret_cast<const uint4*>(src + g * KV4_CODE_BYTES + lane * 16));
    const uint8_t* m = src + NG * KV4_CODE_BYTES + g * KV4_META_BYTES;
    if (kind == 0)
      metas[k].x = __ldg(reinterpret_cast<const uint32_t*>(m + (lane >> 2) * 4));
    else
      metas[k] = __ldg(reinterpret_cast<const uint2*>(m + (lane >> 3) * 8));
  }
  if (RAGGED && kind == 1 && (static_cast<long long>(start) / 16 + item0 / NG) * 16 < end) {
#pragma unroll
    for (int k = 0; k < UNITS; ++k) {
      const long long pos0 = (static_cast<long long>(start) / 16 + (item0 + k) / NG) * 16;
      const uint32_t word[4] = {metas[k].x & 0xFFFFu, metas[k].x >> 16, metas[k].y & 0xFFFFu, metas[k].y >> 16};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = (lane >> 3) * 2 + (j & 1) + (j >> 1) * 8;  // inverse of kv4_value_meta
        if ((word[j] & 0x7F80u) == 0x7F80u && pos0 + r < len) bad[k] |= 1u << r;
      }
      bad[k] = __reduce_or_sync(0xffffffffu, bad[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < UNITS; ++k) {
    const int g = (item0 + k) % NG;
    const long long pos0 = (static_cast<long long>(start) / 16 + (item0 + k) / NG) * 16;
    if (pos0 >= end) return;
    if (RAGGED && kind == 1 && k == 0 && lane == 0) {
      static_assert(UNITS == 4 || !RAGGED, "four words of 16 bits; the pitch leaves room for those behind the last item");
      *reinterpret_cast<uint2*>(p.out[1] + static_cast<long long>(p.B) * p.Hkv * p.n * D + bh * kv4_nan_pitch(p.n, D) +
                                item0) = make_uint2(bad[0] | bad[UNITS > 1 ? 1 : 0] << 16,
                                                    bad[UNITS > 2 ? 2 : 0] | bad[UNITS > 3 ? 3 : 0] << 16);
    }
    uint16_t* out = p.out[kind] + (static_cast<long long>(b) * p.Hkv + h) * p.n * D + g * KV4_GROUP;
    auto value = [&](int r, uint32_t c, uint32_t m) {
      if (pos0 + r >= len) return make_uint4(0, 0, 0, 0);
      if (RAGGED && ((bad[k] >> r) & 1u)) return make_uint4(0, 0, 0, 0);
      return kv4_values<BF16>(c, m);
    };
    auto store = [&](int r, int j, uint32_t c, uint32_t m) {
      const long long i = pos0 + r - start;
      if (i < 0 || i >= n) return;
      uint4* at = reinterpret_cast<uint4*>(out + i * D + j * 8);
      if constexpr (RAGGED)
        *at = value(r, c, m);
      else
        __stcs(at, value(r, c, m));
    };
    auto store_pair = [&](int r, int t, uint32_t c0, uint32_t c1, uint32_t m) {
      const long long i = pos0 + r - start;
      if (i < 0 || i >= n) return;
      const uint4 v = value(r, c0, m), w = value(r, c1, m);
      if constexpr (RAGGED)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + i * D + t * 16), "r"(v.x),
                     "r"(v.y), "r"(v.z), "r"(v.w), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                     : "memory");
      else
        asm volatile("st.global.cs.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out + i * D + t * 16),
                     "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                     : "memory");
    };
    const uint2 m = metas[k];
    if (kind == 0) {
      // words 2t and 2t + 1 of a token in one 32-byte store: whole sectors
      const int r = lane >> 2, t = lane & 3;
      store_pair(r, t, kv4_key_values(codes[k].x), kv4_key_values(codes[k].y), m.x & 0xFFFFu);
      store_pair(r + 8, t, kv4_key_values(codes[k].z), kv4_key_values(codes[k].w), m.x >> 16);
    } else {
      const int t = lane >> 3, j = (lane & 7) ^ (2 * t);
      store(2 * t, j, codes[k].x, m.x & 0xFFFFu);
      store(2 * t + 1, j, codes[k].y, m.x >> 16);
      store(2 * t + 8, j, codes[k].z, m.y & 0xFFFFu);
      store(2 * t + 9, j, codes[k].w, m.y >> 16);
    }
  }
}

// ------------------------------------------------------------------ NaNs
struct Kv4SpreadParams {
  const uint16_t* nans;  // see kv4_nan_pitch
  uint16_t* o;
  long long o_sb, o_sh, o_sn;
  const int *kv_lens, *q_lens;
  int Hkv, G, N, n, capacity, causal, window;  // n: rows of keys that were written out
};

// After the ragged forward: the dims of a value group that is not finite become
// NaN in the rows that see its token, as P * NaN would make them. One CTA per
// request and KV head; without such a group it reads the bits (16 KB for 16384
// keys at head_dim 512) and leaves: a launch more, 48 tokens of 2 requests behind
// 7K keys at head_dim 512 take 177.6 us instead of 172.0, 100 tokens of 8 at 64
// 149.7 instead of 148.1.
template <int D>
__global__ void __launch_bounds__(512) kv4_spread_nan_kernel(const Kv4SpreadParams p) {
  constexpr int NG = D / KV4_GROUP;
  const int b = blockIdx.x / p.Hkv, h = blockIdx.x - b * p.Hkv;
  const RaggedLens len = ragged_lens(p.kv_lens, p.q_lens, b, p.capacity, p.N, p.window);
  const int Nk = min(len.Nk, p.n), off = Nk - len.N;
  const uint16_t* nans = p.nans + blockIdx.x * kv4_nan_pitch(p.n, D);
  const int items = (Nk + 15) / 16 * NG;
  uint32_t any = 0;
  for (int i = threadIdx.x * 8; i < items; i += 512 * 8) {
    if (i + 8 <= items) {
      const uint4 w = *reinterpret_cast<const uint4*>(nans + i);
      any |= w.x | w.y | w.z | w.w;
    } else {
      for (int j = i; j < items; ++j) any |= nans[j];
    }
  }
  if (!__syncthreads_or(any != 0)) return;
  for (int at = threadIdx.x; at < len.N * NG; at += 512) {
    const int n = at / NG, g = at - n * NG;
    const int hi = p.causal ? min(Nk, n + off + 1) : Nk;
    const int lo = (p.causal && p.window > 0) ? max(0, n + off - p.window + 1) : 0;
    bool hit = false;
    for (int blk = lo >> 4; !hit && blk * 16 < hi; ++blk) {
      uint32_t bits = nans[blk * NG + g];
      if (blk * 16 < lo) bits &= 0xFFFFu << (lo - blk * 16);
      if (blk * 16 + 16 > hi) bits &= 0xFFFFu >> (blk * 16 + 16 - hi);
      hit = bits != 0;
    }
    if (!hit) continue;
    for (int i = 0; i < p.G; ++i) {
      uint4* row = reinterpret_cast<uint4*>(p.o + b * p.o_sb + (h * p.G + i) * p.o_sh + n * p.o_sn + g * KV4_GROUP);
#pragma unroll
      for (int j = 0; j < 8; ++j) row[j] = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
    }
  }
}

}  // namespace gqafa
