// Attention of a few new tokens over the paged 4-bit KV cache (kv4_layout.cuh):
//
//   O[n] = sum_j softmax_j(scale * q_n . k_j) v_j over the keys j that the
//   causal mask and the window leave to token n, k and v read from the codes.
//
// Mathematics. Scores run on integer MMAs: two ANDs and a shift split a word of
// eight codes into two registers of bytes, and the query goes to the other
// operand as two signed bytes, round(q * 32512 / max|q|) = 256 hi + lo, off by
// at most 2^-16 of its row's largest value. A group's part of a score is then
// s * (256 q_hi . c + q_lo . c - z * sum(q)) with an exact integer in the
// brackets; scales are applied in fp32. A row whose largest value is more than 32
// times its mean gets a third byte (2^-24 of the largest value) in a pass of its
// own over the block: its other dims would lose their bits to that one (a channel
// of 10000 that the keys do not use put 9 % on the output). (16-bit operands took 28 ALU
// instructions per 16 tokens x 64 dims to make instead of 12, and the ALU is
// the busiest pipe; fp8 MMAs of this shape are not native on sm_100.)
//
// Values: P' = round16(s * P) is the B operand (integers have not the range of
// a softmax's tail), a code is set into a 16-bit number F + c, F a power of two,
// by one AND-OR of a (shifted) word. bf16: F = 128 for every nibble. fp16:
// F = 256 and 16 for even and odd nibbles, so that one shift serves two. One
// more MMA subtracts sum_j (F + z_j) P'_j with the same rounded P', so the
// offset cancels exactly and only P' itself is rounded. The two accumulators
// are joined after every tile: F * sum(P') would otherwise outgrow the result
// over a long cache and cost it its low bits.
//
// fp16 has not the exponents for s * P: with s = 3e-4 (values of 1e-3) and P =
// 2^-3 it would begin among the subnormals and lose every weight below 2^-10 of
// the largest. So P carries a power of two that brings the largest scale met so
// far (of all groups) to the exponent of TOP, and the accumulators give it back
// at the end: P' of the largest key is then at least 2^10 for the largest scale,
// 24 powers of two above the least normal number, whatever the values' size.
// (16384 keys of values near 0.02 with one score 9.7 above the others: 16 % of
// the result were lost without it.) The warps look at the value blocks' scales
// before a tile's barrier, a word per thread; a larger one is published as a
// raised maximum is. That costs 109 us against 104 at head_dim 512, 16 requests of
// 8K to 16K keys, 46.5 against 42.6 at 128 (each warp looking after its own groups
// in the value loop, with a power for each: 113 and 49.5). Groups whose scales are
// below 2^-10 of the head's largest have that much less room.
// bf16 needs none of it.
//
// Shape. A decode step has G = H_Q / H_KV query rows per KV head, far below
// the 128 rows of a tcgen05 tile, and reads each cached byte once: it is bound
// by HBM. The products therefore run transposed on m16n8 MMAs with the
// CACHE as the A operand (16 tokens, or 16 dims, by 8 query rows): padding
// costs at most 8 rows, and the codes go from shared memory to registers to
// the tensor cores without a dequantised copy in between.
//
// One CTA: eight compute warps and one producer warp. The producer walks the
// block table and brings whole blocks (codes and scales together) into a ring
// of stages with bulk copies. Work is cut into tiles of TB blocks. Scores: warp
// w takes blocks w, w + 8, ... over all of head_dim; P goes to shared memory
// (fp32), one barrier per tile. Values: warp (dim group, slice) takes 64 dims
// of every KS-th block, so the output accumulator is 16 registers per 8 query
// rows. All warps share one reference maximum per row; a warp that meets a
// larger score publishes its own for this tile, and only then are P and the
// accumulators rescaled.
// The ninth warp costs registers (96 a thread, two CTAs per SM, instead of 128),
// but warp 0 issuing the copies between its own tiles delays the other seven:
// 130 us against 106 at head_dim 512, 16 requests of 8K to 16K keys, 54 against
// 38 at head_dim 128 (both before the third byte and fp16's power of two). A producer
// warpgroup that gives its registers away (104 for the others) made the first 1 %
// faster and the second 5 % slower.
//
// Measured: 16 requests of 8K to 16K keys, 32/4 heads, head_dim 512: 107.8 us for 430
// MB of codes, 4.0 TB/s (fp16 111); 131072 keys of one request, 16/2 heads: 46.0 us,
// 3.1 TB/s. Bound by neither alone: 57 % of the issue slots, 56 % of the ALU
// (profiles/kv4_decode_d512.md); without the products the first took 83 us. 20 rows
// at head_dim 128 (three units): 40.4 us, fp16 43.6, bound by instructions.
//
// Split. The tiles of all (request, row tile, KV head) units form one list,
// cut into equal contiguous shares, one per CTA: ragged lengths and a single
// long request both fill the GPU. A unit inside one share is written straight
// to the output; parts of a cut unit go to a workspace (fp32, with maximum and
// sum) and kv4_combine_kernel joins them in list order, so results do not
// depend on timing. (The last CTA to arrive joining them inside this kernel was
// slower: 16 parts of 16 KB take one CTA 10 us.) A unit has at most 8 rows; more
// rows take more units, which read the keys again from L2: units of 16 and 32
// rows (more registers, one CTA per SM) were slower, 50 and 67 us against 41
// for 20 rows at head_dim 128.
#pragma once
#include <type_traits>

#include "kv4_layout.cuh"
#include "ptx_sm100.cuh"

namespace gqafa {

// The powers of two that codes are set into (see codes16), and their negatives.
struct Kv4Tops {
  uint32_t even, odd, minus_even, minus_odd;
};
inline Kv4Tops kv4_tops(bool bf16) {
  return bf16 ? Kv4Tops{0x43004300u, 0x43004300u, 0xC300C300u, 0xC300C300u}
              : Kv4Tops{0x5C005C00u, 0x4C004C00u, 0xDC00DC00u, 0xCC00CC00u};
}

struct Kv4Params {
  Kv4Tops tops;
  const uint16_t* q;
  long long q_sb, q_sh, q_sn;
  uint16_t* o;
  long long o_sb, o_sh, o_sn;
  float* lse;  // [B, Hq, N] or null
  const uint8_t* pages;
  const int* table;  // [B][cols]
  long long table_stride;
  const int* kv_lens;
  const int* q_lens;  // [B] or null (N)
  int B, Hq, Hkv, G, N;
  int cols, page_shift, num_pages;  // page_shift: log2 of the page's tokens
  int causal, window;
  float scale_log2;
  int row_tiles;  // row tiles (8 rows each) of G * N rows
  int ctas;       // CTAs of the attention launch (the combine launch needs it)
  float* part_o;  // [2 * ctas][8][D]
  float2* part_ml;  // [2 * ctas][8]: maximum (log2 units), sum
  int join_blocks;  // CTAs of the join per unit
  int* status;
  long long wait_limit;
  int no_loads;
};

// Blocks per warp and tile: enough work between barriers, or (wide false) tiles
// that spread a few keys over more CTAs.
__host__ __device__ constexpr int kv4_warp_blocks(int D, bool wide) {
  return D == 512 ? 1 : (D == 256 ? (wide ? 2 : 1) : (D == 128 ? (wide ? 4 : 1) : (wide ? 4 : 2)));
}

template <int D_, bool BF16_, bool WIDE_>
struct Kv4Cfg {
  static constexpr int D = D_;
  static constexpr bool BF16 = BF16_;
  static constexpr int ROWS = 8;              // query rows of a unit
  static constexpr int NG = D / KV4_GROUP;    // groups of a token
  static constexpr int KS = 8 / NG;           // value-side slices of a tile's blocks
  static constexpr int KB = kv4_warp_blocks(D, WIDE_);
  static constexpr int TB = 8 * KB;           // blocks per tile
  static constexpr int SB = TB / 2;           // blocks per stage
  static constexpr int BLOCK_BYTES = kv4_block_bytes(D);
  static constexpr int STAGE_BYTES = SB * BLOCK_BYTES;
  static constexpr int Q_PITCH = D * 2 + 16;  // bytes; +16: fragment loads hit all banks
  static constexpr int Q_BYTES = ROWS * Q_PITCH;
  static constexpr int SUMQ_BYTES = NG * ROWS * 4;
  static constexpr int Q3_PITCH = D + 16;     // third bytes of the query
  static constexpr int Q3_BYTES = ROWS * Q3_PITCH;
  static constexpr int P_PITCH = 20;          // floats of a row's 16 probabilities
  static constexpr int P_BYTES = TB * ROWS * P_PITCH * 4;  // one of two buffers
  static constexpr int M_BYTES = 8 * ROWS * 4;             // one of two buffers
  static constexpr int MISC_BYTES = 2 * P_BYTES + 2 * M_BYTES + Q_BYTES + Q3_BYTES + 2 * SUMQ_BYTES + ROWS * 20 + 256;
  static constexpr int CTAS_PER_SM = 2;
  // half of an SM's 228 KB, less 1 KB that a CTA takes and its static variables
  static constexpr int NST_FIT = (115400 - MISC_BYTES) / STAGE_BYTES;
  static constexpr int NST = NST_FIT < 12 ? NST_FIT : 12;
  static constexpr int SMEM_BYTES = NST * STAGE_BYTES + MISC_BYTES;
  static constexpr int THREADS = 288;
  // Reference of a row's softmax: its largest score so far plus RAISE when it
  // was last raised, and it is raised again when a score passes it by more than
  // SLACK (log2 units), so P stays within 2^SLACK. bf16 P' has the range for
  // that; fp16 P' = s * P must stay below 65504, with s brought to at most
  // 1.875 * 2^13 (TOP).
  static constexpr float RAISE = BF16 ? 8.f : 3.f;
  static constexpr int SLACK2 = BF16 ? 8 : 2;
  static constexpr float SLACK = SLACK2;
  // fp16: exponent fields of the format's smallest and largest scales (2^-21 and
  // 9216, the 4-bit number above 2 * 65504 / 15).
  static constexpr int BOTTOM = 127 - 21, TOP = 127 + 13;
  static_assert(BF16 || 1.875 * (1 << (TOP - 127)) * (1 << SLACK2) <= 65504 * 0.99, "P' stays finite");
  static_assert(NST >= 4, "two stages of keys and two of values");
  // the slices' sums are joined through the P buffers
  static_assert(KS == 1 || (KS / 2) * ROWS * D * 4 <= 2 * P_BYTES, "slice exchange");
};

// One unit's keys: tiles of blocks [b0, b0 + nblk) of request b.
struct Kv4Unit {
  int b, rt, len, qlen;
  int b0, nblk, tiles;
};

template <class C>
__device__ __forceinline__ Kv4Unit kv4_unit(const Kv4Params& p, int entry) {
  Kv4Unit u;
  u.b = entry / p.row_tiles;
  u.rt = entry - u.b * p.row_tiles;
  const int capacity = p.cols << p.page_shift;
  u.len = min(max(p.kv_lens[u.b], 0), capacity);
  u.qlen = p.q_lens ? min(max(p.q_lens[u.b], 0), p.N) : p.N;
  u.b0 = u.nblk = u.tiles = 0;
  const int r0 = u.rt * C::ROWS, rows = p.G * u.qlen;
  if (r0 >= rows) return u;
  const int n0 = r0 / p.G, n1 = (min(r0 + C::ROWS, rows) - 1) / p.G;
  const int off = u.len - u.qlen;
  const int hi = p.causal ? min(u.len, off + n1 + 1) : u.len;
  const int lo = (p.causal && p.window > 0) ? max(0, off + n0 - p.window + 1) : 0;
  if (hi <= lo) return u;
  u.b0 = lo >> 4;
  u.nblk = ((hi + 15) >> 4) - u.b0;
  u.tiles = (u.nblk + C::TB - 1) / C::TB;
  return u;
}

// Position of a CTA's share in the list of tiles: entries in order, the KV
// heads of an entry one after the other.
struct Kv4Share {
  int entry;      // entry that holds the share's first tile
  int base;       // index of that entry's first tile
  int total;      // tiles in all
};

// Block-wide (NTHR threads): total number of tiles, and the entry that holds
// tile `per * index` with per = ceil(total / ctas). Every thread gets the
// result. `scratch`: 40 ints of shared memory.
template <class C, int NTHR>
__device__ __forceinline__ Kv4Share kv4_find(const Kv4Params& p, int index, int* scratch) {
  const int entries = p.B * p.row_tiles;
  const int each = (entries + NTHR - 1) / NTHR;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int e0 = min(entries, static_cast<int>(threadIdx.x) * each), e1 = min(entries, e0 + each);
  int sum = 0;
  for (int e = e0; e < e1; ++e) sum += kv4_unit<C>(p, e).tiles * p.Hkv;
  int s = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) scratch[warp] = s;
  if (threadIdx.x == 0) {
    scratch[32] = 0;
    scratch[33] = 0;
  }
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NTHR / 32; ++w) {
    const int v = scratch[w];
    if (w < warp) before += v;
    total += v;
  }
  const int first = before + s - sum;
  const int per = max(1, (total + p.ctas - 1) / p.ctas);
  const long long at = static_cast<long long>(per) * index;
  if (at >= first && at < first + sum) {
    int base = first;
    for (int e = e0; e < e1; ++e) {
      const int t = kv4_unit<C>(p, e).tiles * p.Hkv;
      if (at < base + t) {
        scratch[32] = e;
        scratch[33] = base;
        break;
      }
      base += t;
    }
  }
  __syncthreads();
  Kv4Share r;
  r.entry = scratch[32];
  r.base = scratch[33];
  r.total = total;
  return r;
}

// ------------------------------------------------------------------ fragments
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}

template <bool BF16>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

// Bytes: d = a (unsigned) * b (signed) + c.
__device__ __forceinline__ void imma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, int c0, int c1, int c2, int c3) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3));
}

// (x & mask) | top as one LOP3. An instruction takes one immediate: `top` comes
// from the kernel's parameters, so it stays in a register (as a second
// immediate it cost another instruction per MMA operand: 61 ALU instructions
// per 16 tokens x 64 dims, the busiest pipe, at head_dim 512).
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t top) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(top));
  return r;
}

// F + code for the four nibbles of both 16-bit halves of w. bf16: 0x4300 is
// 128, its last mantissa bit worth 1. fp16: the even nibbles of w << 2 and
// w >> 6 lie at bits 2..5 of 256 (0x5C00), the odd ones at bits 6..9 of 16.
template <bool BF16>
__device__ __forceinline__ void codes16(uint32_t w, const Kv4Tops& f, uint32_t (&a)[4]) {
  if constexpr (BF16) {
    a[0] = and_or(w, 0x000F000Fu, f.even);
    a[1] = and_or(w >> 4, 0x000F000Fu, f.even);
    a[2] = and_or(w >> 8, 0x000F000Fu, f.even);
    a[3] = and_or(w >> 12, 0x000F000Fu, f.even);
  } else {
    const uint32_t l = w << 2, r = w >> 6;
    a[0] = and_or(l, 0x003C003Cu, f.even);
    a[1] = and_or(l, 0x03C003C0u, f.odd);
    a[2] = and_or(r, 0x003C003Cu, f.even);
    a[3] = and_or(r, 0x03C003C0u, f.odd);
  }
}
// -(F + zero point) of two packed meta words, for even and odd nibbles.
template <bool BF16>
__device__ __forceinline__ uint32_t minus_zero_even(uint32_t w, const Kv4Tops& f) {
  return BF16 ? and_or(w, 0x000F000Fu, f.minus_even) : and_or(w << 2, 0x003C003Cu, f.minus_even);
}
template <bool BF16>
__device__ __forceinline__ uint32_t minus_zero_odd(uint32_t w, const Kv4Tops& f) {
  return BF16 ? and_or(w, 0x000F000Fu, f.minus_even) : and_or(w << 6, 0x03C003C0u, f.minus_odd);
}
__device__ __forceinline__ uint32_t max2_u16(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Scale of the meta word in w's upper half.
__device__ __forceinline__ float meta_scale(uint32_t w) { return __uint_as_float(w & 0xFFF00000u); }

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
      "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void compute_barrier() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
// The same barrier; returns whether any thread brought a true predicate.
__device__ __forceinline__ bool compute_barrier_or(bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}\n"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(v))
      : "memory");
  return r != 0;
}
// The slow side of a wait, out of line: the fast side is one try_wait.
__device__ __noinline__ void kv4_wait_slow(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status,
                                           long long limit) {
  mbar_wait(bar, parity, abort_flag, status, ST_TIMEOUT_RING_FULL, limit);
}

// Adds what the query's third bytes give to a block's scores, times w0 and w1 for
// the lane's two rows.
template <int NG>
__device__ __forceinline__ void kv4_third_bytes(float (&v)[4], uint32_t codes, uint32_t metas,
                                                const uint8_t* query, const int* sums, float w0, float w1) {
#pragma unroll 1
  for (int g = 0; g < NG; ++g) {
    const uint4 w = lds128(codes + g * KV4_CODE_BYTES);
    const uint32_t m = lds32(metas + g * KV4_META_BYTES);
    const uint4 q = lds128(smem_u32(query) + g * 64);
    const int2 sq = *reinterpret_cast<const int2*>(sums + g * 8);
    constexpr uint32_t M = 0x0F0F0F0Fu;
    int t[4];
    imma16832(t, w.x & M, w.z & M, (w.x >> 4) & M, (w.z >> 4) & M, q.x, q.y, 0, 0, 0, 0);
    imma16832(t, w.y & M, w.w & M, (w.y >> 4) & M, (w.w >> 4) & M, q.z, q.w, t[0], t[1], t[2], t[3]);
    const float s0 = meta_scale(m << 16), s1 = meta_scale(m);
    const int z0 = m & 15, z1 = (m >> 16) & 15;
    v[0] = fmaf(s0, static_cast<float>(t[0] - z0 * sq.x) * w0, v[0]);
    v[1] = fmaf(s0, static_cast<float>(t[1] - z0 * sq.y) * w1, v[1]);
    v[2] = fmaf(s1, static_cast<float>(t[2] - z1 * sq.x) * w0, v[2]);
    v[3] = fmaf(s1, static_cast<float>(t[3] - z1 * sq.y) * w1, v[3]);
  }
}
// Out of line where a warp has several blocks of a tile, each a copy of code that
// few queries run: 46.5 us against 48.8 at head_dim 128, fp16; with one block
// (head_dim 512) 109.5 against 107.7.
template <int NG>
__device__ __noinline__ float4 kv4_third_bytes_call(uint32_t codes, uint32_t metas, const uint8_t* query,
                                                    const int* sums, float w0, float w1) {
  float v[4] = {};
  kv4_third_bytes<NG>(v, codes, metas, query, sums, w0, w1);
  return make_float4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }

template <class C>
__global__ void __launch_bounds__(C::THREADS, C::CTAS_PER_SM) kv4_attn_kernel(const Kv4Params p) {
  constexpr int D = C::D, NG = C::NG, KS = C::KS, KB = C::KB, TB = C::TB, SB = C::SB, ROWS = C::ROWS;
  constexpr int NST = C::NST, BB = C::BLOCK_BYTES, PP = C::P_PITCH;
  constexpr bool BF16 = C::BF16;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* sRing = smem;
  float* sP = reinterpret_cast<float*>(smem + NST * C::STAGE_BYTES);  // [2][TB][ROWS][PP]
  float* sM = sP + 2 * C::P_BYTES / 4;                                 // [2][8 warps][ROWS]
  uint8_t* sQ = reinterpret_cast<uint8_t*>(sM + 2 * 8 * ROWS);         // [ROWS] rows of Q_PITCH bytes
  uint8_t* sQ3 = sQ + C::Q_BYTES;                                      // [ROWS] rows of Q3_PITCH bytes
  int* sSum = reinterpret_cast<int*>(sQ3 + C::Q3_BYTES);               // [NG][ROWS] sum of the integer query
  int* sSum3 = sSum + C::SUMQ_BYTES / 4;                               // [NG][ROWS] sum of the third bytes
  int2* sMask = reinterpret_cast<int2*>(sSum3 + C::SUMQ_BYTES / 4);    // [ROWS]: first key, number of keys
  float* sScale = reinterpret_cast<float*>(sMask + ROWS);              // [ROWS]: log2 units per unit of MMA result
  int* sMost = reinterpret_cast<int*>(sScale + ROWS);                  // [ROWS]: largest |q|, as bits
  int* sAbs = sMost + ROWS;                                            // [ROWS]: sum of the integer query's magnitudes
  uint64_t* bars = reinterpret_cast<uint64_t*>(sAbs + ROWS);
  __shared__ int scratch[40];
  __shared__ __align__(16) int raised[2][8];  // warps that published a maximum for a tile
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(bars);
  auto FULL = [&](int s) { return bar0 + 8u * s; };
  auto EMPTY = [&](int s) { return bar0 + 8u * (NST + s); };
  if (threadIdx.x == 0) {
    for (int s = 0; s < NST; ++s) {
      mbar_init(FULL(s), 1);
      mbar_init(EMPTY(s), 8);
    }
    abort_word = 0;
    fence_mbar_init();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const Kv4Share share = kv4_find<C, C::THREADS>(p, blockIdx.x, scratch);  // also orders the barrier setup
  const int per = max(1, (share.total + p.ctas - 1) / p.ctas);
  const long long begin = static_cast<long long>(per) * blockIdx.x;
  if (begin >= share.total) return;
  const int first_tile = static_cast<int>(begin);
  const int last_tile = min(share.total, first_tile + per);

  // Walk the pieces of the share: f(unit, head, tile range inside the unit).
  // Producer and compute warps walk the same way.
  auto pieces = [&](auto&& f) {
    int entry = share.entry, base = share.base, at = first_tile;
    while (at < last_tile) {
      const Kv4Unit u = kv4_unit<C>(p, entry);
      const int end = base + u.tiles * p.Hkv;
      while (at < end && at < last_tile) {
        const int h = (at - base) / u.tiles;
        const int t0 = (at - base) - h * u.tiles;
        const int t1 = min(u.tiles, t0 + (last_tile - at));
        f(u, h, t0, t1);
        at += t1 - t0;
      }
      base = end;
      ++entry;
    }
  };

  if (warp == 8) {
    // ======================= producer =======================
    if (p.no_loads) return;
    uint32_t cnt = 0;
    bool ok = true;
    const int bpp_shift = p.page_shift - 4, bpp_mask = (1 << bpp_shift) - 1;
    pieces([&](const Kv4Unit& u, int h, int t0, int t1) {
      const int* row = p.table + u.b * p.table_stride;
      // lane's page of the tile's block `lane`; the next tile's is fetched ahead
      auto page_at = [&](int tile) -> int {
        const int a = u.b0 + tile * TB + lane;
        return (tile < t1 && lane < TB && tile * TB + lane < u.nblk) ? __ldg(row + (a >> bpp_shift)) : 0;
      };
      int next = page_at(t0);
      for (int tile = t0; tile < t1; ++tile) {
        int page = next;
        next = page_at(tile + 1);
        if (page < 0 || page >= p.num_pages) {
          atomicCAS(p.status, 0, ST_KV4_PAGE);
          page = 0;  // stays in bounds; the status word tells
        }
        const int nv = min(TB, u.nblk - tile * TB);  // blocks of this tile
        const int a = u.b0 + tile * TB + lane;
        const int off = a & bpp_mask;
#pragma unroll
        for (int st4 = 0; st4 < 4; ++st4) {  // keys: two stages, values: two stages
          const int kind = st4 >> 1, half = st4 & 1;
          const int slot = cnt % NST;
          if (ok) ok = mbar_wait(EMPTY(slot), ((cnt / NST) & 1u) ^ 1u, abort_flag, p.status, ST_TIMEOUT_RING_EMPTY,
                                 p.wait_limit);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) continue;
          const int cn = min(max(nv - half * SB, 0), SB);  // blocks of this stage
          if (lane == 0) {
            if (cn > 0)
              mbar_arrive_expect_tx(FULL(slot), cn * BB);
            else
              mbar_arrive(FULL(slot));
          }
          __syncwarp();
          const int j = lane - half * SB;
          // one copy for the blocks of a page that follow each other
          if (j >= 0 && j < cn && (j == 0 || off == 0)) {
            const int run = min(bpp_mask + 1 - off, cn - j);
            const uint8_t* src = p.pages +
                                 ((((static_cast<long long>(page) * 2 + kind) * p.Hkv + h) << bpp_shift) + off) * BB;
            bulk_load(smem_u32(sRing + slot * C::STAGE_BYTES + j * BB), src, run * BB, FULL(slot));
          }
          ++cnt;
        }
      }
    });
    if (!ok) {
      // aborted: the copies in flight land before the CTA's memory goes
      for (uint32_t c = cnt > NST ? cnt - NST : 0; c < cnt; ++c) {
        const long long t0 = clock64();
        while (!mbar_try_wait(FULL(c % NST), (c / NST) & 1u) && clock64() - t0 < p.wait_limit) {
        }
      }
    }
    return;
  }

  // ======================= compute warps =======================
  const int gid = lane >> 2, tig = lane & 3;
  const int dg = warp % NG, ks = warp / NG;  // value side: dim group, slice of the blocks
  const Kv4Tops tops = p.tops;
  const uint32_t ring = smem_u32(sRing);
  const uint32_t qbase = smem_u32(sQ + gid * C::Q_PITCH + tig * 32);
  // Does row i take third bytes? 32512 * D / sAbs is its largest value over its mean.
  auto wide_row = [&](int i) { return sMost[i] > 0 && sMost[i] < 0x7F800000 && sAbs[i] < 1016 * D; };
  int slot = 0, buf = 0;  // next ring stage, P buffer
  uint32_t phase = 0;
  auto wait_at = [&](int s, uint32_t ph) {
    if (!mbar_try_wait(FULL(s), ph)) kv4_wait_slow(FULL(s), ph, abort_flag, p.status, p.wait_limit);
    __syncwarp();
  };
  auto wait_full = [&]() { wait_at(slot, phase); };
  // Gives the stage back and moves on. A warp that has nothing to read in a
  // key stage gives it back unseen: it cannot come round to the same stage
  // again before the others, there is a barrier in every tile and a tile is
  // four stages, the ring's least length.
  auto release = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(EMPTY(slot));
    if (++slot == NST) {
      slot = 0;
      phase ^= 1;
    }
  };

  pieces([&](const Kv4Unit& u, int h, int t0, int t1) {
    // ---- queries of the unit, their sums per group, the rows' key ranges
    if (threadIdx.x < 2 * ROWS) sMost[threadIdx.x] = 0;  // and sAbs: last read before the previous piece's last barrier
    compute_barrier();  // the previous piece's readers are done
    const int r0 = u.rt * ROWS, rows = p.G * u.qlen, off = u.len - u.qlen;
    constexpr int CH = D / 8, RSTEP = 256 / CH, RN = (ROWS + RSTEP - 1) / RSTEP;
    const int qc = threadIdx.x % CH, qi = threadIdx.x / CH;
    uint4 raw[RN];
#pragma unroll
    for (int k = 0; k < RN; ++k) {
      const int i = qi + k * RSTEP, r = r0 + i;
      raw[k] = make_uint4(0, 0, 0, 0);
      if (i < ROWS && r < rows) {
        const int n = r / p.G, hq = h * p.G + r - n * p.G;
        raw[k] = *reinterpret_cast<const uint4*>(p.q + u.b * p.q_sb + hq * p.q_sh + n * p.q_sn + qc * 8);
      }
    }
    auto load8 = [](const uint4& v, float (&x)[8]) {
      x[0] = unpack_lo<BF16>(v.x), x[1] = unpack_hi<BF16>(v.x);
      x[2] = unpack_lo<BF16>(v.y), x[3] = unpack_hi<BF16>(v.y);
      x[4] = unpack_lo<BF16>(v.z), x[5] = unpack_hi<BF16>(v.z);
      x[6] = unpack_lo<BF16>(v.w), x[7] = unpack_hi<BF16>(v.w);
    };
#pragma unroll
    for (int k = 0; k < RN; ++k) {
      float x[8];
      load8(raw[k], x);
      int most = 0;  // magnitudes order like their bits, infinities and NaNs last
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, static_cast<int>(__float_as_uint(x[e]) & 0x7FFFFFFFu));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      if ((qc & 7) == 0 && qi + k * RSTEP < ROWS) atomicMax(&sMost[qi + k * RSTEP], most);
    }
    compute_barrier();
#pragma unroll
    for (int k = 0; k < RN; ++k) {
      const int i = qi + k * RSTEP;
      const int bits = sMost[min(i, ROWS - 1)];
      const float most = __int_as_float(bits);
      // an integer's worth, and integers per unit: 1e-38 at least, whose reciprocal
      // is still a number (a row of zeros: its integers are 0)
      const float worth = fmaxf(most / 32512.f, 1e-38f), up = fminf(32512.f / most, 1e38f);
      float x[8];
      load8(raw[k], x);
      int v[8], third[8], sum = 0, sum3 = 0, abs = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = __float2int_rn(x[e] * up);
        third[e] = min(__float2int_rn(fmaf(x[e], up, -static_cast<float>(v[e])) * 256.f), 127);
        sum += v[e];
        sum3 += third[e];
        abs += v[e] < 0 ? -v[e] : v[e];
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        sum3 += __shfl_xor_sync(0xffffffffu, sum3, o);
        abs += __shfl_xor_sync(0xffffffffu, abs, o);
      }
      if (i < ROWS) {
        uint32_t hi[2] = {0, 0}, lo[2] = {0, 0}, lo3[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // byte order of a word's nibbles: even ones dims 0, 4, 1, 5, odd ones 2, 6, 3, 7
          const int reg = (e >> 1) & 1, byte = (e & 1) * 2 + (e >> 2);
          const int vh = (v[e] + 128) >> 8;
          hi[reg] |= (static_cast<uint32_t>(vh) & 0xFFu) << (8 * byte);
          lo[reg] |= (static_cast<uint32_t>(v[e] - (vh << 8)) & 0xFFu) << (8 * byte);
          lo3[reg] |= (static_cast<uint32_t>(third[e]) & 0xFFu) << (8 * byte);
        }
        *reinterpret_cast<uint2*>(sQ3 + i * C::Q3_PITCH + qc * 8) = make_uint2(lo3[0], lo3[1]);
        *reinterpret_cast<uint4*>(sQ + i * C::Q_PITCH + qc * 16) = make_uint4(hi[0], hi[1], lo[0], lo[1]);
        if ((qc & 7) == 0) {
          sSum[(qc >> 3) * ROWS + i] = sum;
          sSum3[(qc >> 3) * ROWS + i] = sum3;
          if (bits < 0x7F800000) atomicAdd(&sAbs[i], abs);
        }
        // a row with an infinity or a NaN has no finite scores
        if (qc == 0) sScale[i] = bits >= 0x7F800000 ? NAN : p.scale_log2 * worth;
      }
    }
    if (threadIdx.x < ROWS) {
      const int r = r0 + threadIdx.x;
      int lo = 0, hi = 0;
      if (r < rows) {
        const int pos = off + r / p.G;
        hi = p.causal ? min(u.len, pos + 1) : u.len;
        lo = (p.causal && p.window > 0) ? max(0, pos - p.window + 1) : 0;
      }
      sMask[threadIdx.x] = make_int2(lo, max(0, hi - lo));
    }
    compute_barrier();
    const bool wide = __any_sync(0xffffffffu, wide_row(lane & 7));
    // keys that every row of the unit sees: [all_lo, all_hi) (what its padding rows see is not used)
    const int nlast = (min(r0 + ROWS, rows) - 1) / p.G;
    const int any_hi = p.causal ? min(u.len, off + nlast + 1) : u.len;  // and keys that some row sees
    const int any_lo = (p.causal && p.window > 0) ? max(0, off + r0 / p.G - p.window + 1) : 0;
    const int all_hi = p.causal ? min(u.len, off + r0 / p.G + 1) : u.len;
    const int all_lo = (p.causal && p.window > 0) ? max(0, off + nlast - p.window + 1) : 0;

    float acc[4][4];
    // Rows 2 tig, 2 tig + 1: reference maximum (the same in all warps) and sum
    // of P over this warp's blocks.
    float mref[2], l_run[2];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    mref[0] = mref[1] = -INFINITY;
    l_run[0] = l_run[1] = 0.f;
    // fp16: exponent field of the largest scale so far; P and the accumulators
    // hold 2^(TOP - top) times their values.
    int top = C::BOTTOM;
    auto power = [](int e) { return __int_as_float((127 + e) << 23); };

    for (int tile = t0; tile < t1; ++tile) {
      const int nv = min(TB, u.nblk - tile * TB);
      const int key_tile = (u.b0 + tile * TB) * 16;
      // some row of the unit does not see all of the tile's keys
      const bool edge = key_tile < all_lo || key_tile + nv * 16 > all_hi;
      // ---------------- scores ----------------
      float s[KB][4];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (KB > 1 || warp / SB == half) wait_full();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          const int blk = warp + 8 * kb;
          if (blk / SB != half || blk >= nv) continue;
          const uint32_t base = ring + slot * C::STAGE_BYTES + (blk - half * SB) * BB;
          const uint32_t codes = base + lane * 16, metas = base + NG * KV4_CODE_BYTES + gid * 4;
#pragma unroll
          for (int e = 0; e < 4; ++e) s[kb][e] = 0.f;
#pragma unroll 4
          for (int g = 0; g < NG; ++g) {
            const uint4 w = lds128(codes + g * KV4_CODE_BYTES);
            const uint32_t m = lds32(metas + g * KV4_META_BYTES);  // tokens gid, gid + 8
            const float s0 = meta_scale(m << 16), s1 = meta_scale(m);
            const int z0 = m & 15, z1 = (m >> 16) & 15;
            const uint32_t xl = w.x & 0x0F0F0F0Fu, xh = (w.x >> 4) & 0x0F0F0F0Fu;  // token gid, word 2 tig
            const uint32_t yl = w.y & 0x0F0F0F0Fu, yh = (w.y >> 4) & 0x0F0F0F0Fu;  // token gid, word 2 tig + 1
            const uint32_t zl = w.z & 0x0F0F0F0Fu, zh = (w.z >> 4) & 0x0F0F0F0Fu;  // token gid + 8
            const uint32_t wl = w.w & 0x0F0F0F0Fu, wh = (w.w >> 4) & 0x0F0F0F0Fu;
            const uint32_t qa = qbase + g * 128;
            const uint4 q0 = lds128(qa), q1 = lds128(qa + 16);
            int th[4], tl[4];
            imma16832(th, xl, zl, xh, zh, q0.x, q0.y, 0, 0, 0, 0);
            imma16832(tl, xl, zl, xh, zh, q0.z, q0.w, 0, 0, 0, 0);
            imma16832(th, yl, wl, yh, wh, q1.x, q1.y, th[0], th[1], th[2], th[3]);
            imma16832(tl, yl, wl, yh, wh, q1.z, q1.w, tl[0], tl[1], tl[2], tl[3]);
            const int2 sq = *reinterpret_cast<const int2*>(sSum + g * ROWS + 2 * tig);
            float* v = s[kb];
            v[0] = fmaf(s0, static_cast<float>(th[0] * 256 + (tl[0] - z0 * sq.x)), v[0]);
            v[1] = fmaf(s0, static_cast<float>(th[1] * 256 + (tl[1] - z0 * sq.y)), v[1]);
            v[2] = fmaf(s1, static_cast<float>(th[2] * 256 + (tl[2] - z1 * sq.x)), v[2]);
            v[3] = fmaf(s1, static_cast<float>(th[3] * 256 + (tl[3] - z1 * sq.y)), v[3]);
          }
          if (wide) {
            const float w0 = wide_row(2 * tig) ? 0x1p-8f : 0.f, w1 = wide_row(2 * tig + 1) ? 0x1p-8f : 0.f;
            const uint8_t* third = sQ3 + gid * C::Q3_PITCH + tig * 16;
            const int* sums = sSum3 + 2 * tig;
            if constexpr (KB == 1) {
              kv4_third_bytes<NG>(s[kb], codes, metas, third, sums, w0, w1);
            } else {
              const float4 t = kv4_third_bytes_call<NG>(codes, metas, third, sums, w0, w1);
              s[kb][0] += t.x;
              s[kb][1] += t.y;
              s[kb][2] += t.z;
              s[kb][3] += t.w;
            }
          }
        }
        release();
      }

      // fp16: this thread's word (four tokens) of the tile's value scales; the
      // loads are under way during the softmax
      const int scale_blk = threadIdx.x / (NG * 4);
      const uint32_t limit = top * 0x00800080u + 0x007F007Fu;
      uint2 mv = make_uint2(0, 0);
      if constexpr (!BF16) {
        static_assert(TB * NG * 4 <= 256, "a word per thread");
        const int slot1 = slot + 1 == NST ? 0 : slot + 1;
        wait_full();
        wait_at(slot1, slot1 == 0 ? phase ^ 1 : phase);
        if (scale_blk < nv)
          mv = lds64(ring + (scale_blk < SB ? slot : slot1) * C::STAGE_BYTES + scale_blk % SB * BB +
                     NG * KV4_CODE_BYTES + threadIdx.x % (NG * 4) * 8);
      }

      // ---------------- softmax over this warp's blocks ----------------
      float* P = sP + buf * (C::P_BYTES / 4);
      float* M = sM + buf * 8 * ROWS;
      bool above = false;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int blk = warp + 8 * kb;
        if (blk >= nv) continue;
        float* v = s[kb];
        const float2 sc = *reinterpret_cast<const float2*>(sScale + 2 * tig);
        v[0] *= sc.x;
        v[1] *= sc.y;
        v[2] *= sc.x;
        v[3] *= sc.y;
        if (edge) {
          const int4 mk = *reinterpret_cast<const int4*>(sMask + 2 * tig);  // two rows' (first, count)
          const int key = key_tile + blk * 16 + gid;
          if (static_cast<unsigned>(key - mk.x) >= static_cast<unsigned>(mk.y)) v[0] = -INFINITY;
          if (static_cast<unsigned>(key - mk.z) >= static_cast<unsigned>(mk.w)) v[1] = -INFINITY;
          if (static_cast<unsigned>(key + 8 - mk.x) >= static_cast<unsigned>(mk.y)) v[2] = -INFINITY;
          if (static_cast<unsigned>(key + 8 - mk.z) >= static_cast<unsigned>(mk.w)) v[3] = -INFINITY;
        }
        above |= fmaxf(v[0], v[2]) > mref[0] + C::SLACK || fmaxf(v[1], v[3]) > mref[1] + C::SLACK;
      }
      bool raise, larger = false;
      int mytop = top;
      if constexpr (BF16) {
        raise = __any_sync(0xffffffffu, above);
      } else {
        raise = __any_sync(0xffffffffu, above || max2_u16(max2_u16(mv.x, mv.y), limit) != limit);
        if (raise) {
          raise = __any_sync(0xffffffffu, above);
          const uint32_t word[4] = {mv.x & 0xFFFFu, mv.x >> 16, mv.y & 0xFFFFu, mv.y >> 16};
          const int key0 = key_tile + scale_blk * 16 + (threadIdx.x & 3) * 2;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = key0 + (j & 1) + (j >> 1) * 8;
            // not a NaN's, nor that of a token that no row sees (which may be anything)
            if (word[j] < 0x7F80u && (!edge || (key >= any_lo && key < any_hi)))
              mytop = max(mytop, static_cast<int>(word[j] >> 7));
          }
          mytop = min(__reduce_max_sync(0xffffffffu, mytop), C::TOP);
          larger = mytop != top;
        }
      }
      // bit 0: a maximum is published; fp16: above it, the largest scale's exponent field
      if (lane == 0) raised[buf][warp] = BF16 ? raise : 2 * mytop + raise;
      const int perm = (gid >> 1) * 4 + (gid & 1);  // order (2t, 2t+1, 2t+8, 2t+9) of the value side
      float f0 = mref[0], f1 = mref[1];
      if (raise) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          if (warp + 8 * kb >= nv) continue;
          f0 = fmaxf(f0, fmaxf(s[kb][0], s[kb][2]) + C::RAISE);
          f1 = fmaxf(f1, fmaxf(s[kb][1], s[kb][3]) + C::RAISE);
        }
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          f0 = fmaxf(f0, __shfl_xor_sync(0xffffffffu, f0, o));
          f1 = fmaxf(f1, __shfl_xor_sync(0xffffffffu, f1, o));
        }
        l_run[0] *= ex2(mref[0] - finite_or_zero(f0));
        l_run[1] *= ex2(mref[1] - finite_or_zero(f1));
        if (gid == 0) *reinterpret_cast<float2*>(M + warp * ROWS + 2 * tig) = make_float2(f0, f1);
      }
      f0 = finite_or_zero(f0);
      f1 = finite_or_zero(f1);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int blk = warp + 8 * kb;
        if (blk >= nv) continue;
        float* v = s[kb];
        bool seen[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) seen[e] = v[e] != -INFINITY;
        v[0] = ex2(v[0] - f0);
        v[1] = ex2(v[1] - f1);
        v[2] = ex2(v[2] - f0);
        v[3] = ex2(v[3] - f1);
        if (edge) {  // P = 0 marks a masked key: one that is seen has at least the least normal number
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (seen[e] && v[e] == 0.f) v[e] = 1.17549435e-38f;
        }
        l_run[0] += v[0] + v[2];
        l_run[1] += v[1] + v[3];
        if constexpr (!BF16) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= power(C::TOP - mytop);
        }
        float* d = P + (blk * ROWS + 2 * tig) * PP + perm;
        d[0] = v[0];
        d[2] = v[2];
        d[PP] = v[1];
        d[PP + 2] = v[3];
      }
      // ---------------- new maxima, if any warp published some ----------------
      const bool rescale = compute_barrier_or(raise || larger);
      // A warp's P refers to its own published maximum, or to the old one: in
      // the value loop row gid's factor brings it to the new one.
      float vold = 0.f, vnew = 0.f;
      int newtop = top;
      if (rescale) {
        float m0 = mref[0], m1 = mref[1];
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          if (!BF16) newtop = max(newtop, raised[buf][w] >> 1);
          if (raised[buf][w] & 1) {
            const float2 x = *reinterpret_cast<const float2*>(M + w * ROWS + 2 * tig);
            m0 = fmaxf(m0, x.x);
            m1 = fmaxf(m1, x.y);
          }
        }
        float2 mine = make_float2(mref[0], mref[1]);
        if (raise) mine = *reinterpret_cast<const float2*>(M + warp * ROWS + 2 * tig);
        l_run[0] *= ex2(mine.x - finite_or_zero(m0));
        l_run[1] *= ex2(mine.y - finite_or_zero(m1));
        float a0 = ex2(mref[0] - finite_or_zero(m0)), a1 = ex2(mref[1] - finite_or_zero(m1));
        if constexpr (!BF16) {
          a0 *= power(top - newtop);
          a1 *= power(top - newtop);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[j][0] *= a0;
          acc[j][1] *= a1;
          acc[j][2] *= a0;
          acc[j][3] *= a1;
        }
        // row gid belongs to lanes with tig = gid / 2
        const float o0 = __shfl_sync(0xffffffffu, mref[0], gid >> 1), o1 = __shfl_sync(0xffffffffu, mref[1], gid >> 1);
        const float n0 = __shfl_sync(0xffffffffu, m0, gid >> 1), n1 = __shfl_sync(0xffffffffu, m1, gid >> 1);
        vold = (gid & 1) ? o1 : o0;
        vnew = finite_or_zero((gid & 1) ? n1 : n0);
        mref[0] = m0;
        mref[1] = m1;
        top = newtop;
      }

      // ---------------- values ----------------
      float wz[4];  // -sum (F + z) P' of this tile
#pragma unroll
      for (int e = 0; e < 4; ++e) wz[e] = 0.f;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        if (BF16) wait_full();  // fp16: before the barrier
        const uint32_t stage = ring + slot * C::STAGE_BYTES;
        const uint32_t codes = stage + dg * KV4_CODE_BYTES + (tig * 8 + (gid ^ (2 * tig))) * 16;
        const uint32_t metas = stage + NG * KV4_CODE_BYTES + dg * KV4_META_BYTES + tig * 8;
        const float* prow = P + (half * SB * ROWS + gid) * PP + tig * 4;
        auto block = [&](int sblk, auto special) {
          constexpr bool SPECIAL = decltype(special)::value;
          const uint2 mv = lds64(metas + sblk * BB);
          const uint4 c = lds128(codes + sblk * BB);
          uint32_t x0[4], x1[4], x2[4], x3[4];  // nibbles 0..3 and 4..7, tokens (2t, 2t+1) and (2t+8, 2t+9)
          codes16<BF16>(__byte_perm(c.x, c.y, 0x5410), tops, x0);
          codes16<BF16>(__byte_perm(c.x, c.y, 0x7632), tops, x1);
          codes16<BF16>(__byte_perm(c.z, c.w, 0x5410), tops, x2);
          codes16<BF16>(__byte_perm(c.z, c.w, 0x7632), tops, x3);
          const float s0 = meta_scale(mv.x << 16), s1 = meta_scale(mv.x), s2 = meta_scale(mv.y << 16),
                      s3 = meta_scale(mv.y);
          float4 pr = *reinterpret_cast<const float4*>(prow + sblk * ROWS * PP);
          if constexpr (SPECIAL) {
            const bool off0 = edge && pr.x == 0.f, off1 = edge && pr.y == 0.f;  // masked
            const bool off2 = edge && pr.z == 0.f, off3 = edge && pr.w == 0.f;
            if (rescale) {
              const int w = (half * SB + sblk) & 7;
              const float from = (raised[buf][w] & 1) ? M[w * ROWS + gid] : vold;
              float f = ex2(finite_or_zero(from) - vnew);
              if (!BF16) f *= power((raised[buf][w] >> 1) - newtop);
              pr.x *= f;
              pr.y *= f;
              pr.z *= f;
              pr.w *= f;
            }
            // a masked token's scale may be anything (a slot never written): its product must be 0
            pr.x = off0 ? 0.f : pr.x * s0;
            pr.y = off1 ? 0.f : pr.y * s1;
            pr.z = off2 ? 0.f : pr.z * s2;
            pr.w = off3 ? 0.f : pr.w * s3;
          } else {
            pr.x *= s0;
            pr.y *= s1;
            pr.z *= s2;
            pr.w *= s3;
          }
          const uint32_t b0 = pack2<BF16>(pr.x, pr.y), b1 = pack2<BF16>(pr.z, pr.w);
          mma16816<BF16>(acc[0], x0[0], x0[1], x2[0], x2[1], b0, b1);
          mma16816<BF16>(acc[1], x0[2], x0[3], x2[2], x2[3], b0, b1);
          mma16816<BF16>(acc[2], x1[0], x1[1], x3[0], x3[1], b0, b1);
          mma16816<BF16>(acc[3], x1[2], x1[3], x3[2], x3[3], b0, b1);
          mma16816<BF16>(wz, minus_zero_even<BF16>(mv.x, tops), minus_zero_odd<BF16>(mv.x, tops),
                         minus_zero_even<BF16>(mv.y, tops), minus_zero_odd<BF16>(mv.y, tops), b0, b1);
        };
        if (!rescale && !edge && nv == TB) {
#pragma unroll(SB / KS > 4 ? 4 : SB / KS)
          for (int i = 0; i < SB / KS; ++i) block(i * KS + ks, std::false_type{});
        } else {
#pragma unroll 1
          for (int i = 0; i < SB / KS; ++i) {
            if (half * SB + i * KS + ks >= nv) break;
            block(i * KS + ks, std::true_type{});
          }
        }
        release();
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] += wz[e];
      buf ^= 1;
    }

    // ---------------- epilogue of the piece ----------------
    if constexpr (!BF16) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] *= power(top - C::TOP);
    }
    // every warp has the rows' maximum; the sums of the eight warps' l
    compute_barrier();  // all value-side reads of P and M are done
    float* xM = sM;             // [ROWS] maxima
    float* xL = sM + 8 * ROWS;  // [8][ROWS] sums
    float l0 = l_run[0], l1 = l_run[1];
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    if (gid == 0) {
      if (warp == 0) *reinterpret_cast<float2*>(xM + 2 * tig) = make_float2(mref[0], mref[1]);
      *reinterpret_cast<float2*>(xL + warp * ROWS + 2 * tig) = make_float2(l0, l1);
    }
    // value-side slices: halve their number until one is left
    if constexpr (KS > 1) {
#pragma unroll
      for (int live = KS / 2; live >= 1; live >>= 1) {
        float* X = sP;
        const int lane_at = ((dg * live + (ks % live)) * 32 + lane) * 4;
        if (ks >= live && ks < 2 * live) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4*>(X + j * (NG * live * 128) + lane_at) =
                make_float4(acc[j][0], acc[j][1], acc[j][2], acc[j][3]);
        }
        compute_barrier();
        if (ks < live) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 v = *reinterpret_cast<const float4*>(X + j * (NG * live * 128) + lane_at);
            acc[j][0] += v.x;
            acc[j][1] += v.y;
            acc[j][2] += v.z;
            acc[j][3] += v.w;
          }
        }
        compute_barrier();
      }
    } else {
      compute_barrier();
    }
    const bool whole = t0 == 0 && t1 == u.tiles;
    const int part = 2 * blockIdx.x + (t0 == 0 ? 1 : 0);  // a unit's later parts start a share
    if (ks == 0) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {  // rows 2 tig, 2 tig + 1
        const int i = 2 * tig + e, r = r0 + i;
        const float m = xM[i];
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) l += xL[w * ROWS + i];
        // dims 64 dg + 8 gid + (0..7): MMA rows gid and gid + 8 of tile j are dims 2j and 2j + 1
        if (whole) {
          if (r < rows) {
            const float inv = l == 0.f ? 0.f : 1.f / l;  // no key seen: zeros
            const int n = r / p.G, hq = h * p.G + r - n * p.G;
            uint4 v;
            v.x = pack2<BF16>(acc[0][e] * inv, acc[0][2 + e] * inv);
            v.y = pack2<BF16>(acc[1][e] * inv, acc[1][2 + e] * inv);
            v.z = pack2<BF16>(acc[2][e] * inv, acc[2][2 + e] * inv);
            v.w = pack2<BF16>(acc[3][e] * inv, acc[3][2 + e] * inv);
            *reinterpret_cast<uint4*>(p.o + u.b * p.o_sb + hq * p.o_sh + n * p.o_sn + dg * 64 + gid * 8) = v;
            if (p.lse && dg == 0 && gid == 0)
              p.lse[(static_cast<long long>(u.b) * p.Hq + hq) * p.N + n] =
                  l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
          }
        } else {
          float* d = p.part_o + (static_cast<long long>(part) * ROWS + i) * D + dg * 64 + gid * 8;
          *reinterpret_cast<float4*>(d) = make_float4(acc[0][e], acc[0][2 + e], acc[1][e], acc[1][2 + e]);
          *reinterpret_cast<float4*>(d + 4) = make_float4(acc[2][e], acc[2][2 + e], acc[3][e], acc[3][2 + e]);
          if (dg == 0 && gid == 0) p.part_ml[static_cast<long long>(part) * ROWS + i] = make_float2(m, l);
        }
      }
    }
  });
}

// Joins the parts of units that several CTAs worked on, and writes zeros for
// rows that no unit covers (no token, or no key to see): join_blocks CTAs per
// unit, each a slice of its [rows][D] output, every lane four neighbouring
// floats. Where a slice is narrower than the CTA, groups of warps take every
// n-th part and are added up in order at the end; four parts are in flight per
// warp, so a unit cut into 148 parts takes a few memory latencies.
template <class C>
__global__ void __launch_bounds__(512, 2) kv4_combine_kernel(const Kv4Params p) {
  constexpr int D = C::D, ROWS = C::ROWS;
  __shared__ float4 sAcc[16][32];
  __shared__ float2 sMl[16][32];
  __shared__ int scratch[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int unit = blockIdx.x / p.join_blocks, slice = blockIdx.x - unit * p.join_blocks;
  const int entry = unit / p.Hkv, h = unit - entry * p.Hkv;
  // Where the unit lies in the list of tiles. This reads the lengths only,
  // which the attention launch does not write: it may run beside it.
  const int entries = p.B * p.row_tiles;
  int before = 0, total = 0;
  for (int e = threadIdx.x; e < entries; e += 512) {
    const int t = kv4_unit<C>(p, e).tiles * p.Hkv;
    total += t;
    if (e < entry) before += t;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  total = __reduce_add_sync(0xffffffffu, total);
  if (lane == 0) {
    scratch[warp] = before;
    scratch[16 + warp] = total;
  }
  __syncthreads();
  before = __reduce_add_sync(0xffffffffu, lane < 16 ? scratch[lane] : 0);
  total = __reduce_add_sync(0xffffffffu, lane < 16 ? scratch[16 + lane] : 0);
  const Kv4Unit u = kv4_unit<C>(p, entry);
  const int per = max(1, (total + p.ctas - 1) / p.ctas);
  const int begin = before + h * u.tiles;
  const int c0 = begin / per, c1 = u.tiles == 0 ? c0 : (begin + u.tiles - 1) / per;
  const int limit = min(ROWS, p.G * p.N - u.rt * ROWS);                      // rows of the output
  const int rows = u.tiles == 0 ? 0 : min(limit, p.G * u.qlen - u.rt * ROWS);  // of them with keys
  if (slice == 0 && h == 0 && threadIdx.x == 0 && p.kv_lens[u.b] > (p.cols << p.page_shift))
    atomicCAS(p.status, 0, ST_KV4_LENGTH);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (c0 == c1 && rows == limit) return;  // written by its one CTA
  // columns of 128 floats; the slice's are [first, first + columns)
  const int columns = (ROWS * D / 128) / p.join_blocks, first = slice * columns;
  const int groups = columns < 16 ? 16 / columns : 1;  // warps per column
  // part of CTA c: its share's first piece unless the unit starts there
  auto part_of = [&](int c) { return static_cast<long long>(2 * c + (c == c0 ? 1 : 0)); };
  for (int k = warp / groups; k < columns; k += 16 / groups) {
    const int at = ((first + k) * 32 + lane) * 4, i = at / D, d = at - i * D;
    const int grp = warp % groups;
    float m = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < rows && c0 < c1) {
      constexpr int U = 4;  // parts in flight
#pragma unroll 1
      for (int c = c0 + grp; c <= c1; c += U * groups) {
        float2 q[U];
        float4 v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
          const long long row = part_of(min(c + j * groups, c1)) * ROWS + i;
          q[j] = __ldcg(p.part_ml + row);
          v[j] = __ldcg(reinterpret_cast<const float4*>(p.part_o + row * D + d));
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          if (c + j * groups > c1) q[j] = make_float2(-INFINITY, 0.f);
          top = fmaxf(top, q[j].x);
        }
        const float ft = finite_or_zero(top), f0 = ex2(m - ft);
        m = top;
        l *= f0;
        a.x *= f0, a.y *= f0, a.z *= f0, a.w *= f0;
#pragma unroll
        for (int j = 0; j < U; ++j) {
          if (c + j * groups <= c1) {
            const float f = ex2(q[j].x - ft);
            l = fmaf(q[j].y, f, l);
            a.x = fmaf(v[j].x, f, a.x);
            a.y = fmaf(v[j].y, f, a.y);
            a.z = fmaf(v[j].z, f, a.z);
            a.w = fmaf(v[j].w, f, a.w);
          }
        }
      }
    }
    if (groups > 1) {  // then every warp has exactly one column
      sAcc[warp][lane] = a;
      sMl[warp][lane] = make_float2(m, l);
      __syncthreads();
      if (grp != 0) return;
      float top = m;
      for (int w = 1; w < groups; ++w) top = fmaxf(top, sMl[warp + w][lane].x);
      const float ft = finite_or_zero(top), f0 = ex2(m - ft);
      m = top;
      l *= f0;
      a.x *= f0, a.y *= f0, a.z *= f0, a.w *= f0;
      for (int w = 1; w < groups; ++w) {
        const float2 q = sMl[warp + w][lane];
        const float4 v = sAcc[warp + w][lane];
        const float f = ex2(q.x - ft);
        l = fmaf(q.y, f, l);
        a.x = fmaf(v.x, f, a.x);
        a.y = fmaf(v.y, f, a.y);
        a.z = fmaf(v.z, f, a.z);
        a.w = fmaf(v.w, f, a.w);
      }
    }
    if (i < limit && (i >= rows || c0 < c1)) {
      const int r = u.rt * ROWS + i, n = r / p.G, hq = h * p.G + r - n * p.G;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      *reinterpret_cast<uint2*>(p.o + u.b * p.o_sb + hq * p.o_sh + n * p.o_sn + d) =
          make_uint2(pack2<C::BF16>(a.x * inv, a.y * inv), pack2<C::BF16>(a.z * inv, a.w * inv));
      if (p.lse && d == 0)
        p.lse[(static_cast<long long>(u.b) * p.Hq + hq) * p.N + n] =
            l == 0.f ? -INFINITY : (m + __log2f(l)) * 0.6931471805599453f;
    }
  }
}

}  // namespace gqafa
