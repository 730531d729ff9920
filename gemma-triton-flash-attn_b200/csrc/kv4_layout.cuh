// The paged 4-bit KV cache: number format and memory layout.
//
// Number format. A group is 64 consecutive values along head_dim of one token
// of one head. It is held as value = s * (c - z): a 4-bit code c per value, a
// zero point z in 0..15 and a scale s with 4 significant bits per group. c - z
// has at most 4 bits, so every value has at most 8 significant bits: it is
// exact in bf16 and in fp16, and reading the cache rounds nothing. Per group
// 32 bytes of codes and one 16-bit word: the bf16 pattern of s, whose low 4
// mantissa bits are zero, with z in their place (4.25 bits a value).
//
// Quantisation of 16-bit values x (all steps exact or correctly rounded in
// fp32, and no input lies so near a rounding border that fp32 and real
// arithmetic differ):
//   hi = max(0, max x), lo = min(0, min x)
//   s  = (hi/2 - lo/2) / 7.5 rounded up to 4 significant bits, at least
//        2^-126 (bf16) or 2^-21 (fp16: s's last bit is then 2^-24)
//   z  = floor(-lo/s + 1/2)
//   c  = min(15, floor(x/s + 1/2) + z); a code whose value would pass the
//        type's largest finite number moves one step towards z
// A group that holds an infinity or a NaN gets s = NaN: it reads back as NaN.
//
// Layout. Sixteen tokens of one head form a block: for each group 512 bytes of
// codes, then for each group 32 bytes of meta words (544 * head_dim/64 bytes).
// A page holds page_size/16 blocks of every head, keys and then values:
// [page][2][head][block]. Codes lie in the order in which an m16n8k16 MMA's
// A fragment takes them, so that a warp reads one group's codes of a block
// with one conflict-free 16-byte load per lane:
//   keys   (A rows = tokens, contraction = head_dim): lane 4*(r%8) + t holds
//          words 2t, 2t+1 of token r%8 and of token r%8 + 8. Word j covers
//          dims 8j..8j+7; nibble i holds dim 8j+2i, nibble 4+i dim 8j+2i+1, so
//          a nibble pair (i, i+4) is one 16-bit pair of neighbouring dims.
//   values (A rows = head_dim, contraction = tokens): 16-byte piece
//          8t + (j ^ 2t) holds word j (dims 8j..8j+7, lowest nibble first) of
//          tokens 2t, 2t+1, 2t+8, 2t+9; the XOR spreads the eight lanes of a
//          load phase over all banks.
// Meta words: keys in order (0, 8, 1, 9, ...), values in order
// (0, 1, 8, 9, 2, 3, 10, 11, ...).
#pragma once
#include <cstdint>

namespace gqafa {

constexpr int KV4_GROUP = 64;        // values per scale
constexpr int KV4_TOKENS = 16;       // tokens per block
constexpr int KV4_CODE_BYTES = 512;  // codes of one group of a block
constexpr int KV4_META_BYTES = 32;   // meta words of one group of a block

__host__ __device__ constexpr int kv4_block_bytes(int head_dim) {
  return head_dim / KV4_GROUP * (KV4_CODE_BYTES + KV4_META_BYTES);
}
// Byte offset of code word j (0..7) of token r (0..15) inside a group's codes.
__host__ __device__ constexpr int kv4_key_word(int r, int j) {
  return ((r & 7) * 4 + (j >> 1)) * 16 + (r >> 3) * 8 + (j & 1) * 4;
}
__host__ __device__ constexpr int kv4_value_word(int r, int j) {
  return (((r & 7) >> 1) * 8 + (j ^ (((r & 7) >> 1) * 2))) * 16 + ((r >> 3) * 2 + (r & 1)) * 4;
}
// Index of token r's 16-bit meta word inside a group's.
__host__ __device__ constexpr int kv4_key_meta(int r) { return (r & 7) * 2 + (r >> 3); }
__host__ __device__ constexpr int kv4_value_meta(int r) { return ((r & 7) >> 1) * 4 + (r >> 3) * 2 + (r & 1); }

constexpr uint16_t KV4_META_NAN = 0x7FF0;  // scale of a group with a non-finite value

// Codes of the status word that the cache's kernels may record beside the wait
// codes: a page outside the pool, a slot outside the cache, a length beyond
// the block table. Such entries are skipped or clamped, never followed.
enum Kv4Status : int { ST_KV4_PAGE = 16, ST_KV4_SLOT = 17, ST_KV4_LENGTH = 18 };

}  // namespace gqafa
