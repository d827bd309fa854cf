// The key / value cache of 4-bit codes: where everything lies (kv4_cache.hip writes and reads it, kv4_attention.hip attends over it).
//
// A group of `group` channels (32, 64 or 128) of one token is 4-bit codes and one 16-bit word, value = scale * (code - zero):
// the word holds the scale's bits as a half of 7 significant bits (low 4 bits clear) and the zero point, 0..15, in those 4.
// (code - zero) has at most 4 significant bits, so every value is a half exactly (11 bits): dequantization rounds nothing, whichever
// kernel does it and in whatever order, and a group costs 2 bytes where a scale and a minimum would cost 4.
//
// cache = [pages][kv_heads][block]; a block holds one head's `page` tokens: codes of the keys, codes of the values, words of the keys,
// words of the values.  All four are runs of tiles of 16 tokens, the tokens of one matrix instruction:
//   key codes    [tile][plane][token 16][quarter 4][word][8 nibbles]     channel = plane * PLANE + 32 word + 8 quarter + nibble
//                a lane of a 16x16x32 product (token, quarter) reads its operands of all the plane's products as one piece
//   value codes  [tile][plane][token quad 4][cell 16][PLANE / 64][pair 2][token of the pair 2][4 nibbles]
//                channel = plane * PLANE + cell * PLANE / 16 + 4 * (third index) + nibble, token = 4 quad + 2 pair + (token of the pair):
//                a lane (cell, quad) reads its four tokens of all its channels as one piece, tokens in pairs as a packed half operation wants
//                them; the four tokens of a quad are those whose probabilities the lane holds after the first product
//   words        [tile][group][token 16]
// PLANE = min(head_dim, 128) channels, so that a piece is 16 bytes (8 where head_dim is 64).
#ifndef MLDHIP_CSRC_KV4_H_
#define MLDHIP_CSRC_KV4_H_

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kernels.h"

namespace mldhip {

constexpr float kKv4Largest = 57344.0f;  // inputs are held to +-this: scale * 15 of the widest group stays a finite half
constexpr int kKv4Tile = 16;

__host__ __device__ constexpr int Kv4Plane(int head_dim) { return head_dim < 128 ? head_dim : 128; }
__host__ __device__ constexpr size_t Kv4BlockBytes(int page, int head_dim, int groups) {
  return (size_t)page * head_dim + (size_t)4 * page * groups;
}
// Byte offsets inside a block
__host__ __device__ constexpr int Kv4ValueCodes(int page, int head_dim) { return page * head_dim / 2; }
__host__ __device__ constexpr int Kv4KeyWords(int page, int head_dim) { return page * head_dim; }
__host__ __device__ constexpr int Kv4ValueWords(int page, int head_dim, int groups) { return page * head_dim + 2 * page * groups; }

// The rows of sequence s: row `start` + i (i < count) is position first + i; positions 0 .. held - 1 are in the cache.
// Whatever the device arrays hold, rows stay inside the tensors and positions inside the table.
struct Kv4Sequence {
  int start, count, first, held;
};
__host__ __device__ constexpr int Kv4Within(int v, int low, int high) { return v < low ? low : v > high ? high : v; }
__host__ __device__ constexpr Kv4Sequence Kv4SequenceFrom(int from, int to, int length, int tokens, int pages_per_sequence, int page_shift) {
  Kv4Sequence q{};
  q.start = Kv4Within(from, 0, tokens);
  q.count = Kv4Within(to, q.start, tokens) - q.start;  // (both ends in range first: a difference of what the arrays hold may overflow)
  length = Kv4Within(length, 0, 1 << 30);
  q.first = length - q.count;
  const long long room = (long long)pages_per_sequence << page_shift;
  q.held = length < room ? length : (int)room;
  return q;
}
__device__ __forceinline__ Kv4Sequence Kv4SequenceOf(const Kv4Where& w, int s) {
  return Kv4SequenceFrom(w.starts[s], w.starts[s + 1], w.lengths[s], w.tokens, w.pages_per_sequence, w.page_shift);
}

}  // namespace mldhip

#endif  // MLDHIP_CSRC_KV4_H_
