// Writing new keys and values into the cache of 4-bit codes and reading cached ones back (kv4.h: the layout).
//
// A group of G channels x of one token, lo = min(x, 0), hi = max(x, 0):
//   scale = the smallest half of 7 significant bits with 15 * scale >= hi - lo,  zero = rint(-lo / scale),
//   code = min(max(rint(x / scale) + zero, 0), 15),  value = scale * (code - zero);  rint: ties to even.
// All of it is exact: the span in fp64, the quotients by a product with the approximate reciprocal and one exact correction, so that the
// codes do not depend on how a division rounds.  Inputs are held to +-57344 and NaN counts as 0: a cached value is always a finite half,
// and a masked position can never turn a product into NaN.
//
// A wave is 16 tokens (one tile of the cache, so that a tile's bytes are written by one wave) x 4 lanes that share a head of a token, each
// with head_dim / 4 neighbouring channels.  Memory bounds it: tensors of 2 or 4 bytes a channel against 0.53 .. 0.56.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "kernels.h"
#include "kv4.h"

#pragma clang fp contract(off)

namespace mldhip {
namespace {

__device__ __forceinline__ float Held(float x) { return x != x ? 0.0f : fminf(fmaxf(x, -kKv4Largest), kKv4Largest); }

// The smallest half of 7 significant bits (a multiple of 2^-20 at the small end) with 15 * scale >= span.
__device__ __forceinline__ uint32_t ScaleBits(double span) {
  const float r = (float)(span * (1.0 / 15.0));
  // an estimate at most one step off: r's bits as a half's, without the low 4, rounded down
  const uint32_t bits = r < 0x1p-14f ? (uint32_t)(r * 0x1p20f) << 4 : ((__float_as_uint(r) >> 13) - (112u << 10)) & 0xFFF0u;
  uint32_t b = bits > 16u ? bits - 16u : 0u;
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (15.0 * (double)__half2float(__ushort_as_half((unsigned short)b)) < span) b += 16u;
  return b;
}

// rint(x / s), ties to even, exactly: |x / s| < 2^10, s a half of 7 significant bits.  r * s is exact in fp32 (10 + 7 bits) and so is
// x - r * s for an r next to the quotient (a multiple of x's last place that is at most a few s).
__device__ __forceinline__ float RoundedQuotient(float x, float s, float inv) {
  const float r = rintf(x * inv);
  const float left = fmaf(-r, s, x), half = 0.5f * s;
  const bool odd = ((int)r & 1) != 0;
  if (left > half || (left == half && odd)) return r + 1.0f;
  if (left < -half || (left == -half && odd)) return r - 1.0f;
  return r;
}

template <typename T>
struct Slice;
template <>
struct Slice<__half> {
  using type = uint2;
};
template <>
struct Slice<float> {
  using type = float4;
};
__device__ __forceinline__ void Load4(const uint2& raw, float v[4]) {
  const __half2 lo = __builtin_bit_cast(__half2, raw.x), hi = __builtin_bit_cast(__half2, raw.y);
  v[0] = __low2float(lo);
  v[1] = __high2float(lo);
  v[2] = __low2float(hi);
  v[3] = __high2float(hi);
}
__device__ __forceinline__ void Load4(const float4& raw, float v[4]) {
  v[0] = raw.x;
  v[1] = raw.y;
  v[2] = raw.z;
  v[3] = raw.w;
}
__device__ __forceinline__ void Store4(uint2* p, const float v[4]) {  // (every value is a half: nothing is rounded)
  uint2 raw;
  raw.x = __builtin_bit_cast(uint32_t, __floats2half2_rn(v[0], v[1]));
  raw.y = __builtin_bit_cast(uint32_t, __floats2half2_rn(v[2], v[3]));
  *p = raw;
}
__device__ __forceinline__ void Store4(float4* p, const float v[4]) { *p = make_float4(v[0], v[1], v[2], v[3]); }

// Byte offsets inside a tile's codes: of the word of 8 key channels from `channel` on, of the 2 bytes of 4 value channels.
template <int D>
__device__ __forceinline__ int KeyWordAt(int token, int channel) {
  constexpr int P = Kv4Plane(D);
  const int i = channel % P;
  return channel / P * (8 * P) + (token * 4 + i % 32 / 8) * (P / 8) + i / 32 * 4;
}
template <int D>
__device__ __forceinline__ int ValuePairAt(int token, int channel) {
  constexpr int P = Kv4Plane(D), kCell = P / 16;
  const int i = channel % P;
  return channel / P * (8 * P) + (token / 4 * 16 + i / kCell) * (2 * kCell) + i % kCell / 4 * 8 + token % 4 * 2;
}

// What a wave works on: 16 positions of a sequence and one head of the keys or the values.
struct Tile {
  bool inside;     // the lane's token is one of the sequence's new rows, at a position of a page that there is
  bool row_only;   // it is a row, but its position is on no page
  int row;         // of the tensors
  int in_page;     // first token of the tile in its page
  uint8_t* block;  // the page's block of this head
};
__device__ __forceinline__ Tile TileOf(const Kv4Where& w, const Kv4Sequence& q, int s, int tile, int head, int token, const uint8_t* cache) {
  Tile r;
  const int position = tile * kKv4Tile + token;
  const int i = position - q.first;
  const bool is_row = i >= 0 && i < q.count;
  r.row = q.start + i;
  int page = -1;
  if (tile >= 0 && tile * kKv4Tile < q.held) page = w.table[(size_t)s * w.pages_per_sequence + (tile * kKv4Tile >> w.page_shift)];
  const bool there = page >= 0 && page < w.pages && position < q.held;
  r.inside = is_row && there;
  r.row_only = is_row && !there;
  r.in_page = (tile * kKv4Tile) & ((1 << w.page_shift) - 1);
  r.block = const_cast<uint8_t*>(cache) + ((size_t)(there ? page : 0) * w.kv_heads + head) * w.block_bytes;
  return r;
}

// Grid: tiles of a sequence's new rows x (head, keys or values) x sequences; a work-group of 4 waves takes 4 tiles, then those
// 4 * gridDim.x on (more rows than the op was made for only take longer).
template <typename T, int D, bool READ>
__global__ __launch_bounds__(256) void kv4_move_kernel(const Kv4MoveArgs p) {
  using Raw = typename Slice<T>::type;
  constexpr int kMine = D / 4;  // channels of a lane
  const Kv4Where& w = p.where;
  const int lane = threadIdx.x & 63, token = lane & 15, quarter = lane >> 4;
  const bool is_value = blockIdx.y & 1;
  const int head = blockIdx.y >> 1, s = blockIdx.z;
  const Kv4Sequence q = Kv4SequenceOf(w, s);
  if (q.count == 0) return;
  const int page_tokens = 1 << w.page_shift, groups = D >> w.group_shift, group = 1 << w.group_shift;
  const int codes_at = is_value ? Kv4ValueCodes(page_tokens, D) : 0;
  const int words_at = is_value ? Kv4ValueWords(page_tokens, D, groups) : Kv4KeyWords(page_tokens, D);
  const int tile_begin = q.first >> 4, tile_end = (q.first + q.count + 15) >> 4;  // (first may be negative: rows without a position)
  Raw* tensor = static_cast<Raw*>(is_value ? p.v : p.k) + (size_t)(head * D + quarter * kMine) / 4 * w.tokens;
  for (int tile = tile_begin + (int)(blockIdx.x * 4 + (threadIdx.x >> 6)); tile < tile_end; tile += gridDim.x * 4) {
    const Tile at = TileOf(w, q, s, tile, head, token, static_cast<const uint8_t*>(p.cache));
    uint8_t* codes = at.block + codes_at + (size_t)at.in_page * (D / 2);
    uint16_t* words = reinterpret_cast<uint16_t*>(at.block + words_at) + at.in_page * groups + token;  // [group][16]
    if constexpr (READ) {
      if (!at.inside && !at.row_only) continue;
#pragma unroll
      for (int c = 0; c < kMine; c += 8) {
        const int channel = quarter * kMine + c;
        float v[2][4] = {};
        if (at.inside) {
          const uint32_t word = words[(channel >> w.group_shift) * 16];
          const float scale = __half2float(__ushort_as_half((unsigned short)(word & 0xFFF0u)));
          const int zero = (int)(word & 15u);
          uint32_t nibbles;
          if (is_value) {
            nibbles = *reinterpret_cast<const uint16_t*>(codes + ValuePairAt<D>(token, channel));
            nibbles |= (uint32_t)*reinterpret_cast<const uint16_t*>(codes + ValuePairAt<D>(token, channel + 4)) << 16;
          } else {
            nibbles = *reinterpret_cast<const uint32_t*>(codes + KeyWordAt<D>(token, channel));
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e / 4][e % 4] = scale * (float)((int)((nibbles >> (4 * e)) & 15u) - zero);
        }
        Store4(tensor + (size_t)(c / 4) * w.tokens + at.row, v[0]);
        Store4(tensor + (size_t)(c / 4 + 1) * w.tokens + at.row, v[1]);
      }
    } else {
      // (lanes without a token take part in the reductions with zeros)
      float x[kMine];
#pragma unroll
      for (int c = 0; c < kMine; c += 4) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (at.inside) Load4(tensor[(size_t)(c / 4) * w.tokens + at.row], v);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[c + e] = Held(v[e]);
      }
      // lowest and highest of blocks of 16 channels, then of the groups: inside a lane, then across the lanes that share one
      constexpr int kBlocks = kMine / 16;
      float low[kBlocks], high[kBlocks];
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        low[b] = high[b] = 0.0f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          low[b] = fminf(low[b], x[16 * b + e]);
          high[b] = fmaxf(high[b], x[16 * b + e]);
        }
      }
#pragma unroll
      for (int width = 2; width <= 8; width *= 2) {  // blocks of a group so far
        if (width * 16 > group) break;
        if (width <= kBlocks) {
#pragma unroll
          for (int b = 0; b < kBlocks; b += width)
#pragma unroll
            for (int e = 0; e < width / 2 && b + e + width / 2 < kBlocks; ++e) {
              low[b + e] = low[b + e + width / 2] = fminf(low[b + e], low[b + e + width / 2]);
              high[b + e] = high[b + e + width / 2] = fmaxf(high[b + e], high[b + e + width / 2]);
            }
        } else {
          const int across = width / kBlocks * 8;  // 16 or 32: the lane of the neighbouring run of channels
          low[0] = fminf(low[0], __shfl_xor(low[0], across));
          high[0] = fmaxf(high[0], __shfl_xor(high[0], across));
          if (kBlocks > 1) {
#pragma unroll
            for (int b = 1; b < kBlocks; ++b) low[b] = low[0], high[b] = high[0];
          }
        }
      }
      if (!at.inside) continue;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int channel0 = quarter * kMine + 16 * b;
        const uint32_t bits = ScaleBits((double)high[b] - (double)low[b]);
        const float scale = __half2float(__ushort_as_half((unsigned short)bits));
        const float inv = bits ? 1.0f / scale : 0.0f;
        const float zero = bits ? RoundedQuotient(-low[b], scale, inv) : 0.0f;
        if ((channel0 & (group - 1)) == 0) words[(channel0 >> w.group_shift) * 16] = (uint16_t)(bits | (uint32_t)zero);
#pragma unroll
        for (int c = 0; c < 16; c += 8) {
          uint32_t nibbles = 0;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float code = bits ? RoundedQuotient(x[16 * b + c + e], scale, inv) + zero : 0.0f;
            nibbles |= (uint32_t)fminf(fmaxf(code, 0.0f), 15.0f) << (4 * e);
          }
          if (is_value) {
            *reinterpret_cast<uint16_t*>(codes + ValuePairAt<D>(token, channel0 + c)) = (uint16_t)nibbles;
            *reinterpret_cast<uint16_t*>(codes + ValuePairAt<D>(token, channel0 + c + 4)) = (uint16_t)(nibbles >> 16);
          } else {
            *reinterpret_cast<uint32_t*>(codes + KeyWordAt<D>(token, channel0 + c)) = nibbles;
          }
        }
      }
    }
  }
}

template <typename T, bool READ>
void LaunchTyped(const Kv4MoveArgs& p, hipStream_t stream) {
  // tiles that max_new rows can touch, 4 to a work-group
  const int tiles = DivUp(p.max_new, kKv4Tile) + 1;
  const dim3 grid(DivUp(tiles, 4), 2 * p.where.kv_heads, p.where.sequences);
  if (p.head_dim == 64)
    kv4_move_kernel<T, 64, READ><<<grid, 256, 0, stream>>>(p);
  else if (p.head_dim == 128)
    kv4_move_kernel<T, 128, READ><<<grid, 256, 0, stream>>>(p);
  else
    kv4_move_kernel<T, 256, READ><<<grid, 256, 0, stream>>>(p);
}

}  // namespace

hipError_t LaunchKv4Append(const Kv4MoveArgs& a, hipStream_t stream, const char** kernel_name) {
  *kernel_name = "kv4_move_kernel";
  if (a.f16)
    LaunchTyped<__half, false>(a, stream);
  else
    LaunchTyped<float, false>(a, stream);
  return hipGetLastError();
}

hipError_t LaunchKv4Read(const Kv4MoveArgs& a, hipStream_t stream, const char** kernel_name) {
  *kernel_name = "kv4_move_kernel";
  if (a.f16)
    LaunchTyped<__half, true>(a, stream);
  else
    LaunchTyped<float, true>(a, stream);
  return hipGetLastError();
}

}  // namespace mldhip
