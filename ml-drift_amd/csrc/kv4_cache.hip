// Writing new keys and values into the cache of 4-bit codes and reading cached ones back (kv4.h: the layout).
//
// A group of G channels x of one token, lo = min(x, 0), hi = max(x, 0):
//   scale = the smallest half of 7 significant bits with 15 * scale >= hi - lo,  zero = rint(-lo / scale),
//   code = min(max(rint(x / scale) + zero, 0), 15),  value = scale * (code - zero);  rint: ties to even.
// All of it is exact: the span in fp64, the quotients by a product with the approximate reciprocal and one exact correction, so that the
// codes do not depend on how a division rounds.  Inputs are held to +-57344 and NaN counts as 0: a cached value is always a finite half,
// and a masked position can never turn a product into NaN.
//
// Memory bounds it: tensors of 2 or 4 bytes a channel against 0.53 .. 0.63.  Reading 8 sequences of 8192 tokens, 8 heads of 128 (340 MB): 69 us,
// 4.9 TB/s as a large copy (four fifths of the bytes are stores; 75 us under the profiler).  5000 fp32 tokens of one head of 256 (12 MB) are 8.0 us to append,
// bound by the branches of the corrected quotients between 2-byte stores, and 6.8 to read, where each piece's words are waited for behind the stores of
// the piece before.  One token of 64 sequences: 3.7 and 2.8, lengths, table and data, one after the other.
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

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

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Stores past the L2, for results that are larger (8 sequences of 8192 tokens, 8 heads of 128: 82 -> 70 us; 83.6 -> 75.4 under the profiler).
__device__ __forceinline__ void Stream4(uint2* p, const float v[4]) {
  uint2 raw;
  Store4(&raw, v);
  __builtin_nontemporal_store(u32x2{raw.x, raw.y}, reinterpret_cast<u32x2*>(p));
}
__device__ __forceinline__ void Stream4(float4* p, const float v[4]) {
  typedef float f32x4 __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store(f32x4{v[0], v[1], v[2], v[3]}, reinterpret_cast<f32x4*>(p));
}

// Byte offsets inside a tile's codes: of the 2 bytes of 4 channels from `channel` on.
template <int D>
__device__ __forceinline__ int KeyCodesAt(int token, int channel) {
  constexpr int P = Kv4Plane(D);
  const int i = channel % P;
  return channel / P * (8 * P) + (token * 4 + i % 32 / 8) * (P / 8) + i / 32 * 4 + i % 8 / 2;
}
template <int D>
__device__ __forceinline__ int ValueCodesAt(int token, int channel) {
  constexpr int P = Kv4Plane(D), kCell = P / 16;
  const int i = channel % P;
  return channel / P * (8 * P) + (token / 4 * 16 + i / kCell) * (2 * kCell) + i % kCell / 4 * 8 + token % 4 * 2;
}

// Grid: runs of a sequence's new rows x (head, keys or values) x sequences.  A wave takes kRows neighbouring rows of one head, a row shared
// by the D / CH lanes that have CH neighbouring channels each (rows run along the lanes, so that loads and stores of the tensors are runs of
// 8 or 16 bytes times kRows).  More rows than the launch was sized for only take longer.
template <typename T, int D, int CH, bool READ>
__global__ __launch_bounds__(256) void kv4_move_kernel(const Kv4MoveArgs p) {
  using Raw = typename Slice<T>::type;
  constexpr int kRows = 64 * CH / D;
  const Kv4Where& w = p.where;
  const int lane = threadIdx.x & 63;
  const bool is_value = blockIdx.y & 1;
  const int head = blockIdx.y >> 1, s = blockIdx.z;
  const Kv4Sequence q = Kv4SequenceOf(w, s);
  const int page_tokens = 1 << w.page_shift, groups = D >> w.group_shift, group = 1 << w.group_shift;
  const int codes_at = is_value ? Kv4ValueCodes(page_tokens, D) : 0;
  const int words_at = is_value ? Kv4ValueWords(page_tokens, D, groups) : Kv4KeyWords(page_tokens, D);
  const int channel0 = lane / kRows * CH;  // the lane's first
  Raw* tensor = static_cast<Raw*>(is_value ? p.v : p.k) + (size_t)(head * D + channel0) / 4 * w.tokens + q.start;
  for (int first = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kRows; first < q.count; first += gridDim.x * 4 * kRows) {
    const int i = first + lane % kRows, position = q.first + i;
    const bool is_row = i < q.count;
    int page = -1;
    if (is_row && position >= 0 && position < q.held) page = w.table[(size_t)s * w.pages_per_sequence + (position >> w.page_shift)];
    const bool there = page >= 0 && page < w.pages;
    uint8_t* block = static_cast<uint8_t*>(p.cache) + ((size_t)(there ? page : 0) * w.kv_heads + head) * w.block_bytes;
    const int token = position & 15, in_page = position & (page_tokens - 1) & ~15;
    uint8_t* codes = block + codes_at + in_page * (D / 2);
    uint16_t* words = reinterpret_cast<uint16_t*>(block + words_at) + in_page * groups + token;  // [group][16]
    if constexpr (READ) {
      if (!is_row) continue;
#pragma unroll
      for (int c = 0; c < CH; c += 4) {
        const int channel = channel0 + c;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (there) {
          const uint32_t word = words[(channel >> w.group_shift) * 16];
          const float scale = __half2float(__ushort_as_half((unsigned short)(word & 0xFFF0u)));
          const int zero = (int)(word & 15u);
          const uint32_t nibbles = *reinterpret_cast<const uint16_t*>(codes + (is_value ? ValueCodesAt<D>(token, channel) : KeyCodesAt<D>(token, channel)));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = scale * (float)((int)((nibbles >> (4 * e)) & 15u) - zero);
        }
        Store4(tensor + (size_t)(c / 4) * w.tokens + i, v);
      }
    } else {
      // (lanes without a place take part in the reductions with zeros)
      float x[CH];
#pragma unroll
      for (int c = 0; c < CH; c += 4) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (is_row) Load4(tensor[(size_t)(c / 4) * w.tokens + i], v);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[c + e] = Held(v[e]);
      }
      float low = 0.0f, high = 0.0f;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        low = fminf(low, x[c]);
        high = fmaxf(high, x[c]);
      }
      for (int lanes = kRows; lanes * CH < group * kRows; lanes *= 2) {  // the lanes that share the group
        low = fminf(low, __shfl_xor(low, lanes));
        high = fmaxf(high, __shfl_xor(high, lanes));
      }
      if (!there) continue;
      const uint32_t bits = ScaleBits((double)high - (double)low);
      const float scale = __half2float(__ushort_as_half((unsigned short)bits));
      const float inv = bits ? 1.0f / scale : 0.0f;
      const float zero = bits ? RoundedQuotient(-low, scale, inv) : 0.0f;
      if ((channel0 & (group - 1)) == 0) words[(channel0 >> w.group_shift) * 16] = (uint16_t)(bits | (uint32_t)zero);
#pragma unroll
      for (int c = 0; c < CH; c += 4) {
        uint32_t nibbles = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float code = bits ? RoundedQuotient(x[c + e], scale, inv) + zero : 0.0f;
          nibbles |= (uint32_t)fminf(fmaxf(code, 0.0f), 15.0f) << (4 * e);
        }
        *reinterpret_cast<uint16_t*>(codes + (is_value ? ValueCodesAt<D>(token, channel0 + c) : KeyCodesAt<D>(token, channel0 + c))) = (uint16_t)nibbles;
      }
    }
  }
}

// Reading many rows: a wave takes one tile of the cache, whose codes it reads as a lane of attention's products does, 8 or 16 bytes at a time
// (kv4.h); tokens run along the lanes of the stores, so that these are runs of 16 tokens.
// Grid: tiles of a sequence's rows x (head, keys or values) x sequences.
template <typename T, int D>
__global__ __launch_bounds__(256) void kv4_read_tiles_kernel(const Kv4MoveArgs p) {
  using Raw = typename Slice<T>::type;
  constexpr int P = Kv4Plane(D), kPlanes = D / P, kWords = P / 32, kCell = P / 16;
  const Kv4Where& w = p.where;
  const int lane = threadIdx.x & 63, n = lane & 15, quad = lane >> 4;
  const bool is_value = blockIdx.y & 1;
  const int head = blockIdx.y >> 1, s = blockIdx.z;
  const Kv4Sequence q = Kv4SequenceOf(w, s);
  const int page_tokens = 1 << w.page_shift, groups = D >> w.group_shift;
  __shared__ uint32_t exchange[4][kPlanes * 64 * kWords];
  const int tile_begin = q.first >> 4, tile_end = (q.first + q.count + 15) >> 4;  // (first may be negative: rows without a position)
  // row i of the sequence, slice c of the head: tensor[c * tokens + i]
  Raw* tensor = static_cast<Raw*>(is_value ? p.v : p.k) + (size_t)head * (D / 4) * w.tokens + q.start;
  for (int tile = tile_begin + (int)(blockIdx.x * 4 + (threadIdx.x >> 6)); tile < tile_end; tile += gridDim.x * 4) {
    int page = -1;
    if (tile >= 0 && tile * kKv4Tile < q.held) page = w.table[(size_t)s * w.pages_per_sequence + (tile * kKv4Tile >> w.page_shift)];
    const bool there = page >= 0 && page < w.pages;
    const uint8_t* block = static_cast<const uint8_t*>(p.cache) + ((size_t)(there ? page : 0) * w.kv_heads + head) * w.block_bytes;
    const int in_page = (tile * kKv4Tile) & (page_tokens - 1);
    const uint8_t* codes = block + (is_value ? Kv4ValueCodes(page_tokens, D) : 0) + in_page * (D / 2) + (is_value ? quad * 16 + n : n * 4 + quad) * (P / 8);
    const uint16_t* words = reinterpret_cast<const uint16_t*>(block + (is_value ? Kv4ValueWords(page_tokens, D, groups) : Kv4KeyWords(page_tokens, D))) + in_page * groups;
    uint32_t piece[kPlanes][kWords];
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl) {
      if constexpr (P == 128) {
        const u32x4 a = *reinterpret_cast<const u32x4*>(codes + pl * 8 * P);
#pragma unroll
        for (int k = 0; k < 4; ++k) piece[pl][k] = a[k];
      } else {
        const u32x2 a = *reinterpret_cast<const u32x2*>(codes);
        piece[0][0] = a.x, piece[0][1] = a.y;
      }
    }
    // the lane's token, and its place among the tensors' rows
    const int position = tile * kKv4Tile + n, row = position - q.first;
    const bool is_row = row >= 0 && row < q.count, held = there && position < q.held;
    if (is_value) {  // a lane has the values of four tokens: through LDS to the lanes of these
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
        for (int k = 0; k < kWords; ++k) exchange[threadIdx.x >> 6][(pl * 64 + quad * 16 + n) * kWords + k] = piece[pl][k];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    const uint32_t* mine = exchange[threadIdx.x >> 6];
    const uint32_t of_token = n % 2 ? 0x07060302u : 0x05040100u;  // the half of a word that is the lane's token's
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
      for (int k = 0; k < kWords; ++k) {
        // 8 channels: of a word of the keys; of the values those of two (four) cells, 8 (4) channels each
        const int channel = is_value ? pl * P + quad * (P / 4) + 8 * k : pl * P + 32 * k + 8 * quad;
        uint32_t nibbles = piece[pl][k];
        if (is_value) {
          const int i = channel % P, j = i + 4;  // (of 4 channels each)
          const int at = (pl * 64 + n / 4 * 16) * kWords + n % 4 / 2;
          nibbles = __builtin_amdgcn_perm(mine[at + j / kCell * kWords + j % kCell / 4 * 2], mine[at + i / kCell * kWords + i % kCell / 4 * 2], of_token);
        }
        const uint32_t word = held ? words[(channel >> w.group_shift) * 16 + n] : 0;  // (scale 0: zeros)
        const float scale = __half2float(__ushort_as_half((unsigned short)(word & 0xFFF0u)));
        float v[2][4];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e / 4][e % 4] = scale * (float)((int)((nibbles >> (4 * e)) & 15u) - (int)(word & 15u));
        if (is_row) {
          Stream4(tensor + (size_t)(channel / 4) * w.tokens + row, v[0]);
          Stream4(tensor + (size_t)(channel / 4 + 1) * w.tokens + row, v[1]);
        }
      }
    if (is_value) {  // the exchange is written again: behind all lanes' reads
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
  }
}

template <typename T, int D, int CH, bool READ>
void LaunchForm(const Kv4MoveArgs& p, hipStream_t stream) {
  const dim3 grid(DivUp(std::min(p.max_new, p.where.tokens), 4 * (64 * CH / D)), 2 * p.where.kv_heads, p.where.sequences);
  kv4_move_kernel<T, D, CH, READ><<<grid, 256, 0, stream>>>(p);
}
constexpr int kFewNew = 8;
template <typename T, int D, bool READ>
void LaunchHead(const Kv4MoveArgs& p, hipStream_t stream) {
  // few rows: a lane has one slice, so that a row is spread over as many lanes as it can; else 16 channels (reading: a tile for each wave).
  // Appending and reading back for 64 sequences, 8 heads of 128: 5.8 us against 9.9 at one row each, 7.5 against 8.4 at 8, 10.7 against 9.2 at 16.
  if (p.max_new <= kFewNew) {
    LaunchForm<T, D, 4, READ>(p, stream);
  } else if constexpr (READ) {
    const int tiles = DivUp(std::min(p.max_new, p.where.tokens), kKv4Tile) + 1;
    kv4_read_tiles_kernel<T, D><<<dim3(DivUp(tiles, 4), 2 * p.where.kv_heads, p.where.sequences), 256, 0, stream>>>(p);
  } else {
    LaunchForm<T, D, 16, false>(p, stream);
  }
}
template <typename T, bool READ>
void LaunchTyped(const Kv4MoveArgs& p, hipStream_t stream) {
  if (p.head_dim == 64)
    LaunchHead<T, 64, READ>(p, stream);
  else if (p.head_dim == 128)
    LaunchHead<T, 128, READ>(p, stream);
  else
    LaunchHead<T, 256, READ>(p, stream);
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
  *kernel_name = a.max_new <= kFewNew ? "kv4_move_kernel" : "kv4_read_tiles_kernel";
  if (a.f16)
    LaunchTyped<__half, true>(a, stream);
  else
    LaunchTyped<float, true>(a, stream);
  return hipGetLastError();
}

}  // namespace mldhip
