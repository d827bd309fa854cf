// Attention over the cache of 4-bit keys and values (kv4.h: the layout).
//
//   out_r = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale * (q_r . k_t) - max),  t over the positions that row r sees:
//   t < length, t <= position of r (causal), t > position of r - window.  A row that sees nothing is 0.
//
// One pass over the cache with the running maximum and sum of each row.  The heads of a group share the keys they read: the rows of a
// tile are (new token, head of the group).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include <algorithm>

#include "kernels.h"
#include "kv4.h"

namespace mldhip {
namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ half2_t AsHalf2(uint32_t v) { return __builtin_bit_cast(half2_t, v); }
__device__ __forceinline__ uint32_t AsU32(half2_t v) { return __builtin_bit_cast(uint32_t, v); }

// A nibble at bits 0..3 of a half's mantissa under the exponent of 1024 is 1024 + nibble, at bits 4..7 under that of 64 it is 64 + nibble:
// one and-or unpacks two nibbles, and only every other pair needs a shift.
constexpr uint32_t kLowMask = 0x000F000Fu, kHighMask = 0x00F000F0u, kLowBase = 0x64006400u, kHighBase = 0x54005400u;
constexpr float kLowOffset = 1024.0f, kHighOffset = 64.0f;
constexpr uint32_t kScaleMask = 0xFFF0FFF0u;

constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are exp2(x - max + kLift): the largest is 2^14, so that as halfs (the operands of the second product) they keep all
// their 11 bits down to 2^-28 of it.  The common factor leaves with the division by their sum, which is taken in fp32.
constexpr float kLift = 14.0f;

constexpr int kStep = 64;  // positions that a wave takes at a time

struct FewParams {
  Kv4Where w;
  const __half* q;
  const uint8_t* cache;
  __half* out;
  float* part_o;   // [parts][rows of the tensors][D]
  float2* part_ml; // [parts][rows]: maximum (of q . k) and sum
  int heads, share, parts, causal, window;
  float c;  // scale * log2(e)
  int rows_from, rows_to;  // sequences of rows_from .. rows_to rows are this kernel's
};

__device__ __forceinline__ float MaxAcrossQuarters(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float SumAcrossQuarters(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// Few rows for each key head (single tokens, speculated ones): the cache's bytes bound it, so the keys of a sequence are dealt to the
// waves of `parts` work-groups, each wave with its own maximum, sum and output, joined at the end.
//
// A wave takes 64 positions at a time against RT tiles of 16 rows, by 16x16x32 products:
//   scores^T [16 positions][16 rows] = codes of keys x q^T     a lane has one row (lane & 15) and 4 positions (4 (lane >> 4) + i)
//   out^T   [16 cells][16 rows]     += values^T x p^T          of 32 positions: those that the lanes hold are the operand's order, so the
//                                                              probabilities go from one product to the next in registers
// The first product runs on the codes as they are, exact small integers; their scale and zero point, which belong to (position, group),
// are applied to its fp32 sums, one pair of multiply-adds per 32 .. 128 codes: sum q (code - zero) = sum q (base + code) - base sum q - zero
// sum q.  The values are dequantized, exactly (kv4.h).
template <int D, int GJ, int RT>
__global__ __launch_bounds__(256) void kv4_attention_few_kernel(const FewParams p) {
  constexpr int P = Kv4Plane(D), kPlanes = D / P, kWords = P / 32, kCell = P / 16;
  constexpr int kGroups = D / 32 / GJ;          // groups of a head
  constexpr int kKeyRegs = kPlanes * kWords;    // 32-bit words of a lane's keys per tile (8 channels each)
  constexpr int kValueRegs = kPlanes * kCell / 2;  // and of its values (4 channels of 2 positions each)
  constexpr int kTiles = kStep / 16;
  const Kv4Where& w = p.w;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  const int kv_head = blockIdx.y, s = blockIdx.z;
  const Kv4Sequence q = Kv4SequenceOf(w, s);
  const int rows = q.count * p.share;
  if (rows < p.rows_from || rows > p.rows_to) return;
  const int part = blockIdx.x % p.parts;
  const int page_tokens = 1 << w.page_shift;
  __shared__ float4 sum_lds[4][16][D / 4 + 1];
  __shared__ float2 ml_lds[4][16 * RT];

  for (int row0 = (blockIdx.x / p.parts) * 16 * RT; row0 < rows; row0 += gridDim.x / p.parts * 16 * RT) {
    // the positions that the tile's rows see: [lo, hi), in steps of 64 dealt to the parts and, one by one, to their waves
    const int first_row = q.first + row0 / p.share, last_row = q.first + (min(rows, row0 + 16 * RT) - 1) / p.share;
    const int hi = p.causal ? min(q.held, last_row + 1) : q.held;
    const int lo = p.window > 0 ? max(0, first_row + 1 - p.window) : 0;
    const int step0 = lo / kStep, steps = hi > lo ? (hi - 1) / kStep + 1 - step0 : 0;
    const int each = (steps + p.parts - 1) / p.parts;
    const int begin = step0 + min(steps, part * each), end = step0 + min(steps, (part + 1) * each);

    u32x4 qa[RT][kKeyRegs];       // operands of the first product: channel s and channel s + 4 of 8 in each register
    float qsum[RT][kGroups], qbase[RT][kGroups];  // sum of the row's q over a group; the same weighted by the codes' bases
    int row_lo[RT], row_hi[RT];   // what the lane's row sees
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = row0 + rt * 16 + n;
      const bool there = row < rows;
      const int token = (there ? row : 0) / p.share, head = kv_head * p.share + (there ? row : 0) % p.share;
      const u32x2* src = reinterpret_cast<const u32x2*>(p.q) + (size_t)head * (D / 4) * w.tokens + q.start + token;
      const int position = q.first + token;
      row_hi[rt] = there ? (p.causal ? min(q.held, position + 1) : q.held) : 0;
      row_lo[rt] = p.window > 0 ? max(0, position + 1 - p.window) : 0;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) qsum[rt][g] = qbase[rt][g] = 0.0f;
#pragma unroll
      for (int k = 0; k < kKeyRegs; ++k) {
        u32x2 a = {0u, 0u}, b = {0u, 0u};
        if (there) {
          a = src[(size_t)(8 * k + 2 * quad) * w.tokens];
          b = src[(size_t)(8 * k + 2 * quad + 1) * w.tokens];
        }
        qa[rt][k] = u32x4{__builtin_amdgcn_perm(b.x, a.x, 0x05040100u), __builtin_amdgcn_perm(b.x, a.x, 0x07060302u),
                          __builtin_amdgcn_perm(b.y, a.y, 0x05040100u), __builtin_amdgcn_perm(b.y, a.y, 0x07060302u)};
        float low = 0.0f, high = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const half2_t v = AsHalf2(qa[rt][k][e]);
          ((e & 1) ? high : low) += (float)v.x + (float)v.y;
        }
        qsum[rt][k / GJ] += low + high;
        qbase[rt][k / GJ] += kLowOffset * low + kHighOffset * high;
      }
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        qsum[rt][g] = SumAcrossQuarters(qsum[rt][g]);
        qbase[rt][g] = -SumAcrossQuarters(qbase[rt][g]);
      }
    }

    float4_t acc[RT][kPlanes][kCell];
    float top[RT], sum[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      top[rt] = -INFINITY;
      sum[rt] = 0.0f;
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
        for (int j = 0; j < kCell; ++j) acc[rt][pl][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (int step = begin + wave; step < end; step += 4) {
      uint32_t keys[kTiles][kKeyRegs], values[kTiles][kValueRegs];
      u32x2 key_words[kTiles][kGroups], value_words[kTiles][kPlanes];
      bool there[kTiles];
      // a step inside what every row sees, on pages that there are, needs no masks
      bool whole = step * kStep + kStep <= (p.causal ? min(q.held, first_row + 1) : q.held);
      if (p.window > 0) whole = whole && step * kStep > last_row - p.window;
      if (row0 + 16 * RT > rows) whole = whole && true;  // (rows that are not there have q = 0 and are not stored)
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        // (tiles behind the last held position read the last one again: what they hold is masked)
        const int tile = min(step * kTiles + u, (q.held - 1) >> 4);
        const int id = w.table[(size_t)s * w.pages_per_sequence + (tile * 16 >> w.page_shift)];
        there[u] = id >= 0 && id < w.pages;
        whole = whole && there[u];
        const uint8_t* block = p.cache + ((size_t)(there[u] ? id : 0) * w.kv_heads + kv_head) * w.block_bytes;
        const int in_page = (tile * 16) & (page_tokens - 1);
        const uint8_t* kc = block + (size_t)in_page * (D / 2) + (n * 4 + quad) * (P / 8);
        const uint8_t* vc = block + Kv4ValueCodes(page_tokens, D) + (size_t)in_page * (D / 2) + (quad * 16 + n) * (2 * kCell);
#pragma unroll
        for (int pl = 0; pl < kPlanes; ++pl) {
          if constexpr (P == 128) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(kc + pl * 8 * P), b = *reinterpret_cast<const u32x4*>(vc + pl * 8 * P);
#pragma unroll
            for (int e = 0; e < 4; ++e) keys[u][4 * pl + e] = a[e], values[u][4 * pl + e] = b[e];
          } else {
            const u32x2 a = *reinterpret_cast<const u32x2*>(kc), b = *reinterpret_cast<const u32x2*>(vc);
            keys[u][0] = a.x, keys[u][1] = a.y, values[u][0] = b.x, values[u][1] = b.y;
          }
        }
        const uint16_t* kw = reinterpret_cast<const uint16_t*>(block + Kv4KeyWords(page_tokens, D)) + in_page * kGroups + 4 * quad;
        const uint16_t* vw = reinterpret_cast<const uint16_t*>(block + Kv4ValueWords(page_tokens, D, kGroups)) + in_page * kGroups + 4 * quad;
#pragma unroll
        for (int g = 0; g < kGroups; ++g) key_words[u][g] = *reinterpret_cast<const u32x2*>(kw + 16 * g);
#pragma unroll
        for (int pl = 0; pl < kPlanes; ++pl)
          value_words[u][pl] = *reinterpret_cast<const u32x2*>(vw + 16 * ((pl * P + n * kCell) / (32 * GJ)));
      }

      // scores: score[rt][u][i] = q . k of row n and position 16 u + 4 quad + i
      float score[RT][kTiles][4];
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        float4_t raw[RT][kGroups];
#pragma unroll
        for (int k = 0; k < kKeyRegs; ++k) {
          const uint32_t a = keys[u][k], b = a >> 8;
          const u32x4 codes = {(a & kLowMask) | kLowBase, (a & kHighMask) | kHighBase, (b & kLowMask) | kLowBase, (b & kHighMask) | kHighBase};
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const float o = qbase[rt][k / GJ];
            const float4_t from = k % GJ == 0 ? float4_t{o, o, o, o} : raw[rt][k / GJ];
            raw[rt][k / GJ] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, codes),
                                                                    __builtin_bit_cast(half8_t, qa[rt][k]), from, 0, 0, 0);
          }
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int i = 0; i < 4; ++i) score[rt][u][i] = 0.0f;
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t word = key_words[u][g][i / 2];
            const float scale = (float)AsHalf2(word & kScaleMask)[i % 2];
            const float zero = (float)((word >> (16 * (i % 2))) & 15u);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              score[rt][u][i] = fmaf(scale, fmaf(-zero, qsum[rt][g], raw[rt][g][i]), score[rt][u][i]);
          }
      }
      if (!whole) {
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
          const int at = step * kStep + 16 * u + 4 * quad;
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!there[u] || at + i >= row_hi[rt] || at + i < row_lo[rt]) score[rt][u][i] = -INFINITY;
          // what lies behind the held positions may be anything: as values it is 0 (0 * NaN would not be)
#pragma unroll
          for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int two = at + 2 * i;
              const uint32_t keep = !there[u] || two >= q.held ? 0u : two + 1 >= q.held ? 0x0000FFFFu : 0xFFFFFFFFu;
              value_words[u][pl][i] &= keep;
            }
        }
      }

      // the running maximum; what the new one is above the old scales the sums so far
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        float best = score[rt][0][0];
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) best = fmaxf(best, score[rt][u][i]);
        best = MaxAcrossQuarters(best);
        if (__any(best > top[rt])) {
          const float now = fmaxf(top[rt], best);
          const float down = top[rt] == now ? 1.0f : exp2f((top[rt] - now) * p.c);  // (-inf - finite: 0)
          top[rt] = now;
          sum[rt] *= down;
#pragma unroll
          for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
            for (int j = 0; j < kCell; ++j) acc[rt][pl][j] *= down;
        }
      }

      half2_t prob[RT][kTiles][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float base = top[rt] == -INFINITY ? 0.0f : kLift - top[rt] * p.c;
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float a = __builtin_amdgcn_exp2f(fmaf(score[rt][u][2 * i], p.c, base));
            const float b = __builtin_amdgcn_exp2f(fmaf(score[rt][u][2 * i + 1], p.c, base));
            sum[rt] += a + b;
            prob[rt][u][i] = half2_t{(_Float16)a, (_Float16)b};
          }
      }

      // out^T += values^T x p^T, 32 positions at a time
#pragma unroll
      for (int u = 0; u < kTiles; u += 2) {
#pragma unroll
        for (int pl = 0; pl < kPlanes; ++pl) {
          half2_t scale[2][2], low_zero[2][2], high_zero[2][2];
#pragma unroll
          for (int v = 0; v < 2; ++v)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t word = value_words[u + v][pl][i];
              scale[v][i] = AsHalf2(word & kScaleMask);
              low_zero[v][i] = AsHalf2((word & kLowMask) | kLowBase);
              high_zero[v][i] = AsHalf2(((word << 4) & kHighMask) | kHighBase);
            }
#pragma unroll
          for (int h = 0; h < kCell / 4; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              u32x4 op;
#pragma unroll
              for (int v = 0; v < 2; ++v)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  uint32_t word = values[u + v][(pl * (kCell / 4) + h) * 2 + i];
                  if (e >= 2) word >>= 8;
                  const half2_t x = (e & 1) ? AsHalf2((word & kHighMask) | kHighBase) - high_zero[v][i]
                                            : AsHalf2((word & kLowMask) | kLowBase) - low_zero[v][i];
                  op[2 * v + i] = AsU32(x * scale[v][i]);
                }
#pragma unroll
              for (int rt = 0; rt < RT; ++rt) {
                const u32x4 pr = {AsU32(prob[rt][u][0]), AsU32(prob[rt][u][1]), AsU32(prob[rt][u + 1][0]), AsU32(prob[rt][u + 1][1])};
                acc[rt][pl][4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    __builtin_bit_cast(half8_t, op), __builtin_bit_cast(half8_t, pr), acc[rt][pl][4 * h + e], 0, 0, 0);
              }
            }
        }
      }
    }

    // the waves' outputs of each tile of rows, at the common maximum
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      sum[rt] = SumAcrossQuarters(sum[rt]);
      if (quad == 0) ml_lds[wave][rt * 16 + n] = make_float2(top[rt], sum[rt]);
    }
    __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float best = -INFINITY, total = 0.0f;
#pragma unroll
      for (int v = 0; v < 4; ++v) best = fmaxf(best, ml_lds[v][rt * 16 + n].x);
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float2 ml = ml_lds[v][rt * 16 + n];
        total += ml.y * (ml.x == best ? 1.0f : exp2f((ml.x - best) * p.c));
      }
      const float mine = top[rt] == best ? 1.0f : exp2f((top[rt] - best) * p.c);
      const float factor = mine * (p.parts > 1 ? 1.0f : total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total);
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < kCell / 4; ++h)
            sum_lds[wave][n][(pl * P + (4 * quad + i) * kCell) / 4 + h] =
                make_float4(acc[rt][pl][4 * h][i] * factor, acc[rt][pl][4 * h + 1][i] * factor, acc[rt][pl][4 * h + 2][i] * factor,
                            acc[rt][pl][4 * h + 3][i] * factor);
      __syncthreads();
      // 16 rows x D / 4 slices
      for (int item = threadIdx.x; item < 16 * (D / 4); item += 256) {
        const int r = item & 15, slice = item >> 4, row = row0 + rt * 16 + r;
        if (row < rows) {
          float4 v = sum_lds[0][r][slice];
#pragma unroll
          for (int k = 1; k < 4; ++k) {
            const float4 o = sum_lds[k][r][slice];
            v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
          }
          const size_t token = q.start + row / p.share;
          const int head = kv_head * p.share + row % p.share;
          if (p.parts > 1) {
            reinterpret_cast<float4*>(p.part_o)[(((size_t)part * w.tokens + token) * p.heads + head) * (D / 4) + slice] = v;
          } else {
            const half2_t a = {(_Float16)v.x, (_Float16)v.y}, b = {(_Float16)v.z, (_Float16)v.w};
            reinterpret_cast<u32x2*>(p.out)[((size_t)head * (D / 4) + slice) * w.tokens + token] = u32x2{AsU32(a), AsU32(b)};
          }
        }
      }
      if (p.parts > 1 && wave == 0 && quad == 0) {
        const int row = row0 + rt * 16 + n;
        if (row < rows)
          p.part_ml[((size_t)part * w.tokens + q.start + row / p.share) * p.heads + kv_head * p.share + row % p.share] = make_float2(best, total);
      }
      __syncthreads();  // (the arrays are written again)
    }
  }
}

// The parts of each row, joined: a wave per row, lanes over its slices.
struct JoinParams {
  Kv4Where w;
  const float* part_o;
  const float2* part_ml;
  __half* out;
  int heads, parts;
  float c;
  int share, rows_from, rows_to;  // of the sequences that were dealt in parts
};
template <int D>
__global__ __launch_bounds__(256) void kv4_attention_join_kernel(const JoinParams p) {
  const Kv4Where& w = p.w;
  const int lane = threadIdx.x & 63;
  const Kv4Sequence q = Kv4SequenceOf(w, blockIdx.y);
  if (q.count * p.share < p.rows_from || q.count * p.share > p.rows_to) return;
  const int rows = q.count * p.heads;
  for (int row = blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += gridDim.x * 4) {
    const size_t token = q.start + row / p.heads;
    const int head = row % p.heads;
    const size_t at = token * p.heads + head, step = (size_t)w.tokens * p.heads;
    float best = -INFINITY;
    for (int k = lane; k < p.parts; k += 64) best = fmaxf(best, p.part_ml[k * step + at].x);
#pragma unroll
    for (int off = 1; off < 64; off *= 2) best = fmaxf(best, __shfl_xor(best, off));
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float total = 0.0f;
    for (int k = 0; k < p.parts; ++k) {
      const float2 ml = p.part_ml[k * step + at];
      if (ml.y == 0.0f) continue;  // (a part that saw nothing)
      const float f = ml.x == best ? 1.0f : exp2f((ml.x - best) * p.c);
      total += ml.y * f;
      if (lane < D / 4) {
        const float4 o = reinterpret_cast<const float4*>(p.part_o)[(k * step + at) * (D / 4) + lane];
        v.x += o.x * f, v.y += o.y * f, v.z += o.z * f, v.w += o.w * f;
      }
    }
    const float f = total == 0.0f ? 0.0f : 1.0f / total;
    if (lane < D / 4) {
      const half2_t a = {(_Float16)(v.x * f), (_Float16)(v.y * f)}, b = {(_Float16)(v.z * f), (_Float16)(v.w * f)};
      reinterpret_cast<u32x2*>(p.out)[((size_t)head * (D / 4) + lane) * w.tokens + token] = u32x2{AsU32(a), AsU32(b)};
    }
  }
}

// How many work-groups a sequence's keys are dealt to.
int Parts(const Kv4AttentionArgs& a) {
  const int share = a.heads / a.where.kv_heads;
  const long long groups = (long long)a.where.sequences * a.where.kv_heads * DivUp(std::min(a.max_new, a.max_tokens) * share, 16);
  const long long keys = (long long)a.where.pages_per_sequence << a.where.page_shift;
  const long long wanted = (1024 + groups - 1) / groups;
  const long long most = (keys + 4 * kStep - 1) / (4 * kStep);
  return (int)std::max(1LL, std::min(std::min(wanted, most), 512LL));
}

template <int D, int GJ>
void LaunchFew(const Kv4AttentionArgs& a, hipStream_t stream) {
  FewParams p;
  p.w = a.where;
  p.q = static_cast<const __half*>(a.q);
  p.cache = a.cache;
  p.out = static_cast<__half*>(a.out);
  p.heads = a.heads;
  p.share = a.heads / a.where.kv_heads;
  p.parts = Parts(a);
  p.causal = a.causal;
  p.window = a.window;
  p.c = a.scale * kLog2e;
  p.rows_from = 1;
  p.rows_to = INT32_MAX;
  p.part_o = a.partial;
  p.part_ml = reinterpret_cast<float2*>(a.partial + (size_t)p.parts * a.max_tokens * a.heads * D);
  const int row_tiles = DivUp(std::min(a.max_new, a.where.tokens) * p.share, 16);
  const dim3 grid(p.parts * row_tiles, a.where.kv_heads, a.where.sequences);
  SetTiles(a.tiles, 16, 4, p.parts);
  SetVariant(a.variant, "few");
  kv4_attention_few_kernel<D, GJ, 1><<<grid, 256, 0, stream>>>(p);
  if (p.parts > 1) {
    JoinParams j;
    j.w = a.where;
    j.part_o = p.part_o;
    j.part_ml = p.part_ml;
    j.out = p.out;
    j.heads = a.heads;
    j.parts = p.parts;
    j.c = p.c;
    j.share = p.share;
    j.rows_from = p.rows_from;
    j.rows_to = p.rows_to;
    const dim3 join(DivUp(std::min(a.max_new, a.where.tokens) * a.heads, 4), a.where.sequences);
    kv4_attention_join_kernel<D><<<join, 256, 0, stream>>>(j);
  }
}

}  // namespace

size_t Kv4AttentionWorkspaceFloats(const Kv4AttentionArgs& a) {
  const int parts = Parts(a);
  return parts > 1 ? (size_t)parts * a.max_tokens * a.heads * (a.head_dim + 2) : 0;
}

hipError_t LaunchKv4Attention(const Kv4AttentionArgs& a, hipStream_t stream, const char** kernel_name) {
  *kernel_name = "kv4_attention_few_kernel";
  const int gj = 1 << (a.where.group_shift - 5);
  if (a.head_dim == 64)
    gj == 1 ? LaunchFew<64, 1>(a, stream) : LaunchFew<64, 2>(a, stream);
  else if (a.head_dim == 128)
    gj == 1 ? LaunchFew<128, 1>(a, stream) : gj == 2 ? LaunchFew<128, 2>(a, stream) : LaunchFew<128, 4>(a, stream);
  else
    gj == 1 ? LaunchFew<256, 1>(a, stream) : gj == 2 ? LaunchFew<256, 2>(a, stream) : LaunchFew<256, 4>(a, stream);
  return hipGetLastError();
}

}  // namespace mldhip
