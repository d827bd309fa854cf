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

typedef _Float16 half_t;
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ half2_t AsHalf2(uint32_t v) { return __builtin_bit_cast(half2_t, v); }
__device__ __forceinline__ uint32_t AsU32(half2_t v) { return __builtin_bit_cast(uint32_t, v); }

// A nibble at bits 0..3 of a half's mantissa under the exponent of 1024 is 1024 + nibble, at bits 4..7 under that of 64 it is 64 + nibble:
// one and-or unpacks two nibbles, and only every other pair needs a shift.
constexpr uint32_t kLowMask = 0x000F000Fu, kHighMask = 0x00F000F0u, kLowBase = 0x64006400u, kHighBase = 0x54005400u;
constexpr uint32_t kScaleMask = 0xFFF0FFF0u;

constexpr float kLog2e = 1.4426950408889634f;
// Probabilities are exp2(x - max + kLift): the largest is 2^14, so that as halfs (the operands of the second product) they keep all
// their 11 bits down to 2^-28 of it.  The common factor leaves with the division by their sum, which is taken in fp32.
constexpr float kLift = 14.0f;

// x - max is one multiply-add where max * c is small enough that its rounding does not count (2^-12 in the exponent); beyond, the maximum is taken
// away first: ulps of scores of 1e10 are thousands, which would be taken for powers of two.
constexpr float kFar = 4096.0f;

struct AttendParams {
  Kv4Where w;
  const __half* q;
  const uint8_t* cache;
  __half* out;
  float* part_o;   // few rows: [parts][rows of the tensors][D]; many: [parts][heads][D / 4][tokens][4], the outputs' own order
  float2* part_ml; // [parts][rows]: maximum (of q . k) and sum
  int heads, share, parts, causal, window;
  float c;  // scale * log2(e)
  int rows_from, rows_to;  // sequences of rows_from .. rows_to rows are this kernel's
};

// Over the four lanes that share a row (lane & 15), by register exchanges.
__device__ __forceinline__ float MaxAcrossQuarters(float v) {
  u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float SumAcrossQuarters(float v) {
  u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The lane's number, worked out where it is asked for: kept over a kernel's steps it would cost a register there (spilled for heads of 256).
__device__ __forceinline__ int LaneHere() {
  uint32_t all = ~0u;
  asm volatile("" : "+s"(all));
  return (int)__builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0u));
}

// A row of queries with an infinity or a NaN has no softmax: NaN, unless it sees no position, which is 0 whatever the row holds.  Its scores may
// be -inf like the ones that masks leave, or NaN behind the masks too: a row whose sum is not above 0 is looked at again, whether any of the
// positions from .. to - 1, which no mask hides, lies on a page that there is.  All lanes take part, 64 pages of begin .. end - 1 (positions, the same
// in all lanes) at a time.
__device__ __forceinline__ bool SeesAny(const Kv4Where& w, const int32_t* table, int begin, int end, int from, int to) {
  const int lane = LaneHere(), pages = end > begin ? ((end - 1) >> w.page_shift) + 1 : 0;
  const int first = from >> w.page_shift, behind = from < to ? ((to - 1) >> w.page_shift) + 1 : first;
  bool any = false;
  for (int page = begin >> w.page_shift; page < pages && __any(!any && first < behind); page += 64) {
    const int id = page + lane < pages ? table[page + lane] : -1;
    const uint64_t there = __ballot(id >= 0 && id < w.pages);
    const int low = max(first - page, 0), high = min(behind - page, 64);
    if (low < high) any = any || (there << (64 - high) >> (64 - high + low)) != 0;
  }
  return any;
}

// The masks and bases in registers whose values the compiler does not see: as literals each and-or would be two instructions.
struct Unpack {
  uint32_t low_mask = kLowMask, high_mask = kHighMask, low_base = kLowBase, high_base = kHighBase, scale_mask = kScaleMask;
  __device__ __forceinline__ Unpack() { asm volatile("" : "+v"(low_mask), "+v"(high_mask), "+s"(low_base), "+s"(high_base), "+s"(scale_mask)); }
  __device__ __forceinline__ uint32_t Low(uint32_t w) const { return (w & low_mask) | low_base; }
  __device__ __forceinline__ uint32_t High(uint32_t w) const { return (w & high_mask) | high_base; }
};

// Few rows for each key head (single tokens, speculated ones): the cache's bytes bound it, so the keys of a sequence are dealt to the
// waves of `parts` work-groups, each wave with its own maximum, sum and output, joined at the end.
//
// A wave takes 32 positions at a time against a tile of 16 rows, by 16x16x32 products:
//   scores^T [16 positions][16 rows] = codes of keys x q^T     a lane has one row (lane & 15) and 4 positions (4 (lane >> 4) + i)
//   out^T   [16 cells][16 rows]     += values^T x p^T          of 32 positions: those that the lanes hold are the operand's order, so the
//                                                              probabilities go from one product to the next in registers
// Keys and values are dequantized, exactly (kv4.h), so that the scores are fp32 sums of exact products: sums over the codes on their bases
// would be rounded at the size of 1024 sum |q| and lose the small codes of a group with one channel far from zero.
// Measured: 4 sequences of 65536 positions, 8 key heads of 128 (285 MB): 58 us with the join, 4.9 TB/s, what a large copy reaches.  Shorter caches
// are bound by vector instructions (287 for 32 positions of heads of 128, 184 of 64, most of them unpacking, 8 of them exponentials of four times the
// cycles: they alone could take heads of 128 in at 8.6 TB/s, of 64 at 6.8) and by what precedes the first product: lengths, table, codes, one
// after the other, 2 to 4 us.
template <int D, int GJ>
struct FewShape {
  static constexpr int P = Kv4Plane(D), kPlanes = D / P, kWords = P / 32, kCell = P / 16;
  static constexpr int kGroups = D / 32 / GJ;             // groups of a head
  static constexpr int kKeyRegs = kPlanes * kWords;       // 32-bit words of a lane's keys per tile (8 channels each)
  static constexpr int kValueRegs = kPlanes * kCell / 2;  // and of its values (4 channels of 2 positions each)
  static constexpr int kStep = 32;                        // positions that a wave takes at a time: two steps are in registers
  static constexpr int kTiles = kStep / 16;
  // A lane needs the words of the keys of its position (lane & 15) for all groups, as the other quarters do: quarter i loads those of groups
  // i, i + 4, and they change quarters by register exchanges, those of both tiles in one register.
  static constexpr int kGroupsAtOnce = kGroups < 4 ? kGroups : 4, kWordRegs = kGroups / kGroupsAtOnce;
  static_assert(kTiles == 2);
};

// The cached bytes of one step, as a lane holds them.
template <int D, int GJ>
struct FewStep {
  using S = FewShape<D, GJ>;
  uint32_t keys[S::kTiles][S::kKeyRegs], values[S::kTiles][S::kValueRegs];
  uint32_t key_words[S::kTiles][S::kWordRegs];
  u32x2 value_words[S::kTiles][S::kPlanes];
};

// From the registers of all quarters (GROUPS of them with words of their own, the others repeat these) those of every group.
template <int GROUPS>
__device__ __forceinline__ void OfQuarters(uint32_t v, uint32_t* to) {
  if constexpr (GROUPS == 1) {
    to[0] = v;
  } else if constexpr (GROUPS == 2) {
    const u32x2 r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    to[0] = r[0], to[1] = r[1];
  } else {
    const u32x2 r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    OfQuarters<2>(r[0], to);
    OfQuarters<2>(r[1], to + 2);
  }
}

// Waves on a SIMD, as many as their registers allow.
constexpr int FewOnSimd(int head_dim) { return head_dim == 256 ? 2 : head_dim == 128 ? 3 : 4; }

template <int D, int GJ, int WAVES, bool BIG>
__global__ __launch_bounds__(64 * WAVES, FewOnSimd(D)) void kv4_attention_few_kernel(const AttendParams p) {
  using S = FewShape<D, GJ>;
  constexpr int P = S::P, kPlanes = S::kPlanes, kCell = S::kCell, kGroups = S::kGroups, kKeyRegs = S::kKeyRegs, kTiles = S::kTiles, kStep = S::kStep;
  const Kv4Where& w = p.w;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;
  const int kv_head = blockIdx.y, s = blockIdx.z;
  const bool one_tile = (int)gridDim.x == p.parts;
  const int part = one_tile ? blockIdx.x : blockIdx.x % p.parts, tile0 = one_tile ? 0 : blockIdx.x / p.parts, tile_step = one_tile ? 1 : gridDim.x / p.parts;
  const int page_tokens = 1 << w.page_shift;
  const int32_t* table = w.table + (size_t)s * w.pages_per_sequence;
  // the first 64 pages, asked for with the lengths rather than after them
  const int first_pages = lane < w.pages_per_sequence ? table[lane] : -1;
  const Kv4Sequence q = Kv4SequenceOf(w, s);
  const int rows = q.count * p.share;
  if (rows < p.rows_from || rows > p.rows_to) return;
  __shared__ float4 sum_lds[WAVES][16][D / 4 + 1];
  __shared__ float2 ml_lds[WAVES][16];
  const Unpack unpack;
  const uint32_t key_at = (n * 4 + quad) * (P / 8), value_at = (quad * 16 + n) * (2 * kCell);  // a lane's piece of a tile's codes
  const uint32_t key_word_at = 32 * (quad % S::kGroupsAtOnce) + 2 * n;
  const uint32_t value_word_at = 32 * (n * kCell / (32 * GJ)) + 8 * quad;

  // (a sequence with one new token, the common case, divides nothing)
  auto token_of = [&](int row) { return q.count == 1 ? 0 : row / p.share; };
  for (int row0 = tile0 * 16; row0 < rows; row0 += tile_step * 16) {
    // the positions that the tile's rows see: [lo, hi), in steps dealt to the parts and, one by one, to their waves
    const int first_row = q.first + token_of(row0), last_row = q.first + token_of(min(rows, row0 + 16) - 1);
    const int hi = p.causal ? min(q.held, last_row + 1) : q.held;
    const int lo = p.window > 0 ? max(0, first_row + 1 - p.window) : 0;
    const int all_hi = p.causal ? min(q.held, first_row + 1) : q.held, all_lo = p.window > 0 ? last_row + 1 - p.window : 0;  // (what all of them see)
    const int step0 = lo / kStep, steps = hi > lo ? (hi - 1) / kStep + 1 - step0 : 0;
    const int each = p.parts == 1 ? steps : (steps + p.parts - 1) / p.parts;
    const int part_begin = step0 + min(steps, part * each), begin = part_begin + wave, end = step0 + min(steps, (part + 1) * each);

    // The pages of a step are looked up one step ahead of its bytes, and these asked for one step ahead of their use: a wave always has a
    // step's bytes in flight.  Pages of at least a step are one look-up and one address.  (Small pages: tiles behind the last held position
    // read the last one again; what they hold is masked.)
    constexpr int kIds = BIG ? 1 : kTiles;
    struct Ids {
      int id[kIds];
    };
    auto look_up = [&](int step) {
      Ids r;
#pragma unroll
      for (int u = 0; u < kIds; ++u) {
        const int page = BIG ? step * kStep >> w.page_shift : min(step * kTiles + u, (q.held - 1) >> 4) * 16 >> w.page_shift;
        r.id[u] = page < 64 ? __builtin_amdgcn_readlane(first_pages, page) : table[page];
      }
      return r;
    };
    auto block_of = [&](int step, const Ids& ids, int u) {
      const int id = ids.id[BIG ? 0 : u];
      return p.cache + ((size_t)(id >= 0 && id < w.pages ? id : 0) * w.kv_heads + kv_head) * w.block_bytes;
    };
    auto in_page_of = [&](int step, int u) { return (BIG ? step * kStep : min(step * kTiles + u, (q.held - 1) >> 4) * 16) & (page_tokens - 1); };
    constexpr int kCodes = 8 * D, kWordBytes = 32 * kGroups;  // of a tile
    auto load_keys = [&](int step, const Ids& ids, FewStep<D, GJ>& to) {
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        const uint8_t* block = block_of(step, ids, u);
        const int in_page = in_page_of(step, u), t = BIG ? u : 0;
        const uint8_t* kc = block + in_page * (D / 2);
        const uint8_t* kw = block + Kv4KeyWords(page_tokens, D) + in_page * kGroups * 2;
#pragma unroll
        for (int pl = 0; pl < kPlanes; ++pl) {
          if constexpr (P == 128) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(kc + key_at + t * kCodes + pl * 8 * P);
#pragma unroll
            for (int e = 0; e < 4; ++e) to.keys[u][4 * pl + e] = a[e];
          } else {
            const u32x2 a = *reinterpret_cast<const u32x2*>(kc + key_at + t * kCodes);
            to.keys[u][0] = a.x, to.keys[u][1] = a.y;
          }
        }
#pragma unroll
        for (int j = 0; j < S::kWordRegs; ++j) to.key_words[u][j] = *reinterpret_cast<const uint16_t*>(kw + key_word_at + t * kWordBytes + 128 * j);
      }
    };
    auto load_values = [&](int step, const Ids& ids, FewStep<D, GJ>& to) {
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        const uint8_t* block = block_of(step, ids, u);
        const int in_page = in_page_of(step, u), t = BIG ? u : 0;
        const uint8_t* vc = block + Kv4ValueCodes(page_tokens, D) + in_page * (D / 2);
        const uint8_t* vw = block + Kv4ValueWords(page_tokens, D, kGroups) + in_page * kGroups * 2;
#pragma unroll
        for (int pl = 0; pl < kPlanes; ++pl) {
          if constexpr (P == 128) {
            const u32x4 b = *reinterpret_cast<const u32x4*>(vc + value_at + t * kCodes + pl * 8 * P);
#pragma unroll
            for (int e = 0; e < 4; ++e) to.values[u][4 * pl + e] = b[e];
          } else {
            const u32x2 b = *reinterpret_cast<const u32x2*>(vc + value_at + t * kCodes);
            to.values[u][0] = b.x, to.values[u][1] = b.y;
          }
          to.value_words[u][pl] = *reinterpret_cast<const u32x2*>(vw + value_word_at + t * kWordBytes + 32 * (pl * P / (32 * GJ)));
        }
      }
    };
    FewStep<D, GJ> c;
    Ids ids, ids_next;
    if (begin < end) {
      ids = look_up(begin);
      load_keys(begin, ids, c);
      load_values(begin, ids, c);
      ids_next = look_up(min(begin + WAVES, end - 1));
    }

    u32x4 qa[kKeyRegs];  // operands of the first product: channel s and channel s + 4 of 8 in each register
    const int row = row0 + n;
    const bool there = row < rows;
    const int token = token_of(there ? row : 0), head = kv_head * p.share + (there ? row : 0) - token * p.share;
    // (one address of the lane and uniform strides: the lanes' own products would be hoisted out of the loop, two registers each)
    const u32x2* src = reinterpret_cast<const u32x2*>(p.q) + ((size_t)head * (D / 4) + 2 * quad) * w.tokens + q.start + token;
    const int position = q.first + token;
    // what the lane's row sees
    const int row_hi = there ? (p.causal ? min(q.held, position + 1) : q.held) : 0, row_lo = p.window > 0 ? max(0, position + 1 - p.window) : 0;
#pragma unroll
    for (int k = 0; k < kKeyRegs; ++k) {
      u32x2 a = {0u, 0u}, b = {0u, 0u};
      if (there) {
        a = src[(size_t)(8 * k) * w.tokens];
        b = src[(size_t)(8 * k + 1) * w.tokens];
      }
      qa[k] = u32x4{__builtin_amdgcn_perm(b.x, a.x, 0x05040100u), __builtin_amdgcn_perm(b.x, a.x, 0x07060302u),
                    __builtin_amdgcn_perm(b.y, a.y, 0x05040100u), __builtin_amdgcn_perm(b.y, a.y, 0x07060302u)};
    }

    float4_t acc[kPlanes][kCell];
    float top = -INFINITY, sum = 0.0f;
    bool far = false;
#pragma unroll
    for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
      for (int j = 0; j < kCell; ++j) acc[pl][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

    for (int step = begin; step < end; step += WAVES) {
      // The further a wave is in its step, the sooner its instructions go: the waves of a SIMD stay apart, one waits for its bytes while another
      // has the vector unit (32 sequences up to 4096, 8 heads of 128: 28.5 -> 28.1 us; 4 of 65536: 65.3 -> 61.1).
      __builtin_amdgcn_s_setprio(1);
      // scores: score[u][i] = q . k of row n and position 16 u + 4 quad + i
      float score[kTiles][4];
      uint32_t words[kGroups];
#pragma unroll
      for (int j = 0; j < S::kWordRegs; ++j) OfQuarters<S::kGroupsAtOnce>(c.key_words[0][j] | c.key_words[1][j] << 16, words + 4 * j);
#pragma unroll
      for (int u = 0; u < kTiles; ++u) {
        float4_t raw = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kKeyRegs; ++k) {
          const uint32_t a = c.keys[u][k], b = a >> 8, word = words[k / GJ];
          const half_t scale = AsHalf2(word & unpack.scale_mask)[u], low_zero = AsHalf2(unpack.Low(word))[u], high_zero = AsHalf2(unpack.High(word << 4))[u];
          const half2_t scales = {scale, scale}, low_zeros = {low_zero, low_zero}, high_zeros = {high_zero, high_zero};
          const u32x4 key = {AsU32((AsHalf2(unpack.Low(a)) - low_zeros) * scales), AsU32((AsHalf2(unpack.High(a)) - high_zeros) * scales),
                             AsU32((AsHalf2(unpack.Low(b)) - low_zeros) * scales), AsU32((AsHalf2(unpack.High(b)) - high_zeros) * scales)};
          raw = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, key), __builtin_bit_cast(half8_t, qa[k]), raw, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) score[u][i] = raw[i];
        // (a tile's products and sums at a time: left alone, the compiler puts all the step's products first and needs registers for them)
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(score[u][i]));
      }
      __builtin_amdgcn_s_setprio(2);
      // (the next step's keys come while this one's values are taken, and the other way round; behind the last step it comes again: branches
      // around the loads would have the next step wait for all of them)
      load_keys(min(step + WAVES, end - 1), ids_next, c);
      __builtin_amdgcn_sched_barrier(0);
      // a step inside what every row sees, on pages that there are, needs no masks
      bool whole = step * kStep + kStep <= all_hi && step * kStep >= all_lo;
#pragma unroll
      for (int u = 0; u < kIds; ++u) {
        const int id = __builtin_amdgcn_readfirstlane(ids.id[u]);  // (uniform: scalar comparisons)
        whole = whole && id >= 0 && id < w.pages;
      }
      if (!whole) {
#pragma unroll
        for (int u = 0; u < kTiles; ++u) {
          const int id = ids.id[BIG ? 0 : u];
          const bool there = id >= 0 && id < w.pages;
          const int at = step * kStep + 16 * u + 4 * quad;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!there || at + i >= row_hi || at + i < row_lo) score[u][i] = -INFINITY;
          // what lies behind the held positions may be anything: as values it is 0 (0 * NaN would not be)
#pragma unroll
          for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int two = at + 2 * i;
              c.value_words[u][pl][i] &= !there || two >= q.held ? 0u : two + 1 >= q.held ? 0x0000FFFFu : 0xFFFFFFFFu;
            }
        }
      }

      // the running maximum; what the new one is above the old scales the sums so far
      float best = score[0][0];
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) best = fmaxf(best, score[u][i]);
      best = MaxAcrossQuarters(best);
      if (__any(best > top)) {
        const float now = fmaxf(top, best);
        const float down = top == now ? 1.0f : __builtin_amdgcn_exp2f((top - now) * p.c);  // (-inf - finite: 0)
        top = now;
        far = __any(fabsf(top) * p.c > kFar && fabsf(top) != INFINITY);  // (a row of infinities is NaN either way, and its neighbours as without it)
        sum *= down;
#pragma unroll
        for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
          for (int j = 0; j < kCell; ++j) acc[pl][j] *= down;
      }

      half2_t prob[kTiles][2];
      float base = top == -INFINITY ? 0.0f : kLift - top * p.c;
      if (far) {
        base = top == -INFINITY ? 0.0f : kLift;
#pragma unroll
        for (int u = 0; u < kTiles; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) score[u][i] -= top == -INFINITY ? 0.0f : top;
      }
#pragma unroll
      for (int u = 0; u < kTiles; ++u)
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // (the sum takes the probabilities as the product does, rounded to halfs)
          const float a = __builtin_amdgcn_exp2f(fmaf(score[u][2 * i], p.c, base));
          const float b = __builtin_amdgcn_exp2f(fmaf(score[u][2 * i + 1], p.c, base));
          prob[u][i] = half2_t{(_Float16)a, (_Float16)b};
          sum = __builtin_amdgcn_fdot2(prob[u][i], half2_t{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
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
              const uint32_t word = c.value_words[u + v][pl][i];
              scale[v][i] = AsHalf2(word & unpack.scale_mask);
              low_zero[v][i] = AsHalf2(unpack.Low(word));
              high_zero[v][i] = AsHalf2(unpack.High(word << 4));
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
                  uint32_t word = c.values[u + v][(pl * (kCell / 4) + h) * 2 + i];
                  if (e >= 2) word >>= 8;
                  const half2_t x = (e & 1) ? AsHalf2(unpack.High(word)) - high_zero[v][i] : AsHalf2(unpack.Low(word)) - low_zero[v][i];
                  op[2 * v + i] = AsU32(x * scale[v][i]);
                }
              const u32x4 pr = {AsU32(prob[u][0]), AsU32(prob[u][1]), AsU32(prob[u + 1][0]), AsU32(prob[u + 1][1])};
              acc[pl][4 * h + e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  __builtin_bit_cast(half8_t, op), __builtin_bit_cast(half8_t, pr), acc[pl][4 * h + e], 0, 0, 0);
            }
        }
      }
      __builtin_amdgcn_s_setprio(0);
      load_values(min(step + WAVES, end - 1), ids_next, c);
      ids = ids_next;
      ids_next = look_up(min(step + 2 * WAVES, end - 1));
      __builtin_amdgcn_sched_barrier(0);
    }

    // the waves' outputs, at the common maximum
    sum = SumAcrossQuarters(sum);
    if (quad == 0) ml_lds[wave][n] = make_float2(top, sum);
    __syncthreads();
    float best = -INFINITY, total = 0.0f;
#pragma unroll
    for (int v = 0; v < WAVES; ++v) best = fmaxf(best, ml_lds[v][n].x);
#pragma unroll
    for (int v = 0; v < WAVES; ++v) {
      const float2 ml = ml_lds[v][n];
      total += ml.y * (ml.x == best ? 1.0f : __builtin_amdgcn_exp2f((ml.x - best) * p.c));
    }
    if (__any(total == 0.0f)) {
      const int from = max(row_lo, part_begin * kStep), to = min(row_hi, end * kStep);
      if (SeesAny(w, table, part_begin * kStep, min(q.held, end * kStep), from, total == 0.0f ? to : from)) total = __builtin_nanf("");
    }
    const float mine = top == best ? 1.0f : __builtin_amdgcn_exp2f((top - best) * p.c);
    const float factor = mine * (p.parts > 1 ? 1.0f : total > 0.0f ? 1.0f / total : total == 0.0f ? 0.0f : total);
    if (there)
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int h = 0; h < kCell / 4; ++h)
            sum_lds[wave][n][(pl * P + (4 * quad + i) * kCell) / 4 + h] =
              make_float4(acc[pl][4 * h][i] * factor, acc[pl][4 * h + 1][i] * factor, acc[pl][4 * h + 2][i] * factor,
                          acc[pl][4 * h + 3][i] * factor);
    __syncthreads();
    // the rows that there are x D / 4 slices
    const int mine_rows = min(16, rows - row0);
    for (int item = threadIdx.x; item < mine_rows * (D / 4); item += 64 * WAVES) {
      const int r = item / (D / 4), slice = item % (D / 4);
      const int row = row0 + r;
      float4 v = sum_lds[0][r][slice];
#pragma unroll
      for (int k = 1; k < WAVES; ++k) {
        const float4 o = sum_lds[k][r][slice];
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
      }
      const int of_sequence = token_of(row), head = kv_head * p.share + row - of_sequence * p.share;
      const size_t token = q.start + of_sequence;
      if (p.parts > 1) {
        reinterpret_cast<float4*>(p.part_o)[(((size_t)part * w.tokens + token) * p.heads + head) * (D / 4) + slice] = v;
      } else {
        const half2_t a = {(_Float16)v.x, (_Float16)v.y}, b = {(_Float16)v.z, (_Float16)v.w};
        reinterpret_cast<u32x2*>(p.out)[((size_t)head * (D / 4) + slice) * w.tokens + token] = u32x2{AsU32(a), AsU32(b)};
      }
    }
    if (p.parts > 1 && wave == 0 && quad == 0 && there) p.part_ml[((size_t)part * w.tokens + q.start + token) * p.heads + head] = make_float2(best, total);
    __syncthreads();  // (the arrays are written again)
  }
}

// Many rows for each key head (prompts and their chunks): matrix products bound it.  A work-group takes 32 rows of one key head to
// a wave, 8 waves (4 where head_dim is 256), and 16 positions for each wave at a time: it dequantizes them, exactly, into LDS, where all waves
// read all of them as operands of 32x32x16 products.
//   scores^T [32 positions][32 rows] = keys x q^T      a lane has one row (lane & 31) and 16 positions: 8 (i / 4) + 4 (lane >> 5) + i % 4
//   out^T [32 channels][32 rows]    += values^T x p^T   of 16 positions, those that the lanes hold: no exchange in between
// In LDS: keys [head_dim / 8][position 64] pieces of 8 channels; values [16 positions][half][slot] pieces of 8 positions of one channel, the
// positions that a lane of that half holds, the channels of a plane in the order (channel of the cell, cell): the writes of a wave and the
// reads of a product are runs of neighbouring pieces.
// The maximum of a row is left as it is while the scores stay within 2^kSlack of it: the outputs are scaled down rarely.  Probabilities are up
// to 2^(kManyLift + kSlack) = 2^14 then and keep 11 bits as halfs down to 2^-22 of the largest.
// Measured: 8192 tokens, 32 heads over 8 of 128 (550 GFLOP): 561 us, 980 TFLOP/s where a large library product reaches 1156.  Vector
// instructions take 59 % of a SIMD's cycles (exponentials 23, dequantizing 15), products 45 %: with one instruction issued at a time for a wave
// and two waves on a SIMD the two overlap little.  A fill, the first loads and the outputs of a work-group are 10 us around its steps.
constexpr float kManyLift = 8.0f, kSlack = 6.0f;  // (in powers of two)
constexpr int ManyWaves(int head_dim) { return head_dim == 256 ? 4 : 8; }

template <int D, int GJ>
__global__ __launch_bounds__(D == 256 ? 256 : 512, D == 256 ? 1 : 2) void kv4_attention_many_kernel(const AttendParams p) {
  constexpr int P = Kv4Plane(D), kPlanes = D / P, kWords = P / 32, kCell = P / 16, kGroups = D / 32 / GJ;
  constexpr int kKeyRegs = kPlanes * kWords, kValueRegs = kPlanes * kCell / 2;
  constexpr int kWaves = ManyWaves(D), kStep = 16 * kWaves, kRows = 32 * kWaves, kQ = D / 16, kTilesD = D / 32;
  const Kv4Where& w = p.w;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n = lane & 15, quad = lane >> 4;        // of a 16-position tile, dequantizing
  const int col = lane & 31, half = lane >> 5;      // of a product
  const int kv_head = blockIdx.x, s = blockIdx.z, part = blockIdx.y % p.parts;
  const Kv4Sequence q = Kv4SequenceOf(w, s);
  const int rows = q.count * p.share;
  if (rows < p.rows_from || rows > p.rows_to) return;
  const int page_tokens = 1 << w.page_shift;
  const int32_t* table = w.table + (size_t)s * w.pages_per_sequence;
  constexpr int kPieces = kStep * D / 8;
  __shared__ u32x4 lds[2 * 2 * kPieces];  // [2][keys, values]
  __shared__ int there_lds[2][kWaves];
  const Unpack unpack;

  const int row_tiles = (rows + kRows - 1) / kRows;
  for (int turn = blockIdx.y / p.parts; turn < row_tiles; turn += gridDim.y / p.parts) {
    const int row0 = (row_tiles - 1 - turn) * kRows;  // (the rows that see most first)
    const int first_row = q.first + row0 / p.share, last_row = q.first + (min(rows, row0 + kRows) - 1) / p.share;
    const int hi = p.causal ? min(q.held, last_row + 1) : q.held;
    const int lo = p.window > 0 ? max(0, first_row + 1 - p.window) : 0;
    const int step0 = lo / kStep, steps = hi > lo ? (hi - 1) / kStep + 1 - step0 : 0;
    const int each = (steps + p.parts - 1) / p.parts;
    const int begin = step0 + min(steps, part * each), end = step0 + min(steps, (part + 1) * each);

    // the bytes of a step are asked for one step ahead of the LDS, this is filled one step ahead of the products
    uint32_t keys[kKeyRegs], values[kValueRegs], key_words[kGroups];
    u32x2 value_words[kPlanes];
    bool there = false;
    // The page of a step is looked up with the bytes of the step before: a wave would wait for it.  By a vector load, in order with these:
    // scalar ones would be waited for with the next operands from LDS.
    int zero = 0, looked_up = 0;
    asm volatile("" : "+v"(zero));
    auto look_up = [&](int step) { looked_up = table[zero + (min(step * kWaves + wave, (q.held - 1) >> 4) * 16 >> w.page_shift)]; };
    auto load = [&](int step) {
      const int tile = min(step * kWaves + wave, (q.held - 1) >> 4);
      const int id = __builtin_amdgcn_readfirstlane(looked_up);
      there = id >= 0 && id < w.pages;
      const uint8_t* block = p.cache + ((size_t)(there ? id : 0) * w.kv_heads + kv_head) * w.block_bytes;
      const int in_page = (tile * 16) & (page_tokens - 1);
      const uint8_t* kc = block + in_page * (D / 2);
      const uint8_t* vc = block + Kv4ValueCodes(page_tokens, D) + in_page * (D / 2);
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl) {
        if constexpr (P == 128) {
          const u32x4 a = *reinterpret_cast<const u32x4*>(kc + pl * 8 * P + (n * 4 + quad) * 16);
          const u32x4 b = *reinterpret_cast<const u32x4*>(vc + pl * 8 * P + (quad * 16 + n) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) keys[4 * pl + e] = a[e], values[4 * pl + e] = b[e];
        } else {
          const u32x2 a = *reinterpret_cast<const u32x2*>(kc + (n * 4 + quad) * 8), b = *reinterpret_cast<const u32x2*>(vc + (quad * 16 + n) * 8);
          keys[0] = a.x, keys[1] = a.y, values[0] = b.x, values[1] = b.y;
        }
      }
      const uint16_t* kw = reinterpret_cast<const uint16_t*>(block + Kv4KeyWords(page_tokens, D)) + in_page * kGroups;
      const uint16_t* vw = reinterpret_cast<const uint16_t*>(block + Kv4ValueWords(page_tokens, D, kGroups)) + in_page * kGroups;
#pragma unroll
      for (int g = 0; g < kGroups; ++g) key_words[g] = kw[16 * g + n];
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl)
        value_words[pl] = *reinterpret_cast<const u32x2*>(vw + 16 * ((pl * P + n * kCell) / (32 * GJ)) + 4 * quad);
      look_up(step + 1);
    };
    // what lies behind the held positions may be anything: it is made 0 (0 * NaN would not be)
    auto clear = [&](int step, int buffer) {
      if (lane == 0) there_lds[buffer][wave] = there;
      const int valid = there ? q.held - (step * kStep + wave * 16) : 0;
      if (valid < 16) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g)
          if (n >= valid) key_words[g] = 0;
#pragma unroll
        for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int two = 4 * quad + 2 * i;
            value_words[pl][i] &= two >= valid ? 0u : two + 1 >= valid ? 0x0000FFFFu : 0xFFFFFFFFu;
          }
      }
    };
    // into LDS, a plane of channels at a time
    auto dequantize = [&](int buffer, int pl) {
      u32x4* kb = lds + buffer * 2 * kPieces;
#pragma unroll
      for (int g = pl * (P / 32 / GJ); g < (pl + 1) * (P / 32 / GJ); ++g) {
        const uint32_t word = key_words[g] | key_words[g] << 16;
        const half2_t scale = AsHalf2(word & unpack.scale_mask), low_zero = AsHalf2(unpack.Low(word)), high_zero = AsHalf2(unpack.High(word << 4));
#pragma unroll
        for (int k = g * GJ; k < (g + 1) * GJ; ++k) {
          const uint32_t a = keys[k], b = a >> 8;
          const u32x4 piece = {AsU32((AsHalf2(unpack.Low(a)) - low_zero) * scale), AsU32((AsHalf2(unpack.High(a)) - high_zero) * scale),
                               AsU32((AsHalf2(unpack.Low(b)) - low_zero) * scale), AsU32((AsHalf2(unpack.High(b)) - high_zero) * scale)};
          kb[(4 * k + quad) * kStep + wave * 16 + n] = piece;
        }
      }
      u32x2* v2 = reinterpret_cast<u32x2*>(kb + kPieces + (wave * 2 + (quad & 1)) * D) + (quad >> 1);
      half2_t scale[2], low_zero[2], high_zero[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t word = value_words[pl][i];
        scale[i] = AsHalf2(word & unpack.scale_mask);
        low_zero[i] = AsHalf2(unpack.Low(word));
        high_zero[i] = AsHalf2(unpack.High(word << 4));
      }
#pragma unroll
      for (int h = 0; h < kCell / 4; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          u32x2 piece;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            uint32_t word = values[(pl * (kCell / 4) + h) * 2 + i];
            if (e >= 2) word >>= 8;
            const half2_t x = (e & 1) ? AsHalf2(unpack.High(word)) - high_zero[i] : AsHalf2(unpack.Low(word)) - low_zero[i];
            piece[i] = AsU32(x * scale[i]);
          }
          v2[2 * (pl * P + (4 * h + e) * 16 + n)] = piece;
        }
    };

    if (begin < end) look_up(begin);

    const int wave_row = row0 + wave * 32, row = wave_row + col;
    const bool is_row = row < rows;
    const int token = q.start + (is_row ? row : 0) / p.share, head = kv_head * p.share + (is_row ? row : 0) % p.share;
    const int position = q.first + (is_row ? row : 0) / p.share;
    const int row_hi = is_row ? (p.causal ? min(q.held, position + 1) : q.held) : 0, row_lo = p.window > 0 ? max(0, position + 1 - p.window) : 0;
    u32x4 qa[kQ];
    {
      const u32x2* src = reinterpret_cast<const u32x2*>(p.q) + ((size_t)head * (D / 4) + 2 * half) * w.tokens + token;
#pragma unroll
      for (int k = 0; k < kQ; ++k) {  // (behind the last row: the first one again)
        const u32x2 a = src[(size_t)(4 * k) * w.tokens], b = src[(size_t)(4 * k + 1) * w.tokens];
        qa[k] = u32x4{__builtin_amdgcn_perm(b.x, a.x, 0x05040100u), __builtin_amdgcn_perm(b.x, a.x, 0x07060302u),
                      __builtin_amdgcn_perm(b.y, a.y, 0x05040100u), __builtin_amdgcn_perm(b.y, a.y, 0x07060302u)};
      }
    }
    if (begin < end) load(begin);  // (behind the rows' own loads: these wait for no page)
    // what all of the wave's rows see, and what any of them does
    const int wave_first = q.first + min(wave_row, rows - 1) / p.share, wave_last = q.first + min(wave_row + 31, rows - 1) / p.share;
    const int all_hi = p.causal ? min(q.held, wave_first + 1) : q.held, all_lo = p.window > 0 ? max(0, wave_last + 1 - p.window) : 0;
    const int any_hi = wave_row >= rows ? 0 : p.causal ? min(q.held, wave_last + 1) : q.held, any_lo = p.window > 0 ? max(0, wave_first + 1 - p.window) : 0;

    float16_t acc[kTilesD];
    float top = -INFINITY, sum = 0.0f;
    bool far = false;
#pragma unroll
    for (int j = 0; j < kTilesD; ++j)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[j][i] = 0.0f;

    // A step against the wave's rows, 32 positions at a time: the products of the next 32 positions' scores run under the exponentials of
    // these, and every chunk of products has its operands asked for a chunk ahead.
    constexpr int kAhead = 4, kSubs = kStep / 32;
    float16_t bias;
#pragma unroll
    for (int i = 0; i < 16; ++i) bias[i] = 0.0f;
    // heads of 256: the outputs stay in accumulation registers, from which products are added up directly; the rare scaling down moves them
    // out and back (the compiler by itself keeps them where that is quick, and moves all of them around every product)
    auto settle = [&] {
      if constexpr (D == 256) {
#pragma unroll
        for (int j = 0; j < kTilesD; ++j) asm volatile("" : "+a"(acc[j]));
#pragma unroll
        for (int k = 0; k < kQ; ++k) asm volatile("" : "+a"(qa[k]));
      }
    };
    auto attend = [&](int step, int buffer, bool whole) {
      const u32x4* kb = lds + buffer * 2 * kPieces + half * kStep + col;
      const u32x4* vb = lds + buffer * 2 * kPieces + kPieces + half * D + col;
      // operand number k of the scores of all the step's positions, number t of its values' products
      auto key_piece = [&](int k) { return kb[2 * (k % kQ) * kStep + k / kQ * 32]; };
      auto value_piece = [&](int t) { return vb[t / kTilesD * 2 * D + t % kTilesD * 32]; };
      u32x4 kf[kAhead], vf[kAhead];
      float16_t x[2];
      // in steps that not every row sees whole: what the sums of products start from, 0 or -inf where the row does not see the position
      auto start = [&](int sub) {
        if (whole) return;
        const int at = step * kStep + sub * 32 + 4 * half;
        const int from = row_lo - at;
        const int to[2] = {there_lds[buffer][sub * 2] ? row_hi - at : -1, there_lds[buffer][sub * 2 + 1] ? row_hi - at : -1};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int k = 8 * (i / 4) + i % 4;
          bias[i] = k < to[i / 8] && k >= from ? 0.0f : -INFINITY;
        }
      };
      auto key_product = [&](int sub, int k, float16_t& v) {
        v = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, kf[k % kAhead]), __builtin_bit_cast(half8_t, qa[k]), k == 0 ? bias : v, 0, 0, 0);
        if (sub * kQ + k + kAhead < kSubs * kQ) kf[k % kAhead] = key_piece(sub * kQ + k + kAhead);
      };
#pragma unroll
      for (int f = 0; f < kAhead; ++f) kf[f] = key_piece(f);
#pragma unroll
      for (int f = 0; f < kAhead; ++f) vf[f] = value_piece(f);
      start(0);
#pragma unroll
      for (int k = 0; k < kQ; ++k) {
        key_product(0, k, x[0]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int sub = 0; sub < kSubs; ++sub) {
        float16_t &now = x[sub & 1], &next = x[(sub & 1) ^ 1];
        float best = now[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) best = fmaxf(best, now[i]);
        const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(best), __float_as_uint(best), false, false);
        best = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
        settle();
        if (__any(best > top && !((best - top) * p.c <= kSlack))) {
          const float higher = fmaxf(top, best);
          const float down = top == higher ? 1.0f : __builtin_amdgcn_exp2f((top - higher) * p.c);
          top = higher;
          far = __any(fabsf(top) * p.c > kFar && fabsf(top) != INFINITY);  // (a row of infinities is NaN either way, and its neighbours as without it)
          if (__any(sum != 0.0f)) {  // (not the first of the positions: nothing to scale)
            sum *= down;
#pragma unroll
            for (int j = 0; j < kTilesD; ++j)
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[j][i] *= down;
          }
        }
        settle();
        float base = top == -INFINITY ? 0.0f : kManyLift - top * p.c;
        if (far) {
          base = top == -INFINITY ? 0.0f : kManyLift;
#pragma unroll
          for (int i = 0; i < 16; ++i) now[i] -= top == -INFINITY ? 0.0f : top;
        }
        if (sub + 1 < kSubs) start(sub + 1);
        __builtin_amdgcn_sched_barrier(0);
        u32x4 prob[2];
        // two waves on a SIMD: the one with products goes first, the other's vector work fills in (8192 tokens, 32 heads of 128: 576 -> 567 us)
        if (kWaves == 8) __builtin_amdgcn_s_setprio(1);
        if (sub + 1 < kSubs) {
#pragma unroll
          for (int k = 0; k < kQ; ++k) key_product(sub + 1, k, next);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = __builtin_amdgcn_exp2f(fmaf(now[2 * i], p.c, base)), v = __builtin_amdgcn_exp2f(fmaf(now[2 * i + 1], p.c, base));
          const half2_t two = {(_Float16)u, (_Float16)v};
          sum = __builtin_amdgcn_fdot2(two, half2_t{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
          prob[i / 4][i % 4] = AsU32(two);
        }
        if (sub + 1 < kSubs) {  // a product, the operand of a later one, and what of the exponentials the product hides
#pragma unroll
          for (int k = 0; k < kQ; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 48 / kQ, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 2 * kTilesD; ++t) {
          acc[t % kTilesD] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_t, vf[t % kAhead]), __builtin_bit_cast(half8_t, prob[t / kTilesD]),
                                                                  acc[t % kTilesD], 0, 0, 0);
          if (sub * 2 * kTilesD + t + kAhead < kSubs * 2 * kTilesD) vf[t % kAhead] = value_piece(sub * 2 * kTilesD + t + kAhead);
          if (D != 256) __builtin_amdgcn_sched_barrier(0);
        }
        if (kWaves == 8) __builtin_amdgcn_s_setprio(0);
        if constexpr (D == 256) {
          // one wave on a SIMD: its share of filling the other buffer goes under these products (behind the last step it is filled with what
          // is at hand and not looked at)
          static_assert(kSubs == kPlanes || D != 256);
          dequantize(buffer ^ 1, sub);
#pragma unroll
          for (int t = 0; t < 2 * kTilesD; ++t) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, 10, 0);
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (!whole) {
#pragma unroll
        for (int i = 0; i < 16; ++i) bias[i] = 0.0f;
      }
    };

    const auto fill = [&](int step) {  // the buffer of a step that there is
      clear(step, (step - begin) & 1);
#pragma unroll
      for (int pl = 0; pl < kPlanes; ++pl) dequantize((step - begin) & 1, pl);
    };
    if (begin < end) {
      fill(begin);
      if (begin + 1 < end) load(begin + 1);
    }
    __syncthreads();
    for (int step = begin; step < end; ++step) {
      const int buffer = (step - begin) & 1, at = step * kStep;
      const bool more = step + 1 < end, sees = at < any_hi && at + kStep > any_lo;
      settle();
      // eight waves: the two of a SIMD fill the other buffer at different ends of the step, so that one's products meet the other's vector work
      if (kWaves == 8 && wave >= 4 && more) {
        fill(step + 1);
        if (step + 2 < end) load(step + 2);
      }
      if (sees) {
        const bool whole = at >= all_lo && at + kStep <= all_hi;
        int all_there = 1;
#pragma unroll
        for (int u = 0; u < kWaves; ++u) all_there &= there_lds[buffer][u];
        if (kWaves == 4 && more) clear(step + 1, buffer ^ 1);
        attend(step, buffer, whole && __builtin_amdgcn_readfirstlane(all_there));
      }
      settle();
      if ((kWaves == 4 ? !sees : wave < 4) && more) fill(step + 1);
      if ((kWaves == 4 || wave < 4) && step + 2 < end) load(step + 2);
      __syncthreads();
    }

    const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    float total = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    if (__any(!(total > 0.0f))) {
      const int same_row = wave_row + LaneHere() % 32, at = q.first + (same_row < rows ? same_row : 0) / p.share;
      const int from = max(p.window > 0 ? at + 1 - p.window : 0, begin * kStep), to = min(p.causal ? min(q.held, at + 1) : q.held, end * kStep);
      const bool none = !(total > 0.0f), sees = SeesAny(w, table, begin * kStep, min(q.held, end * kStep), from, none && same_row < rows ? to : from);
      if (none) total = sees ? __builtin_nanf("") : 0.0f;
    }
    if (is_row) {
      const float factor = p.parts > 1 ? 1.0f : 1.0f / total;
      auto store = [&](auto to) {  // to(slice behind the half's own first, its 4 channels)
#pragma unroll
        for (int pl = 0; pl < kPlanes; ++pl)
#pragma unroll
          for (int m = 0; m < 8; ++m)  // cells 8 (m / 4) + 4 half + m % 4
#pragma unroll
            for (int h = 0; h < kCell / 4; ++h) {
              float v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = acc[pl * (kCell / 2) + (4 * h + e) / 2][8 * (e % 2) + m] * factor;
              to((pl * P + (8 * (m / 4) + m % 4) * kCell) / 4 + h, v);
            }
      };
      if (p.parts > 1) {
        float4* to = reinterpret_cast<float4*>(p.part_o) + (((size_t)part * p.heads + head) * (D / 4) + half * kCell) * w.tokens + token;
        store([&](int slice, const float(&v)[4]) { to[(size_t)slice * w.tokens] = make_float4(v[0], v[1], v[2], v[3]); });
        if (half == 0) p.part_ml[((size_t)part * w.tokens + token) * p.heads + head] = make_float2(top, total);
      } else {
        u32x2* to = reinterpret_cast<u32x2*>(p.out) + ((size_t)head * (D / 4) + half * kCell) * w.tokens + token;
        if (total > 0.0f) {
          store([&](int slice, const float(&v)[4]) {
            const half2_t a = {(_Float16)v[0], (_Float16)v[1]}, b = {(_Float16)v[2], (_Float16)v[3]};
            to[(size_t)slice * w.tokens] = u32x2{AsU32(a), AsU32(b)};
          });
        } else {  // 0 or NaN, whatever the sums are
          const half2_t same = {(_Float16)total, (_Float16)total};
          store([&](int slice, const float(&)[4]) { to[(size_t)slice * w.tokens] = u32x2{AsU32(same), AsU32(same)}; });
        }
      }
    }
  }
}

// The parts of each row, joined: everything is asked for before the first wait (the loads of the parts' outputs do not depend on their
// sums), and nothing is looked up but where the first sequence begins and the last one ends; where both kernels above have a share of the
// batch, sequence by sequence, those of one kernel only.
struct JoinParams {
  Kv4Where w;
  const float* part_o;
  const float2* part_ml;
  __half* out;
  int heads, parts;
  float c;
  int share, rows_from, rows_to;  // sequence by sequence: those of rows_from .. rows_to rows
  int many;                       // the order of part_o
  // slice 0 of a row's outputs, and how far its slices are apart
  __device__ __forceinline__ const float4* First(int slices, int token, int head) const {
    return reinterpret_cast<const float4*>(part_o) + (many ? (size_t)head * slices * w.tokens + token : ((size_t)token * heads + head) * slices);
  }
  __device__ __forceinline__ size_t Apart() const { return many ? w.tokens : 1; }
};
constexpr int kMostParts = 256, kFewParts = 8;
// Rows of a sequence up to which the kernel for few rows serves it.  It does a tile of 16 rows at a time, the other one up to 256 at once.
// Few against many, 8 sequences of 2048 positions / 32 of 4096.  8 key heads of 128: 19.2, 22.8 / 77.8, 82.2 us at 48 rows, 20.5, 25.5 / 101.1, 94.3 at 64.
// 8 of 64: 14.6, 18.2 / 50.1, 51.7 at 48, 24.6, 22.2 / 126.0, 70.7 at 128.  One of 256: 16.9, 22.4 / 35.0, 38.5 at 64, 18.6, 31.4 / 50.7, 46.9 at 128.
constexpr int FewRows(int head_dim) { return head_dim == 256 ? 128 : 48; }

// Of a part the weight in a row whose largest maximum is `best`: 0 where it saw nothing, whatever its output holds.
__device__ __forceinline__ float PartFactor(float2 ml, float best, float c) {
  return ml.y == 0.0f ? 0.0f : ml.x == best ? 1.0f : __builtin_amdgcn_exp2f((ml.x - best) * c);
}
__device__ __forceinline__ u32x2 Joined(const float4& v, float total) {
  const float g = total == 0.0f ? 0.0f : 1.0f / total;
  const half2_t a = {(_Float16)(v.x * g), (_Float16)(v.y * g)}, b = {(_Float16)(v.z * g), (_Float16)(v.w * g)};
  return u32x2{AsU32(a), AsU32(b)};
}

// Few parts: a work-group takes 8 neighbouring tokens of one head, so that stores are runs of 64 bytes and loads of 128; a thread has one
// token, and one or two slices in all parts.
template <int D, bool BY_SEQUENCE>
__global__ __launch_bounds__(256) void kv4_attention_join_kernel(const JoinParams p) {
  constexpr int kSlices = D / 4, kTokens = 8, kThreads = D == 64 ? 128 : 256, kItems = kTokens * kSlices / kThreads;
  const Kv4Where& w = p.w;
  const int block = blockIdx.x / p.heads, head = blockIdx.x - block * p.heads;
  int token = block * kTokens + threadIdx.x % kTokens;
  if constexpr (BY_SEQUENCE) {
    const Kv4Sequence q = Kv4SequenceOf(w, blockIdx.y);
    const int rows = q.count * p.share;
    if (rows < p.rows_from || rows > p.rows_to || token >= q.count) return;
    token += q.start;
  }
  if (token >= w.tokens) return;
  const size_t rows = (size_t)w.tokens * p.heads, row = (size_t)token * p.heads + head;
  const int slice0 = threadIdx.x / kTokens;
  const size_t apart = p.Apart();
  const float4* from = p.First(kSlices, token, head) + slice0 * apart;
  float2 ml[kFewParts];
  float4 o[kFewParts][kItems];
#pragma unroll
  for (int k = 0; k < kFewParts; ++k)
    if (k < p.parts) {
      ml[k] = p.part_ml[k * rows + row];
#pragma unroll
      for (int i = 0; i < kItems; ++i) o[k][i] = from[k * rows * kSlices + i * (kThreads / kTokens) * apart];
    }
  if (!BY_SEQUENCE && (token < w.starts[0] || token >= w.starts[w.sequences])) return;  // of no sequence
  float best = -INFINITY;
#pragma unroll
  for (int k = 0; k < kFewParts; ++k)
    if (k < p.parts) best = fmaxf(best, ml[k].x);
  float total = 0.0f;
  float4 v[kItems];
#pragma unroll
  for (int i = 0; i < kItems; ++i) v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < kFewParts; ++k)
    if (k < p.parts) {
      const float f = PartFactor(ml[k], best, p.c);
      total += ml[k].y * f;
      if (f != 0.0f)
#pragma unroll
        for (int i = 0; i < kItems; ++i) v[i].x += o[k][i].x * f, v[i].y += o[k][i].y * f, v[i].z += o[k][i].z * f, v[i].w += o[k][i].w * f;
    }
#pragma unroll
  for (int i = 0; i < kItems; ++i)
    reinterpret_cast<u32x2*>(p.out)[((size_t)head * kSlices + slice0 + i * (kThreads / kTokens)) * w.tokens + token] = Joined(v[i], total);
}

// Many parts: a work-group takes one row, its threads share the slices and, in turn, the parts.
template <int D, bool BY_SEQUENCE>
__global__ __launch_bounds__(256) void kv4_attention_join_many_kernel(const JoinParams p) {
  constexpr int kSlices = D / 4, kTurns = 256 / kSlices, kFirst = 4;
  const Kv4Where& w = p.w;
  const int thread = threadIdx.x, slice = thread % kSlices, turn = thread / kSlices;
  const size_t rows = (size_t)w.tokens * p.heads;
  size_t row = blockIdx.x;
  if constexpr (BY_SEQUENCE) {
    const Kv4Sequence q = Kv4SequenceOf(w, blockIdx.y);
    const int of_sequence = q.count * p.share;
    if (of_sequence < p.rows_from || of_sequence > p.rows_to || row >= (size_t)q.count * p.heads) return;
    row += (size_t)q.start * p.heads;
  }
  __shared__ float factors[kMostParts];
  __shared__ float4 sums[kTurns][kSlices];
  __shared__ float2 of_wave[4];
  float2 ml = make_float2(-INFINITY, 0.0f);
  if (thread < p.parts) ml = p.part_ml[thread * rows + row];  // each part's: a thread per part
  const int token = (int)(row / p.heads), head = (int)(row - (size_t)token * p.heads);
  const float4* from = p.First(kSlices, token, head) + slice * p.Apart();
  float4 first[kFirst];
#pragma unroll
  for (int j = 0; j < kFirst; ++j) first[j] = turn + j * kTurns < p.parts ? from[(turn + j * kTurns) * rows * kSlices] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (token < w.starts[0] || token >= w.starts[w.sequences]) return;  // of no sequence (the whole row)
  float best = ml.x;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) best = fmaxf(best, __shfl_xor(best, off));
  if ((thread & 63) == 0) of_wave[thread >> 6].x = best;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 4; ++k) best = fmaxf(best, of_wave[k].x);
  const float f = PartFactor(ml, best, p.c);
  float total = ml.y * f;
#pragma unroll
  for (int off = 1; off < 64; off *= 2) total += __shfl_xor(total, off);
  factors[thread] = f;
  if ((thread & 63) == 0) of_wave[thread >> 6].y = total;
  __syncthreads();
  total = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) total += of_wave[k].y;
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](int k, const float4& o) {
    const float g = factors[k];
    if (g != 0.0f) v.x += o.x * g, v.y += o.y * g, v.z += o.z * g, v.w += o.w * g;
  };
#pragma unroll
  for (int j = 0; j < kFirst; ++j)
    if (turn + j * kTurns < p.parts) add(turn + j * kTurns, first[j]);
  for (int k = kFirst * kTurns + turn; k < p.parts; k += kTurns) add(k, from[k * rows * kSlices]);
  sums[turn][slice] = v;
  __syncthreads();
  if (turn != 0) return;
#pragma unroll
  for (int k = 1; k < kTurns; ++k) {
    const float4 o = sums[k][slice];
    v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
  }
  reinterpret_cast<u32x2*>(p.out)[((size_t)head * kSlices + slice) * w.tokens + token] = Joined(v, total);
}

template <int D, int GJ>
void Launch(const Kv4AttentionArgs& a, hipStream_t stream) {
  const Kv4AttentionPlan& plan = a.plan;
  const int share = a.heads / a.where.kv_heads, most_new = std::min(a.max_new, a.where.tokens);
  AttendParams p;
  p.w = a.where;
  p.q = static_cast<const __half*>(a.q);
  p.cache = a.cache;
  p.out = static_cast<__half*>(a.out);
  p.heads = a.heads;
  p.share = share;
  p.causal = a.causal;
  p.window = a.window;
  p.c = a.scale * kLog2e;
  p.part_o = a.partial;
  p.part_ml = reinterpret_cast<float2*>(a.partial + (size_t)std::max(plan.few_parts, plan.many_parts) * a.max_tokens * a.heads * D);
  const bool both = plan.few_rows > 0 && plan.few_rows < INT32_MAX;
  auto join = [&](int of, int rows_from, int rows_to, int many) {
    if (of == 1) return;
    const JoinParams j = {a.where, p.part_o, p.part_ml, p.out, a.heads, of, p.c, share, rows_from, rows_to, many};
    // (a launch of more rows of a sequence than the op was made for: as many as the tensors have)
    const int tokens = both && rows_to < INT32_MAX ? rows_to / share : a.where.tokens, sequences = both ? a.where.sequences : 1;
    if (of <= kFewParts) {
      const dim3 grid(DivUp(tokens, 8) * a.heads, sequences);
      both ? kv4_attention_join_kernel<D, true><<<grid, D == 64 ? 128 : 256, 0, stream>>>(j) : kv4_attention_join_kernel<D, false><<<grid, D == 64 ? 128 : 256, 0, stream>>>(j);
    } else {
      const dim3 grid(tokens * a.heads, sequences);
      both ? kv4_attention_join_many_kernel<D, true><<<grid, 256, 0, stream>>>(j) : kv4_attention_join_many_kernel<D, false><<<grid, 256, 0, stream>>>(j);
    }
  };
  // (one kernel's parts are joined before the other's are written: their orders are not the same)
  if (plan.few_rows > 0) {
    p.parts = plan.few_parts;
    p.rows_from = 1;
    p.rows_to = plan.few_rows;
    const int row_tiles = std::min(DivUp(std::min(most_new * share, plan.few_rows), 16), 16384);  // (more are taken in turn)
    const dim3 grid(p.parts * row_tiles, a.where.kv_heads, a.where.sequences);
    constexpr int kFull = 4 * FewOnSimd(D);
    const bool big = a.where.page_shift >= 5;
    if (plan.few_waves == kFull)
      big ? kv4_attention_few_kernel<D, GJ, kFull, true><<<grid, 64 * kFull, 0, stream>>>(p) : kv4_attention_few_kernel<D, GJ, kFull, false><<<grid, 64 * kFull, 0, stream>>>(p);
    else
      big ? kv4_attention_few_kernel<D, GJ, 4, true><<<grid, 256, 0, stream>>>(p) : kv4_attention_few_kernel<D, GJ, 4, false><<<grid, 256, 0, stream>>>(p);
    join(plan.few_parts, 1, plan.few_rows, 0);
  }
  if (plan.few_rows < INT32_MAX) {
    p.parts = plan.many_parts;
    p.rows_from = plan.few_rows + 1;
    p.rows_to = INT32_MAX;
    const dim3 grid(a.where.kv_heads, std::min(p.parts * DivUp(most_new * share, 32 * ManyWaves(D)), 65535 / p.parts * p.parts), a.where.sequences);
    kv4_attention_many_kernel<D, GJ><<<grid, 64 * ManyWaves(D), 0, stream>>>(p);
    join(plan.many_parts, plan.few_rows + 1, INT32_MAX, 1);
  }
}

}  // namespace

Kv4AttentionPlan PlanKv4Attention(const Kv4AttentionArgs& a) {
  const Tuning& t = GetTuning();
  Kv4AttentionPlan plan;
  const int share = a.heads / a.where.kv_heads, most_new = std::min(a.max_new, a.max_tokens);
  const long long rows = (long long)most_new * share, heads = (long long)a.where.sequences * a.where.kv_heads;
  const long long keys = (long long)a.where.pages_per_sequence << a.where.page_shift;
  const int few_rows = FewRows(a.head_dim);
  const bool many = t.kv4_many >= 0 ? t.kv4_many > 0 : rows > few_rows;
  // In a ragged batch sequences of few rows go to the kernel for few where they could be many, or see more than the prompts' own work-groups
  // take anyway; else a work-group of the other kernel each, beside the prompts', costs less than one more launch.
  const long long seen = a.window > 0 ? std::min<long long>(keys, a.window) : keys;
  plan.few_rows = !many ? INT32_MAX : a.where.sequences > 1 && share <= few_rows && (heads >= 64 || seen > 4096) ? few_rows : 0;
  // tiles of rows in a batch: sequences of the most rows, but no more rows than the tensors have
  const auto row_tiles = [&](long long most, int tile) {
    return std::min(heads * ((most + tile - 1) / tile), a.where.kv_heads * ((long long)a.max_tokens * share / tile + a.where.sequences));
  };
  // the parts' outputs: at most 256 MB
  const long long row_bytes = (long long)a.max_tokens * a.heads * (a.head_dim + 2) * 4, room = ((long long)256 << 20) / row_bytes;
  const auto parts = [&](long long v) { return (int)std::max(1LL, std::min({v, room, (long long)kMostParts})); };
  if (plan.few_rows > 0) {
    const long long few_keys = a.window > 0 ? std::min<long long>(keys, a.window + most_new) : keys;  // that a tile may see
    const long long groups = row_tiles(many ? std::min<long long>(rows, few_rows) : rows, 16);
    // Work-groups of all the waves that a CU holds where they fill the CUs and each wave has a step: fewer outputs to join, none with as many
    // tiles as CUs (32 sequences of up to 4096 positions, 8 key heads of 128: 28.2 us against 29.0 in 3 parts of 4 waves; 16 of up to 2047,
    // four tokens each, 16 heads of 64: 15.8 against 16.4 in 4).  Else work-groups of 4 waves, as many as are on the chip at once (one sequence of
    // 1000 positions, a key head of 256: 11.1 us in 8 of them, 17.8 in one).
    const int full = 4 * FewOnSimd(a.head_dim), waves = 256 * full;  // of a CU; of the chip
    // And where one such work-group has a step for each wave: no second kernel (one sequence of 256 positions, 8 heads of 128: 6.9 us against 9.6
    // from the host, 6.6 against 7.6 in a graph; of 512, heads of 64: 7.2 / 9.9 and 7.1 / 6.7; up to 128 positions are one of 4 waves).
    const bool fills = 256 / groups * groups >= 192 && 256 / groups * 32 * full <= few_keys, one_step = few_keys > 128 && few_keys <= 32 * full;
    plan.few_waves = groups <= 256 && (fills || one_step) ? full : 4;
    plan.few_parts = parts(t.kv4_parts > 0 ? std::min<long long>(t.kv4_parts, (keys + 127) / 128)
                                             : std::min(waves / plan.few_waves / groups, (few_keys + 32 * plan.few_waves - 1) / (32 * plan.few_waves)));
  }
  if (many) {
    // Parts level the work-groups' shares, and their outputs go through memory: the number with the least estimated time.  Steps that the
    // longest work-group takes, and those that each of the 256 takes where they are level; a step and a byte by what they measured.
    const int step = 16 * ManyWaves(a.head_dim), tile = 32 * ManyWaves(a.head_dim);
    const double step_us = a.head_dim == 64 ? 2.7 : a.head_dim == 128 ? 3.7 : 2.6, around_us = 10;  // (before the first step and behind the last)
    const double groups = (double)row_tiles(rows, tile), longest = std::max<double>(1, (double)(a.window > 0 ? std::min<long long>(keys, a.window + tile / share) : keys) / step);
    const double level = groups * longest / 256 * (a.window > 0 || !a.causal ? 1.0 : 1.0 - 0.5 * std::min<double>(1, (double)most_new / keys));
    double least = 0;
    for (int n = 1; n <= kMostParts && n <= std::max(1.0, longest / 2); ++n) {
      const double steps = groups * n <= 256 ? longest / n : level + 0.5 * longest / n;
      const double us = steps * step_us + around_us * std::max(1.0, groups * n / 256) + (n > 1 ? 5 + 2 * n * (double)row_bytes / 4.5e6 : 0);
      if (n > 1 && us >= least) continue;
      least = us;
      plan.many_parts = n;
    }
    plan.many_parts = parts(t.kv4_parts > 0 ? std::min<long long>(t.kv4_parts, (keys + 127) / 128) : plan.many_parts);
  }
  return plan;
}

hipError_t LaunchKv4Attention(const Kv4AttentionArgs& a, hipStream_t stream, const char** kernel_name) {
  const bool many = a.plan.few_rows < INT32_MAX;
  *kernel_name = many ? "kv4_attention_many_kernel" : "kv4_attention_few_kernel";
  SetVariant(a.variant, !many ? "few" : a.plan.few_rows > 0 ? "many, few" : "many");
  SetTiles(a.tiles, many ? 32 * ManyWaves(a.head_dim) : 16, many ? ManyWaves(a.head_dim) : a.plan.few_waves, many ? a.plan.many_parts : a.plan.few_parts);
  const int gj = 1 << (a.where.group_shift - 5);
  if (a.head_dim == 64)
    gj == 1 ? Launch<64, 1>(a, stream) : Launch<64, 2>(a, stream);
  else if (a.head_dim == 128)
    gj == 1 ? Launch<128, 1>(a, stream) : gj == 2 ? Launch<128, 2>(a, stream) : Launch<128, 4>(a, stream);
  else
    gj == 1 ? Launch<256, 1>(a, stream) : gj == 2 ? Launch<256, 2>(a, stream) : Launch<256, 4>(a, stream);
  return hipGetLastError();
}

}  // namespace mldhip
