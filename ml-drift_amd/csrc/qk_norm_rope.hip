// Norms of the query and key heads and the rotation by position, in one pass over the tensors of the q and k projections.
//
//   y = x / sqrt(mean(x^2) + eps) * (weight_offset + weight)      over the head_dim channels of a head (left out without norms)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t)              for every pair of the first rotary_dim channels, t = position * f_i
//
// in fp32, rounded once to the tensor's type.  Memory bounds it: every channel is read and written once.  4096 tokens, 40 heads of 128 halfs (84 MB):
// 18.2 us, 4.6 TB/s where a large copy reaches 4.9.  Small launches are bound by the launch and by loads that wait for each other (the position, the table's
// entries one by one, the channels, the weights): one token is 2.9 us, 777 fp32 tokens of 32 heads of 64 4.7 where the bytes take 2.6.
//
// The angle.  position * f_i in fp32 is off by position * 2^-24 radians, 0.06 at a million.  f_i / (2 pi) is held as a 64-bit fraction of
// a turn instead (a table of the op): the product with the position modulo 2^64 drops whole turns exactly, and its upper 32 bits are the
// angle within 2^-32 turns, whatever the position (negative ones too).  For fp32 tensors its quarter turns are taken off as whole numbers, so that
// an eighth of a turn at most is rounded to fp32 and small sines and cosines keep their digits; for halfs all of [-1/2, 1/2) is (2^-26 turns off).
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

#include "kernels.h"

namespace mldhip {
namespace {

template <typename T>
struct Slice;  // 4 channels of one token
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
__device__ __forceinline__ void Store4(uint2* p, const float v[4]) {
  uint2 raw;
  raw.x = __builtin_bit_cast(uint32_t, __floats2half2_rn(v[0], v[1]));
  raw.y = __builtin_bit_cast(uint32_t, __floats2half2_rn(v[2], v[3]));
  *p = raw;
}
__device__ __forceinline__ void Store4(float4* p, const float v[4]) { *p = make_float4(v[0], v[1], v[2], v[3]); }

// sin and cos of phase / 2^32 turns.  The hardware's own (argument in turns, a few 2^-22 off) for halfs.  For fp32 the power series of both on
// an eighth of a turn: what is left out is 3e-9 of the sine, 2e-10 of the cosine.
__device__ __forceinline__ void SinCosOf(const __half*, uint32_t phase, float* s, float* c) {
  const float turns = (float)(int32_t)phase * 0x1p-32f;
  *s = __builtin_amdgcn_sinf(turns);
  *c = __builtin_amdgcn_cosf(turns);
}
__device__ __forceinline__ void SinCosOf(const float*, uint32_t phase, float* s, float* c) {
  const uint32_t quarters = (phase + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(phase - (quarters << 30)) * (float)(6.283185307179586 * 0x1p-32), z = x * x;
  const float a = fmaf(x * z, fmaf(z, fmaf(z, fmaf(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
  const float b = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
  const float one = quarters & 1 ? b : a, two = quarters & 1 ? a : b;
  *s = quarters & 2 ? -one : one;
  *c = (quarters + 1) & 2 ? -two : two;
}

// A work-group is 4 waves; a wave is 64 / LANES tokens times LANES lanes that share a head.  The head's channels go in units of 2 slices:
// the two slices whose channels are paired where pairs are half the rotary channels apart, two neighbouring slices otherwise; a lane owns
// units lane, lane + LANES, ...: at most UNITS of them, in registers from the load to the store.  The angles depend on the token alone, so
// a work-group takes `heads_per_group` heads with one set of sines and cosines.
template <typename T, int LANES, int UNITS, bool INTERLEAVED>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(const NormRopeArgs p) {
  using Raw = typename Slice<T>::type;
  constexpr int kTokens = 64 / LANES;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int token = (blockIdx.x * 4 + wave) * kTokens + lane % kTokens;
  const int part = lane / kTokens;
  if (token - lane % kTokens >= p.tokens) return;  // (a whole wave)
  const bool inside = token < p.tokens;
  const int t = inside ? token : p.tokens - 1;
  const int units = p.head_dim / 8, turned = p.rotary_dim / 8;  // units; units whose channels are rotated

  float sn[UNITS][4], cs[UNITS][4];
  int first[UNITS], second[UNITS];  // slices of the head
  const long long position = p.positions[t];
#pragma unroll
  for (int u = 0; u < UNITS; ++u) {
    const int unit = part + u * LANES;
    if (INTERLEAVED) {
      first[u] = 2 * unit;
      second[u] = 2 * unit + 1;
    } else {
      first[u] = unit < turned ? unit : 2 * unit;  // (behind the rotary channels: 2 * turned + 2 * (unit - turned))
      second[u] = unit < turned ? unit + turned : 2 * unit + 1;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sn[u][e] = cs[u][e] = 0.0f;
      if (unit < turned) {
        SinCosOf((const T*)nullptr, (uint32_t)((uint64_t)position * p.turns[4 * unit + e] >> 32), &sn[u][e], &cs[u][e]);
      }
    }
  }
  const int heads = p.heads + p.kv_heads;
  const int head_begin = blockIdx.y * p.heads_per_group, head_end = min(heads, head_begin + p.heads_per_group);
  for (int head = head_begin; head < head_end; ++head) {
    const bool is_k = head >= p.heads;
    const size_t slice0 = (size_t)(is_k ? head - p.heads : head) * (p.head_dim / 4);
    const Raw* src = static_cast<const Raw*>(is_k ? p.src_k : p.src_q) + slice0 * p.tokens + t;
    Raw* dst = static_cast<Raw*>(is_k ? p.dst_k : p.dst_q) + slice0 * p.tokens + t;
    float x[UNITS][2][4];
    Raw raw[UNITS][2];
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
      if (part + u * LANES < units) {
        raw[u][0] = src[(size_t)first[u] * p.tokens];
        raw[u][1] = src[(size_t)second[u] * p.tokens];
      } else {
        raw[u][0] = raw[u][1] = Raw{};
      }
    float sum = 0.0f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        Load4(raw[u][h], x[u][h]);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = fmaf(x[u][h][e], x[u][h][e], sum);
      }
    if (p.norm) {
#pragma unroll
      for (int off = kTokens; off < 64; off *= 2) sum += __shfl_xor(sum, off);
      const float r = 1.0f / sqrtf(sum / (float)p.head_dim + p.eps);
      const Raw* weight = static_cast<const Raw*>(is_k ? p.k_weight : p.q_weight);
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
        if (part + u * LANES < units) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float w[4];
            Load4(weight[h ? second[u] : first[u]], w);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[u][h][e] = x[u][h][e] * r * (p.weight_offset + w[e]);
          }
        }
    }
    if (!inside) continue;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
      if (part + u * LANES < units) {
        float y[2][4];
        if (part + u * LANES >= turned) {  // channels behind the rotary ones stay as they are, whatever their neighbours hold
#pragma unroll
          for (int e = 0; e < 4; ++e) y[0][e] = x[u][0][e], y[1][e] = x[u][1][e];
        } else if (INTERLEAVED) {  // pairs (0, 1), (2, 3) of each slice: the angles are those of pairs 4 unit .. 4 unit + 3
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
              const float s = sn[u][2 * h + e / 2], c = cs[u][2 * h + e / 2], a = x[u][h][e], b = x[u][h][e + 1];
              y[h][e] = a * c - b * s;
              y[h][e + 1] = b * c + a * s;
            }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[0][e] = x[u][0][e] * cs[u][e] - x[u][1][e] * sn[u][e];
            y[1][e] = x[u][1][e] * cs[u][e] + x[u][0][e] * sn[u][e];
          }
        }
        Store4(dst + (size_t)first[u] * p.tokens, y[0]);
        Store4(dst + (size_t)second[u] * p.tokens, y[1]);
      }
  }
}

template <typename T, int LANES, int UNITS>
void Launch(const NormRopeArgs& p, dim3 grid, hipStream_t stream) {
  if (p.interleaved)
    qk_norm_rope_kernel<T, LANES, UNITS, true><<<grid, 256, 0, stream>>>(p);
  else
    qk_norm_rope_kernel<T, LANES, UNITS, false><<<grid, 256, 0, stream>>>(p);
}

template <typename T>
void LaunchTyped(NormRopeArgs p, hipStream_t stream) {
  const int heads = p.heads + p.kv_heads;
  // Few channels: one unit to a lane, as many lanes as that makes.  Many: runs of 8 tokens (64 bytes of halfs), two units to a lane where heads
  // are longer than 64.  Heads of 128, 40 of them: 2.9 us against 3.6 at one token, 3.7 against 4.4 at 256, 8.0 against 7.1 at 777, 19.6 against
  // 18.1 at 4096; of 256, 24 of them: 2.9 / 3.6, 4.4 / 4.6, 11.3 / 10.1, 34.9 / 21.8.
  const bool small = (long long)p.tokens * heads * p.head_dim < 1 << 21;
  const int lanes = p.head_dim <= 64 ? 8 : p.head_dim <= 128 ? (small ? 16 : 8) : small ? 32 : 16;
  const long long waves = (long long)DivUp(p.tokens, 64 / lanes) * heads;
  // heads that share sines and cosines: more where enough waves are left (heads of 128, 40 of them, by 1 / 2 / 4: 7.1 / 7.7 / 9.1 us at 777 tokens,
  // 17.9 / 15.6 / 16.3 at 3000; heads of 64: 17.0 / 15.1 / 13.9 at 6000)
  p.heads_per_group = waves >= 24 << 10 ? 4 : waves >= 6 << 10 ? 2 : 1;
  const dim3 grid(DivUp(p.tokens, 4 * 64 / lanes), DivUp(heads, p.heads_per_group));
  if (p.head_dim <= 64)
    Launch<T, 8, 1>(p, grid, stream);
  else if (p.head_dim <= 128)
    small ? Launch<T, 16, 1>(p, grid, stream) : Launch<T, 8, 2>(p, grid, stream);
  else
    small ? Launch<T, 32, 1>(p, grid, stream) : Launch<T, 16, 2>(p, grid, stream);
}

}  // namespace

hipError_t LaunchQkNormRope(const NormRopeArgs& a, hipStream_t stream, const char** kernel_name) {
  *kernel_name = "qk_norm_rope_kernel";
  if (a.f16)
    LaunchTyped<__half>(a, stream);
  else
    LaunchTyped<float>(a, stream);
  return hipGetLastError();
}

}  // namespace mldhip
