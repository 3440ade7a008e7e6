// Results of attention over parts of a context, with the logarithms of their sums, joined to the result over all of it:
//
//   out = sum_i e^(lse_i - lse) out_i,  lse = log sum_i e^lse_i
//
// Bound: the parts read once and the result written once. A thread takes 16 bytes of a row through all parts, four of them under
// way at a time, with the running maximum and sum (4096 tokens of 32 heads of 128 from four parts: 31.5 us, 83 % of the measured copy
// bandwidth; four tokens from two: 1.5 us in a graph, 6 with the host's call). A part without a key (lse of -inf) has no part in it,
// whatever its values.
#pragma once

#include "glue.cuh"

namespace b200lora {

constexpr int kJoinParts = 64;        // addresses travel with the launch
constexpr int kJoinRowThreads = 256;
constexpr int kJoinAtOnce = 4;

struct JoinArgs {
  const void* outs[kJoinParts];
  const float* lses[kJoinParts];
  int64_t part_token, part_head, lse_token, lse_head;  // strides in elements, the same for all parts
  void* out; int64_t out_token, out_head;
  float* lse;                                          // [T, H] or null
  int n_parts, T, H, vecs;                             // vecs: 16-byte pieces of a row
};

// 16 bytes as fp32
template <int kType>
struct JoinVec {  // kType: B200_LORA_BF16, _F16, _F32
  static constexpr int kN = kType == B200_LORA_F32 ? 4 : 8;
  float v[kN];
  __device__ __forceinline__ void read(const uint4& r) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kType == B200_LORA_F32) {
        v[i] = __uint_as_float(w[i]);
      } else {
        const float2 p = unpack_16x2<kType == B200_LORA_F16>(w[i]);
        v[2 * i] = p.x;
        v[2 * i + 1] = p.y;
      }
    }
  }
  __device__ __forceinline__ uint4 packed(float f) const {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kType == B200_LORA_F32) w[i] = __float_as_uint(v[i] * f);
      else w[i] = pack_16x2<kType == B200_LORA_F16>(v[2 * i] * f, v[2 * i + 1] * f);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <int kType, typename Index>
__global__ void __launch_bounds__(kJoinRowThreads, 4) join_attention_kernel(const __grid_constant__ JoinArgs a) {
  constexpr int kSize = kType == B200_LORA_F32 ? 4 : 2;
  const Index i = (Index)blockIdx.x * kJoinRowThreads + threadIdx.x, row = i / (Index)a.vecs, token = row / (Index)a.H;
  const int vec = (int)(i - row * (Index)a.vecs), head = (int)(row - token * (Index)a.H);
  glue_enter();
  if (token >= (Index)a.T) return;
  const int64_t at = kSize * ((int64_t)token * a.part_token + head * a.part_head) + 16 * vec, lse_at = (int64_t)token * a.lse_token + head * a.lse_head;
  float m = -INFINITY, l = 0.f;
  JoinVec<kType> sum, x;
#pragma unroll
  for (int j = 0; j < x.kN; ++j) sum.v[j] = 0.f;
  for (int p0 = 0; p0 < a.n_parts; p0 += kJoinAtOnce) {
    uint4 raw[kJoinAtOnce];
    float e[kJoinAtOnce];
#pragma unroll
    for (int k = 0; k < kJoinAtOnce; ++k) {
      e[k] = -INFINITY;
      raw[k] = make_uint4(0, 0, 0, 0);
      if (p0 + k < a.n_parts) {
        e[k] = a.lses[p0 + k][lse_at];
        raw[k] = ldg128(static_cast<const char*>(a.outs[p0 + k]) + at);
      }
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < kJoinAtOnce; ++k) top = fmaxf(top, e[k]);
    const float f = m == -INFINITY ? 0.f : __expf(m - top);
    m = top;
    l *= f;
#pragma unroll
    for (int j = 0; j < x.kN; ++j) sum.v[j] *= f;
#pragma unroll
    for (int k = 0; k < kJoinAtOnce; ++k) {
      if (e[k] == -INFINITY) continue;
      const float w = __expf(e[k] - top);  // (NaN stays)
      x.read(raw[k]);
      l += w;
#pragma unroll
      for (int j = 0; j < x.kN; ++j) sum.v[j] += w * x.v[j];
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  *reinterpret_cast<uint4*>(static_cast<char*>(a.out) + kSize * ((int64_t)token * a.out_token + head * a.out_head) + 16 * vec) = sum.packed(inv);
  if (a.lse != nullptr && vec == 0) a.lse[row] = l == 0.f ? -INFINITY : m + logf(l);
}

template <int kType>
inline int join_attention_launch_t(const JoinArgs& a, int64_t ctas, cudaStream_t stream) {
  const dim3 grid((unsigned)ctas);
  if (ctas < (1 << 22)) return launch_dependent(join_attention_kernel<kType, uint32_t>, "join_attention_kernel", grid, kJoinRowThreads, 0, stream, a);
  return launch_dependent(join_attention_kernel<kType, int64_t>, "join_attention_kernel", grid, kJoinRowThreads, 0, stream, a);
}
inline int join_attention_launch(const JoinArgs& a, int dtype, cudaStream_t stream) {
  const int64_t rows = (int64_t)a.T * a.H;
  if (rows > INT32_MAX || rows * a.vecs > (int64_t)INT32_MAX * kJoinRowThreads)
    return fail(B200_LORA_EUNSUPPORTED, "join_attention: %d tokens of %d heads are more than a launch takes", a.T, a.H);
  const int64_t ctas = (rows * a.vecs + kJoinRowThreads - 1) / kJoinRowThreads;
  if (dtype == B200_LORA_BF16) return join_attention_launch_t<B200_LORA_BF16>(a, ctas, stream);
  if (dtype == B200_LORA_F16) return join_attention_launch_t<B200_LORA_F16>(a, ctas, stream);
  return join_attention_launch_t<B200_LORA_F32>(a, ctas, stream);
}

}  // namespace b200lora
