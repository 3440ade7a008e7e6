// RMS norm of every query and key head, rotation by position and the cache store in one pass over the packed qkv rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;  (y_j, y_{j + D/2}) turned by the angle of (position, j);  k and v rows to their cache slot
//
// Bound: the bytes of the rows, once in and once out.
#pragma once

#include "glue.cuh"

namespace b200lora {

struct HeadNormParams {
  RopeKvParams r;  // (its caches are not used)
  const void *q_weight, *k_weight;
  float eps;
  void* q_out; int64_t q_out_ld;
  lora_b200_paged_cache cache;
};

// `lanes` threads (a power of two) keep a head: each 8 columns of the first half and the 8 opposite ones. They take `per_group`
// heads of one token in turn, with the angles in registers.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) head_norm_kernel(const HeadNormParams p, int lanes, int per_group) {
  glue_enter();
  const int half = p.r.D >> 1, heads = p.r.Hq + 2 * p.r.Hk, groups = (heads + per_group - 1) / per_group;
  const int64_t unit = ((int64_t)blockIdx.x * kRopeThreads + threadIdx.x) / lanes;
  const int64_t tok64 = unit / groups;
  const int tok = (int)min(tok64, (int64_t)p.r.T - 1), j = 8 * (threadIdx.x & (lanes - 1));
  const int head0 = (int)(unit - tok64 * groups) * per_group;
  const bool live = tok64 < p.r.T && j < half;  // (the others take part in the sums of their warp)
  T* const row = static_cast<T*>(p.r.qkv) + (int64_t)tok * p.r.qkv_ld + j;

  float c1[8], s1[8], c2[8], s2[8];
  if (p.r.apply_rope && live) {
    int64_t pos = p.r.positions[tok];
    pos = pos < 0 ? 0 : (pos >= p.r.max_pos ? p.r.max_pos - 1 : pos);
    const int64_t tb = pos * p.r.table_dim + j;
    const int hi_off = p.r.table_dim == p.r.D ? half : 0;
    table_load8(p.r.cos, p.r.table_dtype, tb, c1);
    table_load8(p.r.sin, p.r.table_dtype, tb, s1);
    table_load8(p.r.cos, p.r.table_dtype, tb + hi_off, c2);
    table_load8(p.r.sin, p.r.table_dtype, tb + hi_off, s2);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) { c1[e] = c2[e] = 1.f; s1[e] = s2[e] = 0.f; }
  }
  int64_t at_k = -1, at_v = -1;
  if (p.cache.k != nullptr) {
    const int slot = p.r.slot_mapping[tok];
    if (slot >= 0 && slot < (int64_t)p.cache.num_blocks * p.cache.block_size) {
      const int blk = slot / p.cache.block_size, in_block = slot - blk * p.cache.block_size;
      at_k = blk * p.cache.k_block + in_block * p.cache.k_token + j;
      at_v = blk * p.cache.v_block + in_block * p.cache.v_token + j;
    }
  }
  for (int i = 0; i < per_group; ++i) {
    const int head = head0 + i, kv = head - p.r.Hq, v = kv - p.r.Hk;  // kv < 0: a q head; v < 0: a q or k head
    const bool here = live && head < heads;
    Vec8<T> lo, hi;
    lo.raw = hi.raw = make_uint4(0, 0, 0, 0);
    if (here) {
      lo.raw = *reinterpret_cast<const uint4*>(row + (int64_t)head * p.r.D);
      hi.raw = *reinterpret_cast<const uint4*>(row + (int64_t)head * p.r.D + half);
    }
    float x[2][8], ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[0][e] = lo.get(e);
      x[1][e] = hi.get(e);
      ss += x[0][e] * x[0][e] + x[1][e] * x[1][e];
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!here) continue;
    if (v < 0) {
      const float rstd = rsqrtf(ss / (float)p.r.D + p.eps);
      const T* w = static_cast<const T*>(kv < 0 ? p.q_weight : p.k_weight) + j;
      Vec8<T> w1, w2;
      w1.raw = *reinterpret_cast<const uint4*>(w);
      w2.raw = *reinterpret_cast<const uint4*>(w + half);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float a = x[0][e] * rstd * w1.get(e), b = x[1][e] * rstd * w2.get(e);
        lo.set(e, a * c1[e] - b * s1[e]);
        hi.set(e, b * c2[e] + a * s2[e]);
      }
    }
    T* dst = nullptr;
    if (kv < 0 && p.q_out != nullptr) dst = static_cast<T*>(p.q_out) + (int64_t)tok * p.q_out_ld + (int64_t)head * p.r.D + j;
    else if (v < 0 && p.q_out == nullptr) dst = row + (int64_t)head * p.r.D;
    if (dst != nullptr) {
      *reinterpret_cast<uint4*>(dst) = lo.raw;
      *reinterpret_cast<uint4*>(dst + half) = hi.raw;
    }
    if (kv >= 0 && at_k >= 0) {
      T* c = v < 0 ? static_cast<T*>(p.cache.k) + at_k + kv * p.cache.k_head : static_cast<T*>(p.cache.v) + at_v + v * p.cache.v_head;
      *reinterpret_cast<uint4*>(c) = lo.raw;
      *reinterpret_cast<uint4*>(c + half) = hi.raw;
    }
  }
}

inline int paged_cache_check(const lora_b200_paged_cache& c, const char* what) {
  if (c.k == nullptr || c.v == nullptr) return fail(B200_LORA_EINVAL, "%s: a cache is null", what);
  if (c.num_blocks < 1 || c.block_size < 1) return fail(B200_LORA_EINVAL, "%s: %d blocks of %d", what, c.num_blocks, c.block_size);
  if (!aligned16(c.k) || !aligned16(c.v) || c.k_block % 8 || c.k_token % 8 || c.k_head % 8 || c.v_block % 8 || c.v_token % 8 || c.v_head % 8)
    return fail(B200_LORA_EUNSUPPORTED, "%s: cache rows must start on 16-byte boundaries", what);
  return B200_LORA_OK;
}

inline int head_norm_launch(const HeadNormParams& p, int dtype, cudaStream_t stream) {
  const RopeKvParams& r = p.r;
  if (r.T < 0 || r.Hq < 0 || r.Hk < 0 || r.Hq + r.Hk < 1 || r.D < 1) return fail(B200_LORA_EINVAL, "qk_norm_rope_kv_store: bad shape");
  if (dtype != B200_LORA_BF16 && dtype != B200_LORA_F16) return fail(B200_LORA_EUNSUPPORTED, "qk_norm_rope_kv_store: bf16 and fp16 only");
  if (r.D % 16 != 0 || r.D > 256) return fail(B200_LORA_EUNSUPPORTED, "qk_norm_rope_kv_store: head_dim %d (needs a multiple of 16 up to 256)", r.D);
  if (r.T == 0) return B200_LORA_OK;
  if (r.qkv == nullptr || p.q_weight == nullptr || p.k_weight == nullptr) return fail(B200_LORA_EINVAL, "qk_norm_rope_kv_store: null pointer");
  if (p.q_out != nullptr && p.cache.k == nullptr) return fail(B200_LORA_EINVAL, "qk_norm_rope_kv_store: q_out needs a cache for k");
  const int64_t width = (int64_t)(r.Hq + 2 * r.Hk) * r.D;
  if (r.qkv_ld < width || (p.q_out != nullptr && p.q_out_ld < (int64_t)r.Hq * r.D)) return fail(B200_LORA_EINVAL, "qk_norm_rope_kv_store: row stride smaller than row");
  if (r.qkv_ld % 8 || !aligned16(r.qkv) || p.q_out_ld % 8 || !aligned16(p.q_out) || !aligned16(p.q_weight) || !aligned16(p.k_weight) ||
      !aligned16(r.cos) || !aligned16(r.sin))
    return fail(B200_LORA_EUNSUPPORTED, "qk_norm_rope_kv_store: rows, weights and tables must be 16-byte aligned");
  if (r.apply_rope) {
    if (r.positions == nullptr || r.cos == nullptr || r.sin == nullptr || r.max_pos <= 0)
      return fail(B200_LORA_EINVAL, "qk_norm_rope_kv_store: rotation needs positions and cos / sin tables");
    if (r.table_dim != r.D && r.table_dim != r.D / 2)
      return fail(B200_LORA_EINVAL, "qk_norm_rope_kv_store: table width %d is neither head_dim nor head_dim / 2", r.table_dim);
    if (r.table_dtype != B200_LORA_F32 && r.table_dtype != B200_LORA_BF16 && r.table_dtype != B200_LORA_F16)
      return fail(B200_LORA_EINVAL, "qk_norm_rope_kv_store: bad table dtype");
  }
  if (p.cache.k != nullptr) {
    const int rc = paged_cache_check(p.cache, "qk_norm_rope_kv_store");
    if (rc != B200_LORA_OK) return rc;
    if (r.slot_mapping == nullptr) return fail(B200_LORA_EINVAL, "qk_norm_rope_kv_store: a cache needs slot_mapping");
  }
  int lanes = 1;
  while (lanes * 16 < r.D) lanes *= 2;
  const int heads = r.Hq + 2 * r.Hk, per_group = 1;
  const int64_t blocks = ((int64_t)r.T * ceil_div_i(heads, per_group) * lanes + kRopeThreads - 1) / kRopeThreads;
  if (blocks > INT32_MAX) return fail(B200_LORA_EUNSUPPORTED, "qk_norm_rope_kv_store: %d rows of %d heads", r.T, heads);
  if (dtype == B200_LORA_BF16)
    return launch_dependent(head_norm_kernel<__nv_bfloat16>, "head_norm_kernel", dim3((unsigned)blocks), kRopeThreads, 0, stream, p, lanes, per_group);
  return launch_dependent(head_norm_kernel<__half>, "head_norm_kernel", dim3((unsigned)blocks), kRopeThreads, 0, stream, p, lanes, per_group);
}

}  // namespace b200lora
