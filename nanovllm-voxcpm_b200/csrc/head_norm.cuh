// RMS norm of every query and key head, rotation by position and the cache store in one pass over the packed qkv rows.
//
//   y = x * rsqrt(mean(x^2) + eps) * w;  (y_j, y_{j + D/2}) turned by the angle of (position, j);  k and v rows to their cache slot
//
// Bound: the bytes of the rows, once in and once out. Measured: 8192 tokens, 32 / 8 heads of 128 (202 MB with the tables), 42 us = 4.8 TB/s, 0.73
// of the measured copy bandwidth (24 warps on an SM by registers, each waiting for its sums much of the time; a thread per head's piece 62
// to 81 us, two to eight heads a thread 49 to 88); one token 4.2 us.
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

// Weights and rotation of a thread's columns as one: with x = rstd lo and y = rstd hi, lo' = a1 x + b1 y, hi' = a2 x + b2 y. (rstd first:
// of a head whose sum of squares is infinite it is 0, and so is rstd times any finite element, while an element times its factor may
// have overflowed by then. The sum is fp32: 8192 wide tokens take 42.4 us so, 41.4 with rstd last.) Without a rotation lo' = a1 x and
// hi' = b2 y alone: 0 times an infinite element would be NaN in its opposite column.
struct HeadTurn {
  float2 a1[4], b1[4], a2[4], b2[4];
  // at `tb` of the tables: the angles of the first of the thread's columns; w1, w2: its weights in the two halves
  template <typename T>
  __device__ __forceinline__ void load(const RopeKvParams& r, const Vec8<T>& w1, const Vec8<T>& w2, const void* cos, const void* sin, int64_t tb) {
    const int half = r.D >> 1;
    float c[8], s[8];
    if (r.apply_rope) {
      table_load8(cos, r.table_dtype, tb, c);
      table_load8(sin, r.table_dtype, tb, s);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) { c[e] = 1.f; s[e] = 0.f; }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a1[e] = mul2(w1.pair(e), make_float2(c[2 * e], c[2 * e + 1]));
      b1[e] = mul2(w2.pair(e), make_float2(-s[2 * e], -s[2 * e + 1]));
    }
    if (r.apply_rope && r.table_dim == r.D) {  // (the second half has angles of its own)
      table_load8(cos, r.table_dtype, tb + half, c);
      table_load8(sin, r.table_dtype, tb + half, s);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a2[e] = mul2(w1.pair(e), make_float2(s[2 * e], s[2 * e + 1]));
      b2[e] = mul2(w2.pair(e), make_float2(c[2 * e], c[2 * e + 1]));
    }
  }
  template <typename T>
  __device__ __forceinline__ void apply(Vec8<T>& lo, Vec8<T>& hi, float rstd, bool rotate) const {
    const float2 r2 = make_float2(rstd, rstd);
    if (rotate) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 x = mul2(r2, lo.pair(e)), y = mul2(r2, hi.pair(e));
        lo.set_pair(e, fma2(y, b1[e], mul2(x, a1[e])));
        hi.set_pair(e, fma2(y, b2[e], mul2(x, a2[e])));
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo.set_pair(e, mul2(mul2(r2, lo.pair(e)), a1[e]));
        hi.set_pair(e, mul2(mul2(r2, hi.pair(e)), b2[e]));
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ Vec8<T> load8(const T* at) {
  Vec8<T> v;
  v.raw = *reinterpret_cast<const uint4*>(at);
  return v;
}
template <typename T>
__device__ __forceinline__ void store8(T* at, const Vec8<T>& v) { *reinterpret_cast<uint4*>(at) = v.raw; }

// Sum of the squares of a head over its 1 << lane_shift lanes; every lane of the warp calls it
template <typename T>
__device__ __forceinline__ float head_squares(const Vec8<T>& lo, const Vec8<T>& hi, int lane_shift) {
  float2 sum = make_float2(0.f, 0.f);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 a = lo.pair(e), b = hi.pair(e);
    sum = fma2(b, b, fma2(a, a, sum));
  }
  float ss = sum.x + sum.y;
#pragma unroll
  for (int o = (1 << lane_shift) >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  return ss;
}

__device__ __forceinline__ int64_t table_row(const RopeKvParams& r, int tok) {
  const int64_t pos = r.positions[tok];
  return (pos < 0 ? 0 : (pos >= r.max_pos ? r.max_pos - 1 : pos)) * r.table_dim;
}

// Where a token's k and v go: element offsets, -1: nowhere
__device__ __forceinline__ void cache_rows(const HeadNormParams& p, int tok, int64_t* at_k, int64_t* at_v) {
  *at_k = *at_v = -1;
  if (p.cache.k == nullptr) return;
  const int slot = p.r.slot_mapping[tok];
  if (slot < 0 || slot >= (int64_t)p.cache.num_blocks * p.cache.block_size) return;
  const int blk = slot / p.cache.block_size, in_block = slot - blk * p.cache.block_size;
  *at_k = blk * p.cache.k_block + in_block * p.cache.k_token;
  *at_v = blk * p.cache.v_block + in_block * p.cache.v_token;
}

// Results of columns j.. and D/2 + j.. of a head to where they belong
template <typename T>
__device__ __forceinline__ void store_head(const HeadNormParams& p, int tok, int head, int j, int64_t at_k, int64_t at_v, const Vec8<T>& lo, const Vec8<T>& hi) {
  const int half = p.r.D >> 1, kv = head - p.r.Hq, v = kv - p.r.Hk;
  T* dst = nullptr;
  if (kv < 0 && p.q_out != nullptr) dst = static_cast<T*>(p.q_out) + (int64_t)tok * p.q_out_ld + (int64_t)head * p.r.D + j;
  else if (v < 0 && p.q_out == nullptr) dst = static_cast<T*>(p.r.qkv) + (int64_t)tok * p.r.qkv_ld + (int64_t)head * p.r.D + j;
  if (dst != nullptr) {
    store8(dst, lo);
    store8(dst + half, hi);
  }
  if (kv >= 0 && at_k >= 0) {
    T* c = v < 0 ? static_cast<T*>(p.cache.k) + at_k + kv * p.cache.k_head + j : static_cast<T*>(p.cache.v) + at_v + v * p.cache.v_head + j;
    store8(c, lo);
    store8(c + half, hi);
  }
}

// Few tokens: 1 << lane_shift threads keep a head, each 8 columns of the first half and the 8 opposite ones.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) head_norm_kernel(const HeadNormParams p, int lane_shift) {
  glue_enter();
  const int half = p.r.D >> 1, heads = p.r.Hq + 2 * p.r.Hk;
  const uint32_t unit = blockIdx.x * (kRopeThreads >> lane_shift) + (threadIdx.x >> lane_shift), tok_u = unit / (uint32_t)heads;
  const int tok = (int)min(tok_u, (uint32_t)p.r.T - 1), j = 8 * (threadIdx.x & ((1 << lane_shift) - 1)), head = (int)(unit - tok_u * heads);
  const bool live = tok_u < (uint32_t)p.r.T && j < half;  // (the others take part in the sums of their warp)
  Vec8<T> lo, hi;
  lo.raw = hi.raw = make_uint4(0, 0, 0, 0);
  if (live) {
    const T* src = static_cast<const T*>(p.r.qkv) + (int64_t)tok * p.r.qkv_ld + (int64_t)head * p.r.D + j;
    lo = load8(src);
    hi = load8(src + half);
  }
  const float ss = head_squares(lo, hi, lane_shift);
  if (!live) return;
  if (head < p.r.Hq + p.r.Hk) {
    HeadTurn turn;
    const T* w = static_cast<const T*>(head < p.r.Hq ? p.q_weight : p.k_weight) + j;
    turn.load(p.r, load8(w), load8(w + half), p.r.cos, p.r.sin, p.r.apply_rope ? table_row(p.r, tok) + j : 0);
    turn.apply(lo, hi, rsqrtf(ss / (float)p.r.D + p.eps), p.r.apply_rope);
  }
  int64_t at_k, at_v;
  cache_rows(p, tok, &at_k, &at_v);
  store_head(p, tok, head, j, at_k, at_v, lo, hi);
}

// Many tokens: the rows of `tokens` tokens and their table rows come by bulk copies into one of two stages while the other is
// worked on, three CTAs on an SM; a thread keeps the angles and weights of its columns for all heads of its token that it takes.
constexpr int kHeadCtas = 3;  // on an SM (8192 wide tokens: 43 us with two, 41 with three, 59 with four; ptxas spills one word of three's 80 registers, many of four's 64)
struct HeadRing { int tokens, row_bytes, table_bytes, stage_bytes; };

template <typename T, int lane_shift>
__global__ void __launch_bounds__(kRopeThreads, kHeadCtas) head_norm_ring_kernel(const HeadNormParams p, const HeadRing ring) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[2];
  __shared__ volatile int abort_flag;
  const int tid = threadIdx.x, half = p.r.D >> 1, heads = p.r.Hq + 2 * p.r.Hk;
  if (tid == 0) {
    mbar_init(smem_u32(&full[0]), 1);
    mbar_init(smem_u32(&full[1]), 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  __syncthreads();
  glue_enter();
  const int n_groups = (p.r.T + ring.tokens - 1) / ring.tokens;
  const int one = ring.row_bytes + 2 * ring.table_bytes;  // bytes of a token
  auto load = [&](int group, int st) {  // the first warp
    const int t0 = group * ring.tokens, n = min(ring.tokens, p.r.T - t0);
    const uint32_t bar = smem_u32(&full[st]), base = smem_u32(smem) + st * ring.stage_bytes;
    if (tid == 0) mbar_arrive_expect_tx(bar, (uint32_t)(n * one));
    __syncwarp();
    for (int i = tid; i < n; i += 32) {
      const uint32_t dst = base + i * one;
      bulk_g2s(dst, static_cast<const char*>(p.r.qkv) + 2 * (int64_t)(t0 + i) * p.r.qkv_ld, ring.row_bytes, bar);
      if (p.r.apply_rope) {
        const int64_t at = table_row(p.r, t0 + i) * (p.r.table_dtype == B200_LORA_F32 ? 4 : 2);
        bulk_g2s(dst + ring.row_bytes, static_cast<const char*>(p.r.cos) + at, ring.table_bytes, bar);
        bulk_g2s(dst + ring.row_bytes + ring.table_bytes, static_cast<const char*>(p.r.sin) + at, ring.table_bytes, bar);
      }
    }
  };
  if (tid < 32)
    for (int k = 0; k < 2; ++k)
      if ((int)blockIdx.x + k * (int)gridDim.x < n_groups) load(blockIdx.x + k * gridDim.x, k);
  const int sub = tid >> lane_shift, j = 8 * (tid & ((1 << lane_shift) - 1));
  const int per_token = (kRopeThreads >> lane_shift) / ring.tokens;  // subgroups of a token
  const int tok_in = sub / per_token, first = sub - tok_in * per_token;
  for (int k = 0, group = blockIdx.x; group < n_groups; ++k, group += gridDim.x) {
    const int st = k & 1, tok = group * ring.tokens + tok_in;
    const bool live = tok < p.r.T && j < half;
    int64_t at_k = -1, at_v = -1;
    if (live) cache_rows(p, tok, &at_k, &at_v);
    if (!mbar_wait_bounded(smem_u32(&full[st]), (uint32_t)((k >> 1) & 1), &abort_flag)) break;
    const uint8_t* at = smem + st * ring.stage_bytes + tok_in * one;
    const T* row = reinterpret_cast<const T*>(at) + j;
    HeadTurn turn;
    int kind = -1;  // of the weights in `turn`: 0 q, 1 k
    for (int h = first; h - first < heads; h += per_token) {  // (all subgroups go round equally often: their lanes sum together)
      const bool here = live && h < heads;
      Vec8<T> lo, hi;
      lo.raw = hi.raw = make_uint4(0, 0, 0, 0);
      if (here) {
        lo = load8(row + h * p.r.D);
        hi = load8(row + h * p.r.D + half);
      }
      const float ss = head_squares(lo, hi, lane_shift);
      if (!here) continue;
      if (h < p.r.Hq + p.r.Hk) {
        const int want = h < p.r.Hq ? 0 : 1;
        if (kind != want) {
          const T* w = static_cast<const T*>(want == 0 ? p.q_weight : p.k_weight) + j;
          turn.load(p.r, load8(w), load8(w + half), at + ring.row_bytes, at + ring.row_bytes + ring.table_bytes, j);
        }
        kind = want;
        turn.apply(lo, hi, rsqrtf(ss / (float)p.r.D + p.eps), p.r.apply_rope);
      }
      store_head(p, tok, h, j, at_k, at_v, lo, hi);
    }
    __syncthreads();
    if (tid < 32 && group + 2 * (int)gridDim.x < n_groups) load(group + 2 * gridDim.x, st);
  }
  if (tid == 0 && abort_flag != 0) atomicOr(&g_b200_status, kStatusWaitGaveUp);
}

constexpr int kHeadStage = 36 << 10;  // bytes of a stage at most: two of them, and kHeadCtas CTAs on an SM
// Rows of a call, in bytes, from which the copies pay: us, a thread per piece / stages, heads 16 / 2 of 64: 1024 tokens (2.6 MB) 3.6 /
// 4.9, 2048 7.3 / 8.3, 4096 11.0 / 11.1, 8192 20 / 16.4; 32 / 8 of 128: 256 tokens (3.1 MB) 3.5 / 5.6, 512 7.0 / 7.9, 1024 12.6 / 10.4,
// 8192 81 / 41.
constexpr int64_t kHeadRingBytes = 8 << 20;

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
  int lane_shift = 0;
  while ((16 << lane_shift) < r.D) ++lane_shift;
  const int heads = r.Hq + 2 * r.Hk;
  HeadRing ring;
  ring.row_bytes = (int)std::min<int64_t>(2 * width, 1 << 20);
  ring.table_bytes = r.apply_rope ? r.table_dim * (r.table_dtype == B200_LORA_F32 ? 4 : 2) : 0;
  const int one = ring.row_bytes + 2 * ring.table_bytes;
  ring.tokens = 1;
  while (2 * ring.tokens * one <= kHeadStage && 2 * ring.tokens <= (kRopeThreads >> lane_shift) && ceil_div_i(r.T, 2 * ring.tokens) >= kHeadCtas * 148) ring.tokens *= 2;
  ring.stage_bytes = ring.tokens * one;
  if (2 * width * r.T >= kHeadRingBytes && one <= kHeadStage) {
    const int smem = 2 * ring.stage_bytes, grid = std::min(kHeadCtas * 148, ceil_div_i(r.T, ring.tokens));
#define B200_HEAD_RING(TT, SHIFT)                                                                                                              \
  {                                                                                                                                            \
    const cudaError_t e = cudaFuncSetAttribute(head_norm_ring_kernel<TT, SHIFT>, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kHeadStage); \
    if (e != cudaSuccess) return fail(B200_LORA_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));                                    \
    return launch_dependent(head_norm_ring_kernel<TT, SHIFT>, "head_norm_ring_kernel", dim3((unsigned)grid), kRopeThreads, (size_t)smem, stream, p, ring); \
  }
#define B200_HEAD_RINGS(TT)                    \
  {                                            \
    if (lane_shift == 0) B200_HEAD_RING(TT, 0) \
    if (lane_shift == 1) B200_HEAD_RING(TT, 1) \
    if (lane_shift == 2) B200_HEAD_RING(TT, 2) \
    if (lane_shift == 3) B200_HEAD_RING(TT, 3) \
    B200_HEAD_RING(TT, 4)                      \
  }
    if (dtype == B200_LORA_BF16) B200_HEAD_RINGS(__nv_bfloat16)
    B200_HEAD_RINGS(__half)
#undef B200_HEAD_RINGS
#undef B200_HEAD_RING
  }
  const int64_t units = (int64_t)r.T * heads;
  if (units > INT32_MAX) return fail(B200_LORA_EUNSUPPORTED, "qk_norm_rope_kv_store: %d rows of %d heads", r.T, heads);
  const dim3 blocks((unsigned)(((units << lane_shift) + kRopeThreads - 1) / kRopeThreads));
  if (dtype == B200_LORA_BF16) return launch_dependent(head_norm_kernel<__nv_bfloat16>, "head_norm_kernel", blocks, kRopeThreads, 0, stream, p, lane_shift);
  return launch_dependent(head_norm_kernel<__half>, "head_norm_kernel", blocks, kRopeThreads, 0, stream, p, lane_shift);
}

}  // namespace b200lora
