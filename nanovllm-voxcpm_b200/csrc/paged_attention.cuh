// Attention of single tokens over a paged key-value cache: bf16 and fp16, causal, over everything or over a sliding window of
// the last keys plus a few first ones.
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t, h] . k_j - max),  over the keys j that token t sees
//
// Bound: the visible rows of K and V, read once (4 D Hq flop against 4 D Hk bytes a key: tens of operations per byte). One pass
// with the running maximum and sum (Milakov and Gimelshein, "Online normalizer calculation for softmax", 2018).
#pragma once

#include "decode_step.cuh"
#include "glue.cuh"

namespace b200lora {

// The keys that a row sees, side by side: the first `n_sink` of the sequence, then those from `first` on.
struct RowKeys {
  int req, n_sink, first, n_keys;  // n_keys < 0: no row of any sequence
  __device__ __forceinline__ int key(int i) const { return i < n_sink ? i : i - n_sink + first; }
};

struct PagedArgs {
  const void* q; int64_t q_token, q_head;      // [T, Hq, D], strides in elements
  void* out; int64_t out_token, out_head;
  float* lse;                                  // [T, Hq] or null
  lora_b200_paged_cache cache;
  const int32_t* tables; int64_t table_ld; int table_width;
  const int32_t* context_lens;
  const int32_t* cu_seqlens; int n_req;        // null: row t is the last token of request t
  int T, Hq, Hk, heads, chunks;                // heads: of a chunk of a group; chunks of a group
  int window, sinks;
  float sc;                                    // scale * log2(e): scores and maxima are in units of log2
  float *part_o, *part_ml; int4* joins;        // partial results of CTA boundaries, and what there is to join
};

__device__ __forceinline__ RowKeys row_keys(const PagedArgs& a, int row) {
  RowKeys r = {row, 0, 0, -1};
  int64_t ctx;
  if (a.cu_seqlens == nullptr) {
    ctx = a.context_lens[row];
  } else {
    if (row < a.cu_seqlens[0] || row >= a.cu_seqlens[a.n_req]) return r;
    int lo = 0, hi = a.n_req;  // the last request that begins at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu_seqlens[mid] <= row) lo = mid;
      else hi = mid;
    }
    r.req = lo;
    ctx = (int64_t)a.context_lens[lo] - (a.cu_seqlens[lo + 1] - 1 - row);
  }
  ctx = ctx < 0 ? 0 : ctx;
  const int64_t held = min(ctx, (int64_t)a.table_width * a.cache.block_size);
  const int64_t first = a.window > 0 ? max((int64_t)0, ctx - a.window) : 0;
  r.first = (int)first;
  r.n_sink = (int)min((int64_t)a.sinks, min(first, held));
  r.n_keys = r.n_sink + (int)max((int64_t)0, held - first);
  return r;
}

constexpr int kPagedWarps = 4;
constexpr int kPagedThreads = 32 * kPagedWarps;
constexpr int kPagedStages = 3;
constexpr int kPagedCtas = 2 * 148;  // of a launch: two on every SM
template <int D>
__host__ __device__ constexpr int paged_block_keys() { return D == 64 ? 32 : 16; }  // 8 KB of K and V rows
template <int D>
__host__ __device__ constexpr int paged_stage_bytes() { return 2 * paged_block_keys<D>() * (D * 2 + 16); }
template <int D, int NT>
__host__ __device__ constexpr int paged_smem() {
  const int ring = kPagedWarps * kPagedStages * paged_stage_bytes<D>(), merge = kPagedWarps * 8 * NT * (D + 2) * 4;
  return 8 * NT * (D * 2 + 16) + (ring > merge ? ring : merge);
}

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Joined or single result of a head's two columns
template <bool kF16>
__device__ __forceinline__ void store_result(const PagedArgs& a, int row, int head, int d, float x, float y, float m, float l) {
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (no visible key: zeros; NaN stays)
  char* dst = static_cast<char*>(a.out) + 2 * (row * a.out_token + head * a.out_head + d);
  *reinterpret_cast<uint32_t*>(dst) = pack_16x2<kF16>(x * inv, y * inv);
  if (a.lse != nullptr && d == 0) a.lse[(int64_t)row * a.Hq + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// A CTA takes a contiguous share of the (row, kv head and chunk, block of keys) sequence. Its warps take the blocks of an item
// in turn, each through a ring of its own; the keys are the rows of the matrix instruction (S^T = K Q^T, then O^T = V^T P^T), so
// that eight heads fill it.
template <int D, int NT, bool kF16>
__global__ void __launch_bounds__(kPagedThreads, NT == 1 ? 2 : 1) paged_decode_kernel(const PagedArgs a) {
  extern __shared__ __align__(1024) uint8_t smem[];
  constexpr int kPitch = D * 2 + 16, kKeys = paged_block_keys<D>(), kStage = paged_stage_bytes<D>(), kPieces = D / 8;
  constexpr int kMT = kKeys / 16, kPerLoad = 32 / kPieces;  // rows of a load instruction
  __shared__ int s_row;
  __shared__ long long s_at, s_scan[kPagedThreads], s_total;
  __shared__ uint32_t s_live[kPagedWarps][kPagedStages];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int per_row = a.Hk * a.chunks, group = a.Hq / a.Hk;
  glue_enter();

  auto units_of = [&](int row) {
    const RowKeys r = row_keys(a, row);
    return r.n_keys < 0 ? 0 : max(1, (r.n_keys + kKeys - 1) / kKeys);
  };
  // ---- where this CTA's share begins
  const int rows_each = (a.T + kPagedThreads - 1) / kPagedThreads;
  {
    long long sum = 0;
    for (int i = 0, row = tid * rows_each; i < rows_each && row < a.T; ++i, ++row) sum += units_of(row);
    s_scan[tid] = sum;
    __syncthreads();
    if (tid == 0) {
      long long run = 0;
      for (int i = 0; i < kPagedThreads; ++i) { const long long v = s_scan[i]; s_scan[i] = run; run += v; }
      s_total = run * per_row;
    }
    __syncthreads();
  }
  const long long total = s_total;
  const int G = (int)max(1ll, min((long long)gridDim.x, total / kPagedWarps));  // shares of a block for every warp, or more
  if (tid == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
  if ((int)blockIdx.x >= G || total == 0) return;
  const long long begin = total * blockIdx.x / G, end = total * (blockIdx.x + 1) / G;
  {
    const long long from = s_scan[tid] * per_row, to = tid + 1 < kPagedThreads ? s_scan[tid + 1] * per_row : total;
    if (from <= begin && begin < to) {
      long long at = from;
      int row = tid * rows_each;
      for (;; ++row) {
        const long long n = (long long)units_of(row) * per_row;
        if (begin < at + n) break;
        at += n;
      }
      s_row = row;
      s_at = at;
    }
    __syncthreads();
  }
  int row = s_row;
  long long row_at = s_at;  // first unit of the row

  const uint32_t q_u32 = smem_u32(smem), ring = q_u32 + 8 * NT * kPitch + (uint32_t)(warp * kPagedStages * kStage);
  const char *k_base = static_cast<const char*>(a.cache.k), *v_base = static_cast<const char*>(a.cache.v);
  bool first_piece = true;
  for (long long at = begin; at < end;) {
    const RowKeys keys = row_keys(a, row);
    const int n_units = keys.n_keys < 0 ? 0 : max(1, (keys.n_keys + kKeys - 1) / kKeys);
    if (at >= row_at + (long long)n_units * per_row) {
      row_at += (long long)n_units * per_row;
      ++row;
      continue;
    }
    const int item = (int)((at - row_at) / n_units), u0 = (int)((at - row_at) - (long long)item * n_units);
    const int u1 = (int)min((long long)n_units, u0 + (end - at));
    const int kvh = item / a.chunks, chunk = item - kvh * a.chunks;
    const int head0 = kvh * group + chunk * a.heads, n_heads = min(a.heads, group - chunk * a.heads);
    const int32_t* table = a.tables + keys.req * a.table_ld;

    // this warp's blocks: u0 + warp, u0 + warp + 4, ...
    auto load = [&](int u, int stage) {
      if (u < u1) {
        const int i = u * kKeys + lane;
        int64_t kr = 0, vr = 0;
        bool live = false;
        if (lane < kKeys && i < keys.n_keys) {
          const int key = keys.key(i), page = key / a.cache.block_size, in_page = key - page * a.cache.block_size;
          const int blk = table[page];
          live = (unsigned)blk < (unsigned)a.cache.num_blocks;  // (an entry outside the cache: its keys are left out)
          if (live) {
            kr = 2 * (blk * a.cache.k_block + in_page * a.cache.k_token + kvh * a.cache.k_head);
            vr = 2 * (blk * a.cache.v_block + in_page * a.cache.v_token + kvh * a.cache.v_head);
          }
        }
        const uint32_t mask = __ballot_sync(0xffffffffu, live);
        if (lane == 0) s_live[warp][stage] = mask;
        const int p = lane % kPieces;
#pragma unroll
        for (int j = 0; j < kKeys / kPerLoad; ++j) {
          const int r = j * kPerLoad + lane / kPieces;
          const int64_t ks = __shfl_sync(0xffffffffu, kr, r), vs = __shfl_sync(0xffffffffu, vr, r);
          const uint32_t bytes = (mask >> r) & 1u ? 16u : 0u;  // (rows that are not seen are zero: 0 * V must be 0)
          const uint32_t dst = ring + (uint32_t)(stage * kStage + r * kPitch + p * 16);
          cp_async_16(dst, k_base + ks + p * 16, bytes);
          cp_async_16(dst + kKeys * kPitch, v_base + vs + p * 16, bytes);
        }
      }
      cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < kPagedStages - 1; ++s) load(u0 + warp + s * kPagedWarps, s);

    // q of the chunk's heads; unused rows are zero
    for (int i = tid; i < 8 * NT * kPieces; i += kPagedThreads) {
      const int h = i / kPieces, p = i - h * kPieces;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (h < n_heads) v = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.q) + 2 * (row * a.q_token + (head0 + h) * a.q_head + p * 8));
      sts128(q_u32 + (uint32_t)(h * kPitch + p * 16), v);
    }
    __syncthreads();
    uint32_t qf[NT][D / 16][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        uint32_t r[4];
        ldsm_x4(q_u32 + (uint32_t)((8 * n + (lane & 7)) * kPitch + (lane >> 3) * 16 + 64 * k), r);
        qf[n][2 * k][0] = r[0]; qf[n][2 * k][1] = r[1];
        qf[n][2 * k + 1][0] = r[2]; qf[n][2 * k + 1][1] = r[3];
      }
    float o[NT][D / 16][4], m[NT][2], l[NT][2];  // heads 2 t and 2 t + 1 of a tile; o: columns g and g + 8 of 16
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int d = 0; d < D / 16; ++d) o[n][d][0] = o[n][d][1] = o[n][d][2] = o[n][d][3] = 0.f;
    }
    int stage = 0;
    for (int u = u0 + warp; u < u1; u += kPagedWarps) {
      load(u + (kPagedStages - 1) * kPagedWarps, stage == 0 ? kPagedStages - 1 : stage - 1);
      cp_async_wait_group<kPagedStages - 1>();
      __syncwarp();
      const uint32_t ks = ring + (uint32_t)(stage * kStage), vs = ks + kKeys * kPitch, live = s_live[warp][stage];
      float s[NT][kMT][4];
#pragma unroll
      for (int i = 0; i < kMT; ++i) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][i][0] = s[n][i][1] = s[n][i][2] = s[n][i][3] = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t kf[4];
          ldsm_x4(ks + (uint32_t)((16 * i + (lane & 15)) * kPitch + (lane >> 4) * 16 + 32 * k), kf);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816<kF16>(s[n][i], kf[0], kf[1], kf[2], kf[3], qf[n][k][0], qf[n][k][1]);
        }
      }
      // scores, masked; the maximum moves only where it would grow by more than 2^8 (probabilities stay below that)
      bool grows = false;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const bool seen = (live >> (16 * i + g + 8 * (e >> 1))) & 1u;
            s[n][i][e] = seen ? s[n][i][e] * a.sc : -INFINITY;
            grows |= s[n][i][e] > m[n][e & 1] + 8.f;
          }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = m[n][c];
#pragma unroll
            for (int i = 0; i < kMT; ++i) mx = fmaxf(mx, fmaxf(s[n][i][c], s[n][i][c + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float f = mx == -INFINITY ? 1.f : exp2f(m[n][c] - mx);
            m[n][c] = mx;
            l[n][c] *= f;
#pragma unroll
            for (int d = 0; d < D / 16; ++d) { o[n][d][c] *= f; o[n][d][c + 2] *= f; }
          }
      }
      uint32_t pf[NT][kMT][2];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < kMT; ++i) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float top = m[n][e & 1];
            s[n][i][e] = exp2f(s[n][i][e] - (top == -INFINITY ? 0.f : top));
            l[n][e & 1] += s[n][i][e];
          }
          // (probabilities are rounded to the type of V for the matrix product; their sum is that of the unrounded ones)
          pf[n][i][0] = transpose_8x8(pack_16x2<kF16>(s[n][i][0], s[n][i][1]));
          pf[n][i][1] = transpose_8x8(pack_16x2<kF16>(s[n][i][2], s[n][i][3]));
        }
#pragma unroll
      for (int i = 0; i < kMT; ++i)
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          uint32_t vf[4];
          ldsm_x4_t(vs + (uint32_t)((16 * i + (lane & 7) + 8 * (lane >> 4)) * kPitch + ((lane >> 3) & 1) * 16 + 32 * d), vf);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_16816<kF16>(o[n][d], vf[0], vf[1], vf[2], vf[3], pf[n][i][0], pf[n][i][1]);
        }
      __syncwarp();  // every lane has read the stage
      stage = stage + 1 == kPagedStages ? 0 : stage + 1;
    }
    cp_async_wait_group<0>();
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 4);
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 8);
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 16);
      }
    __syncthreads();  // every warp is done with its ring
    float* acc = reinterpret_cast<float*>(smem + 8 * NT * kPitch);
    float* ml = acc + kPagedWarps * 8 * NT * D;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int h = 8 * n + 2 * t + c;
        float* dst = acc + (warp * 8 * NT + h) * D + g;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) { dst[16 * d] = o[n][d][c]; dst[16 * d + 8] = o[n][d][c + 2]; }
        if (g == 0) { ml[(warp * 8 * NT + h) * 2] = m[n][c]; ml[(warp * 8 * NT + h) * 2 + 1] = l[n][c]; }
      }
    __syncthreads();
    const bool whole = u0 == 0 && u1 == n_units;
    const int slot = 2 * blockIdx.x + (first_piece ? 0 : 1);
    for (int i = tid; i < n_heads * (D / 2); i += kPagedThreads) {
      const int h = i / (D / 2), d = 2 * (i - h * (D / 2));
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) top = fmaxf(top, ml[(w * 8 * NT + h) * 2]);
      float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) {
        const float mw = ml[(w * 8 * NT + h) * 2], f = mw == -INFINITY ? 0.f : exp2f(mw - top);
        const float2 v = *reinterpret_cast<const float2*>(acc + (w * 8 * NT + h) * D + d);
        sum += f * ml[(w * 8 * NT + h) * 2 + 1];
        x += f * v.x;
        y += f * v.y;
      }
      if (whole) {
        store_result<kF16>(a, row, head0 + h, d, x, y, top, sum);
      } else {
        const int64_t at_slot = (int64_t)slot * a.heads + h;
        *reinterpret_cast<float2*>(a.part_o + at_slot * D + d) = make_float2(x, y);
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at_slot * 2) = make_float2(top, sum);
      }
    }
    // the CTA that begins an item and does not end it says who ends it: the last one whose share begins before the item's end
    if (u0 == 0 && !whole && tid == 0) {
      const long long item_end = row_at + (long long)(item + 1) * n_units;
      int last = (int)min((long long)G - 1, (item_end * G - 1) / total);
      while (last + 1 < G && total * (last + 1) / G < item_end) ++last;  // (the shares' bounds are rounded down)
      while (total * last / G >= item_end) --last;
      a.joins[blockIdx.x] = make_int4(row, item, slot, last);
    }
    __syncthreads();  // the ring may be filled again
    at += u1 - u0;
    first_piece = false;
  }
}

// Joins the parts of an item that begins in CTA blockIdx.x: its own, then the first one of every CTA up to the last.
template <int D, bool kF16>
__global__ void __launch_bounds__(kPagedThreads) paged_join_kernel(const PagedArgs a) {
  glue_enter();
  const int4 j = a.joins[blockIdx.x];
  if (j.x < 0) return;
  const int group = a.Hq / a.Hk, kvh = j.y / a.chunks, chunk = j.y - kvh * a.chunks;
  const int head0 = kvh * group + chunk * a.heads, n_heads = min(a.heads, group - chunk * a.heads);
  const int parts = j.w - (int)blockIdx.x + 1;
  auto slot_of = [&](int i) { return (int64_t)(i == 0 ? j.z : 2 * ((int)blockIdx.x + i)) * a.heads; };
  for (int i = threadIdx.x; i < n_heads * (D / 2); i += kPagedThreads) {
    const int h = i / (D / 2), d = 2 * (i - h * (D / 2));
    float top = -INFINITY, sum = 0.f, x = 0.f, y = 0.f;
    for (int k = 0; k < parts; ++k) {
      const int64_t at = slot_of(k) + h;
      const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at * 2), v = *reinterpret_cast<const float2*>(a.part_o + at * D + d);
      const float up = fmaxf(top, ml.x), f0 = top == -INFINITY ? 0.f : exp2f(top - up), f1 = ml.x == -INFINITY ? 0.f : exp2f(ml.x - up);
      x = f0 * x + f1 * v.x;
      y = f0 * y + f1 * v.y;
      sum = f0 * sum + f1 * ml.y;
      top = up;
    }
    store_result<kF16>(a, j.x, head0 + h, d, x, y, top, sum);
  }
}

inline size_t paged_parts_bytes(int heads, int D) { return (size_t)2 * kPagedCtas * heads * D * 4; }
inline size_t paged_workspace_bytes(int Hq, int Hk, int D) {
  const int heads = std::min(Hq / Hk, 16);
  return paged_parts_bytes(heads, D) + (size_t)2 * kPagedCtas * heads * 8 + kPagedCtas * sizeof(int4);
}

template <int D, int NT, bool kF16>
inline int paged_decode_launch_t(const PagedArgs& a, cudaStream_t stream) {
  const cudaError_t e = cudaFuncSetAttribute(paged_decode_kernel<D, NT, kF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, paged_smem<D, NT>());
  if (e != cudaSuccess) return fail(B200_LORA_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  const int rc = launch_dependent(paged_decode_kernel<D, NT, kF16>, "paged_decode_kernel", dim3(kPagedCtas), kPagedThreads, paged_smem<D, NT>(), stream, a);
  if (rc != B200_LORA_OK) return rc;
  return launch_dependent(paged_join_kernel<D, kF16>, "paged_join_kernel", dim3(kPagedCtas), kPagedThreads, 0, stream, a);
}

inline int paged_decode_launch(PagedArgs a, int D, int dtype, void* workspace, cudaStream_t stream) {
  const int group = a.Hq / a.Hk;
  a.heads = std::min(group, 16);
  a.chunks = ceil_div_i(group, a.heads);
  char* ws = static_cast<char*>(workspace);
  a.part_o = reinterpret_cast<float*>(ws);
  a.part_ml = reinterpret_cast<float*>(ws + paged_parts_bytes(a.heads, D));
  a.joins = reinterpret_cast<int4*>(ws + paged_parts_bytes(a.heads, D) + (size_t)2 * kPagedCtas * a.heads * 8);
  const bool f16 = dtype == B200_LORA_F16, wide = a.heads > 8;
  if (D == 64) {
    if (wide) return f16 ? paged_decode_launch_t<64, 2, true>(a, stream) : paged_decode_launch_t<64, 2, false>(a, stream);
    return f16 ? paged_decode_launch_t<64, 1, true>(a, stream) : paged_decode_launch_t<64, 1, false>(a, stream);
  }
  if (wide) return f16 ? paged_decode_launch_t<128, 2, true>(a, stream) : paged_decode_launch_t<128, 2, false>(a, stream);
  return f16 ? paged_decode_launch_t<128, 1, true>(a, stream) : paged_decode_launch_t<128, 1, false>(a, stream);
}

}  // namespace b200lora
