// Attention of single tokens over a paged key-value cache: bf16 and fp16, causal, over everything or over a sliding window of
// the last keys plus a few first ones.
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t, h] . k_j - max),  over the keys j that token t sees
//
// Bound: the visible rows of K and V, read once (4 D Hq flop against 4 D Hk bytes a key: tens of operations per byte). One pass
// with the running maximum and sum (Milakov and Gimelshein, "Online normalizer calculation for softmax", 2018). Rows come by
// cp.async, key by key through the block table, so that any block size and stride will do and rows that are not seen are zeros;
// mma.sync, since eight or sixteen heads do not fill a tcgen05 tile and the arithmetic is a few per cent of the time.
// Measured (bytes that must be read, of the measured copy bandwidth): 256 requests of 1000 tokens, 32 / 8 heads of 128, 173 us (93 %); 48 of
// 500 to 8192 139 us (87 %); one of 100003 79 us (79 %: 62.5 at the bandwidth, the rest is the sums over the rows, the first
// blocks and the join); 64 of 2000, 16 / 2 of 128, 27 us (74 %); 128 with a window of 1024, 16 / 2 of 128, 28 us (71 %: 64 to 148 such
// requests 16.9 to 31.5 us, which is 6.0 TB/s behind 5.7 us of launch, first blocks and join); 64 of 128 to 1024, 16 / 2 of 64, 8.2 us
// (33 %: bound by the longest request, whose eight warps have four blocks each, 1.3 us a block behind 3.9 us of launch, look-ups and
// join; 38 requests of 1024 each take 9.0 us, 64 9.3; of 512 6.6 and 6.9, of 256 4.9 and 5.3, of 32 3.9 and 4.0).
#pragma once

#include <atomic>

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
    const int begin = a.cu_seqlens[lo], end = a.cu_seqlens[lo + 1];
    if (begin < 0 || end > a.T) return r;  // (a range that leaves the rows of q counts as none)
    r.req = lo;
    ctx = (int64_t)a.context_lens[lo] - (end - 1 - row);
  }
  ctx = ctx < 0 ? 0 : ctx;
  const int64_t held = min(ctx, (int64_t)a.table_width * a.cache.block_size);
  const int64_t first = a.window > 0 ? max((int64_t)0, ctx - a.window) : 0;
  r.first = (int)first;
  r.n_sink = (int)min((int64_t)a.sinks, min(first, held));
  r.n_keys = r.n_sink + (int)max((int64_t)0, held - first);
  return r;
}

// Probabilities are 2^(score - m) of a reference m that any value near the maximum may be, since it leaves with the sum. It moves, to
// kProbUp below the maximum, where the maximum has grown to more than kProbSlack + kProbUp above it: until then O stays as it is and
// probabilities stay below 2^(kProbSlack + kProbUp). In fp16 they go up to 2^15 of its 2^16, so that those from 2^-21 of the largest
// on are normal numbers and what rounding does to smaller ones is at most 2^-32 of it: keys of a long context that one outweighs by
// 2^25 would else count in the sum and be zero in the product. (Slack 8, 6, 4 of these 15: a window of 1024 over 8001 tokens, heads of
// 128, 91, 93, 96 us.)
template <bool kF16> constexpr float kProbUp = kF16 ? 7.f : 0.f;
constexpr float kProbSlack = 8.f;

constexpr int kJoinThreads = 128;
constexpr int kPagedStages = 3;
constexpr int kPagedCtas = 2 * 148;  // of a launch, of four warps: two on every SM
template <int D>
__host__ __device__ constexpr int paged_block_keys() { return D == 64 ? 32 : 16; }  // 8 KB of K and V rows
template <int D>
__host__ __device__ constexpr int paged_stage_bytes() { return 2 * paged_block_keys<D>() * (D * 2 + 16); }
template <int D, int NT>
__host__ __device__ constexpr int paged_smem(int warps) { return 2 * 8 * NT * (D * 2 + 16) + warps * kPagedStages * paged_stage_bytes<D>(); }

__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Joined or single result of a head's two columns
template <bool kF16>
__device__ __forceinline__ void store_result(const PagedArgs& a, int row, int head, int d, float x, float y, float m, float l) {
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (no visible key: zeros; NaN stays)
  char* dst = static_cast<char*>(a.out) + 2 * (row * a.out_token + head * a.out_head + d);
  *reinterpret_cast<uint32_t*>(dst) = pack_16x2<kF16>(x * inv, y * inv);
  if (a.lse != nullptr && d == 0) a.lse[(int64_t)row * a.Hq + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
}

// Blocks [u0, u1) of the keys of one (row, kv head, chunk of its q heads)
struct PagedPiece {
  int row, kvh, head0, n_heads, u0, u1, n_units;  // n_units: of the whole item; row < 0: none
  RowKeys keys;
};

// Walks the pieces of a CTA: whole items in turn, or an equal share of the blocks of all items.
template <int kKeys>
struct PagedWalk {
  long long at, end, row_at;  // share: units; first unit of `row`
  int row, step;              // step > 0: items `at`, at + step, ..., of each the rank-th of `ranks` parts
  int rank, ranks;
  static __device__ __forceinline__ int units(const RowKeys& r) { return r.n_keys < 0 ? 0 : max(1, (int)(((unsigned)r.n_keys + kKeys - 1u) / kKeys)); }
  __device__ __forceinline__ PagedPiece next(const PagedArgs& a) {
    const int per_row = a.Hk * a.chunks, group = a.Hq / a.Hk;
    PagedPiece w;
    w.row = -1;
    int item = 0;
    while (at < end) {
      if (step > 0) {
        row = (int)(at / per_row);
        item = (int)(at - (long long)row * per_row);
        at += step;
        w.keys = row_keys(a, row);
        w.n_units = units(w.keys);
        if (w.n_units == 0) continue;
        w.u0 = (int)((int64_t)w.n_units * rank / ranks);
        w.u1 = (int)((int64_t)w.n_units * (rank + 1) / ranks);
      } else {
        w.keys = row_keys(a, row);
        w.n_units = units(w.keys);
        if (at >= row_at + (long long)w.n_units * per_row) {
          row_at += (long long)w.n_units * per_row;
          ++row;
          continue;
        }
        const unsigned in_row = (unsigned)(at - row_at);
        item = (int)(in_row / (unsigned)w.n_units);
        w.u0 = (int)(in_row - (unsigned)item * (unsigned)w.n_units);
        w.u1 = (int)min((long long)w.n_units, w.u0 + (end - at));
        at += w.u1 - w.u0;
      }
      w.row = row;
      w.kvh = item / a.chunks;
      const int chunk = item - w.kvh * a.chunks;
      w.head0 = w.kvh * group + chunk * a.heads;
      w.n_heads = min(a.heads, group - chunk * a.heads);
      return w;
    }
    return w;
  }
};

// Four warps (two CTAs on an SM) or eight take the blocks of an item in turn, each through a ring of its own; the keys are the rows of the matrix
// instruction (S^T = K Q^T, then O^T = V^T P^T), so that eight heads fill it. What the next piece needs first (its lengths, table
// entries, queries, two blocks) is asked for ahead of the end of this one.
// kWay: whose the items are
constexpr int kWhole = 0, kShares = 1, kClusters = 2;  // one CTA's each; of a share of all blocks; a cluster's each, joined in its shared memory

template <int D, int NT, bool kF16, int kWay, int kPagedWarps>
__global__ void __launch_bounds__(32 * kPagedWarps, 8 / kPagedWarps) paged_decode_kernel(const PagedArgs a) {
  extern __shared__ __align__(16) uint8_t paged_smem_raw[];  // (a name of its own: 1024-byte alignment would cost heads of 64 the second CTA)
  uint8_t* const smem = paged_smem_raw;
  constexpr int kPagedThreads = 32 * kPagedWarps;
  constexpr int kPitch = D * 2 + 16, kKeys = paged_block_keys<D>(), kStage = paged_stage_bytes<D>(), kPieces = D / 8;
  constexpr int kMT = kKeys / 16, kPerLoad = 32 / kPieces;  // rows of a load instruction
  constexpr int kQ = 8 * NT * kPitch, kQEach = (8 * NT * kPieces + kPagedThreads - 1) / kPagedThreads;
  static_assert(8 * NT * (D + 2) * 4 <= kStage, "a warp's result lies in one stage");
  __shared__ int s_row;
  __shared__ long long s_at, s_sum[kPagedWarps];
  __shared__ uint32_t s_live[kPagedWarps][kPagedStages];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int per_row = a.Hk * a.chunks;
  using Walk = PagedWalk<kKeys>;
  constexpr bool kShare = kWay == kShares;
  uint32_t rank = 0, ranks = 1;
  if (kWay == kClusters) {
    rank = cluster_ctarank();
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  }
  glue_enter();

  Walk walk;
  long long total = 0;
  int G = gridDim.x;
  if (!kShare) {
    walk.step = (int)(gridDim.x / ranks);
    walk.at = blockIdx.x / ranks;
    walk.rank = (int)rank;
    walk.ranks = (int)ranks;
    walk.end = (long long)a.T * per_row;
  } else {
    // where this CTA's share begins: sums over the rows, a thread a run of them
    const int rows_each = (a.T + kPagedThreads - 1) / kPagedThreads;
    long long sum = 0;
    for (int i = 0, row = tid * rows_each; i < rows_each && row < a.T; ++i, ++row) sum += Walk::units(row_keys(a, row));
    long long upto = sum;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    if (lane == 31) s_sum[warp] = upto;
    __syncthreads();
    long long ahead = 0;
#pragma unroll
    for (int w = 0; w < kPagedWarps; ++w) {
      if (w < warp) ahead += s_sum[w];
      total += s_sum[w];
    }
    total *= per_row;
    G = (int)max(1ll, min((long long)gridDim.x, total / kPagedWarps));  // shares of a block for every warp, or more
    if (tid == 0) a.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if ((int)blockIdx.x >= G || total == 0) return;
    walk.step = 0;
    walk.at = total * blockIdx.x / G;
    walk.end = total * (blockIdx.x + 1) / G;
    const long long to = (ahead + upto) * per_row, from = to - sum * per_row;
    if (from <= walk.at && walk.at < to) {
      long long at = from;
      int row = tid * rows_each;
      for (;; ++row) {
        const long long n = (long long)Walk::units(row_keys(a, row)) * per_row;
        if (walk.at < at + n) break;
        at += n;
      }
      s_row = row;
      s_at = at;
    }
    __syncthreads();
    walk.row = s_row;
    walk.row_at = s_at;
  }

  const uint32_t q_u32 = smem_u32(smem), ring_at = 2 * kQ + warp * kPagedStages * kStage, ring = q_u32 + ring_at;
  const char *k_base = static_cast<const char*>(a.cache.k), *v_base = static_cast<const char*>(a.cache.v);
  // The block of the cache that holds the lane's key of block u, -1: none. (One block ahead of its use: a look-up takes as long as
  // the rows themselves.)
  auto entry = [&](const PagedPiece& w, int u) {
    const int i = u * kKeys + lane;
    if (w.row < 0 || u >= w.u1 || lane >= kKeys || i >= w.keys.n_keys) return -1;
    return a.tables[w.keys.req * a.table_ld + w.keys.key(i) / a.cache.block_size];
  };
  auto load = [&](const PagedPiece& w, int u, int blk, int stage) {
    if (w.row >= 0 && u < w.u1) {
      const bool live = (unsigned)blk < (unsigned)a.cache.num_blocks;  // (an entry outside the cache: its keys are left out)
      int64_t kr = 0, vr = 0;
      if (live) {
        const int in_block = w.keys.key(u * kKeys + lane) % a.cache.block_size;
        kr = 2 * (blk * a.cache.k_block + in_block * a.cache.k_token + w.kvh * a.cache.k_head);
        vr = 2 * (blk * a.cache.v_block + in_block * a.cache.v_token + w.kvh * a.cache.v_head);
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
  auto after = [](int stage, int n) { return stage + n >= kPagedStages ? stage + n - kPagedStages : stage + n; };
  // a thread's pieces of q of the piece's heads; unused rows are zero
  uint4 q_piece[kQEach];
  auto load_q = [&](const PagedPiece& w) {
#pragma unroll
    for (int e = 0; e < kQEach; ++e) {
      const int i = tid + e * kPagedThreads, h = i / kPieces, p = i - h * kPieces;
      q_piece[e] = make_uint4(0, 0, 0, 0);
      if (w.row >= 0 && h < w.n_heads)
        q_piece[e] = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.q) + 2 * (w.row * a.q_token + (w.head0 + h) * a.q_head + p * 8));
    }
  };
  auto put_q = [&](int buf) {
#pragma unroll
    for (int e = 0; e < kQEach; ++e) {
      const int i = tid + e * kPagedThreads, h = i / kPieces, p = i - h * kPieces;
      if (h < 8 * NT) sts128(q_u32 + (uint32_t)(buf * kQ + h * kPitch + p * 16), q_piece[e]);
    }
  };

  PagedPiece w = walk.next(a);
  int stage = 0, buf = 0;
  bool first_piece = true;
  {
    const int e0 = entry(w, w.u0 + warp), e1 = entry(w, w.u0 + warp + kPagedWarps);
    load_q(w);
    load(w, w.u0 + warp, e0, 0);
    load(w, w.u0 + warp + kPagedWarps, e1, 1);
    put_q(0);
  }
  while (w.row >= 0) {
    int e = entry(w, w.u0 + warp + 2 * kPagedWarps);
    const PagedPiece following = walk.next(a);
    const int e0 = entry(following, following.u0 + warp), e1 = entry(following, following.u0 + warp + kPagedWarps);
    load_q(following);
    if (kWay == kClusters) {
      cluster_arrive();
      cluster_wait();
    } else {
      __syncthreads();  // q is there; the stages that held results may be filled again
    }
    uint32_t qf[NT][D / 16][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        uint32_t r[4];
        ldsm_x4(q_u32 + (uint32_t)(buf * kQ + (8 * n + (lane & 7)) * kPitch + (lane >> 3) * 16 + 64 * k), r);
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
    for (int u = w.u0 + warp; u < w.u1; u += kPagedWarps) {
      load(w, u + 2 * kPagedWarps, e, after(stage, 2));
      e = entry(w, u + 3 * kPagedWarps);
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
      bool grows = false;  // scores, masked
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < kMT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const bool seen = (live >> (16 * i + g + 8 * (x >> 1))) & 1u;
            s[n][i][x] = seen ? s[n][i][x] * a.sc : -INFINITY;
            grows |= s[n][i][x] > m[n][x & 1] + (kProbSlack + kProbUp<kF16>);
          }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = m[n][c];
#pragma unroll
            for (int i = 0; i < kMT; ++i) mx = fmaxf(mx, fmaxf(s[n][i][c], s[n][i][c + 2]) - kProbUp<kF16>);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float f = mx == -INFINITY ? 1.f : ex2(m[n][c] - mx);
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
          for (int x = 0; x < 4; ++x) {
            const float top = m[n][x & 1];
            s[n][i][x] = ex2(s[n][i][x] - (top == -INFINITY ? 0.f : top));
            l[n][x & 1] += s[n][i][x];
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
      stage = after(stage, 1);
    }
    load(following, following.u0 + warp, e0, stage);
    load(following, following.u0 + warp + kPagedWarps, e1, after(stage, 1));
    put_q(buf ^ 1);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 4);
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 8);
        l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], 16);
      }
    // the warps' results, each in the third stage of its ring, where nothing is under way
    __shared__ int s_third[kPagedWarps];
    float* const mine = reinterpret_cast<float*>(smem + ring_at + after(stage, 2) * kStage);
    if (lane == 0) s_third[warp] = after(stage, 2);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int h = 8 * n + 2 * t + c;
        float* dst = mine + h * D + g;
#pragma unroll
        for (int d = 0; d < D / 16; ++d) { dst[16 * d] = o[n][d][c]; dst[16 * d + 8] = o[n][d][c + 2]; }
        if (g == 0) { mine[8 * NT * D + 2 * h] = m[n][c]; mine[8 * NT * D + 2 * h + 1] = l[n][c]; }
      }
    __syncthreads();
    const float* part[kPagedWarps];
#pragma unroll
    for (int k = 0; k < kPagedWarps; ++k) part[k] = reinterpret_cast<const float*>(smem + 2 * kQ + (k * kPagedStages + s_third[k]) * kStage);
    __shared__ float2 s_ml[8 * NT];
    const bool whole = !kShare || (w.u0 == 0 && w.u1 == w.n_units);
    const int slot = 2 * blockIdx.x + (first_piece ? 0 : 1);
    for (int i = tid; i < w.n_heads * (D / 2); i += kPagedThreads) {
      const int h = i / (D / 2), d = 2 * (i - h * (D / 2));
      float top = -INFINITY;
#pragma unroll
      for (int k = 0; k < kPagedWarps; ++k) top = fmaxf(top, part[k][8 * NT * D + 2 * h]);
      float sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int k = 0; k < kPagedWarps; ++k) {
        const float2 ml = *reinterpret_cast<const float2*>(part[k] + 8 * NT * D + 2 * h), v = *reinterpret_cast<const float2*>(part[k] + h * D + d);
        const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
        sum += f * ml.y;
        x += f * v.x;
        y += f * v.y;
      }
      if (kWay == kClusters) {  // (in place: no other thread reads or writes these two columns)
        *reinterpret_cast<float2*>(const_cast<float*>(part[0]) + h * D + d) = make_float2(x, y);
        if (d == 0) s_ml[h] = make_float2(top, sum);
      } else if (whole) {
        store_result<kF16>(a, w.row, w.head0 + h, d, x, y, top, sum);
      } else {
        const int64_t at_slot = (int64_t)slot * a.heads + h;
        *reinterpret_cast<float2*>(a.part_o + at_slot * D + d) = make_float2(x, y);
        if (d == 0) *reinterpret_cast<float2*>(a.part_ml + at_slot * 2) = make_float2(top, sum);
      }
    }
    if (kWay == kClusters) {
      // the cluster's parts: every CTA joins some of the columns
      cluster_arrive();
      cluster_wait();
      const int all = w.n_heads * (D / 2);
      for (int i = (int)((int64_t)all * rank / ranks) + tid, to = (int)((int64_t)all * (rank + 1) / ranks); i < to; i += kPagedThreads) {
        const int h = i / (D / 2), d = 2 * (i - h * (D / 2));
        float2 ml[8], v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          ml[c] = make_float2(-INFINITY, 0.f);
          v[c] = make_float2(0.f, 0.f);
          if (c < (int)ranks) {
            ml[c] = ld_cluster_f32x2(mapa_shared(smem_u32(&s_ml[h]), c));
            const uint32_t third = ld_cluster_u32(mapa_shared(smem_u32(&s_third[0]), c));
            v[c] = ld_cluster_f32x2(mapa_shared(q_u32 + 2 * kQ + third * kStage + 4 * (h * D + d), c));
          }
        }
        float top = -INFINITY, sum = 0.f, x = 0.f, y = 0.f;
#pragma unroll
        for (int c = 0; c < 8; ++c) top = fmaxf(top, ml[c].x);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          const float f = ml[c].x == -INFINITY ? 0.f : ex2(ml[c].x - top);
          sum += f * ml[c].y;
          x += f * v[c].x;
          y += f * v[c].y;
        }
        store_result<kF16>(a, w.row, w.head0 + h, d, x, y, top, sum);
      }
    }
    // the CTA that begins an item and does not end it says who ends it: the last one whose share begins before the item's end
    if (kShare && w.u0 == 0 && !whole && tid == 0) {
      const long long item_end = total * (blockIdx.x + 1) / G + (w.n_units - w.u1);  // (its last piece)
      int last = (int)min((long long)G - 1, (item_end * G - 1) / total);
      while (last + 1 < G && total * (last + 1) / G < item_end) ++last;  // (the shares' bounds are rounded down)
      while (total * last / G >= item_end) --last;
      a.joins[blockIdx.x] = make_int4(w.row, w.head0, slot, last);
    }
    first_piece = false;
    buf ^= 1;
    w = following;
  }
  cp_async_wait_group<0>();
  if (kWay == kClusters) {  // (no CTA leaves while another reads its part)
    cluster_arrive();
    cluster_wait();
  }
}

// Joins the parts of the item that begins in CTA blockIdx.x: its own, then the first one of every CTA up to the last; one of its
// heads (blockIdx.y). D / 4 threads keep four columns each; groups of them take the parts in turn.
template <int D, bool kF16>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedArgs a) {
  constexpr int kLanes = D / 4, kGroups = kJoinThreads / kLanes;
  __shared__ float4 s_o[kGroups][kLanes];
  __shared__ float2 s_ml[kGroups];
  glue_enter();
  const int4 j = a.joins[blockIdx.x];
  const int group = a.Hq / a.Hk, in_group = j.y % group, n_heads = min(a.heads, group - in_group);
  if (j.x < 0 || (int)blockIdx.y >= n_heads) return;
  const int parts = j.w - (int)blockIdx.x + 1, c = threadIdx.x % kLanes, mine = threadIdx.x / kLanes;
  auto slot_of = [&](int k) { return (int64_t)(k == 0 ? j.z : 2 * ((int)blockIdx.x + k)) * a.heads + blockIdx.y; };
  auto stats = [&](int k) { return *reinterpret_cast<const float2*>(a.part_ml + slot_of(k) * 2); };
  float top = -INFINITY, sum = 0.f;
#pragma unroll 8
  for (int k = 0; k < parts; ++k) top = fmaxf(top, stats(k).x);
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int k = mine; k < parts; k += kGroups) {
    const float2 ml = stats(k);
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + slot_of(k) * D + 4 * c);
    const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
    sum += f * ml.y;
    o = make_float4(o.x + f * v.x, o.y + f * v.y, o.z + f * v.z, o.w + f * v.w);
  }
  s_o[mine][c] = o;
  if (c == 0) s_ml[mine].y = sum;
  __syncthreads();
  if (mine != 0) return;
  for (int k = 1; k < kGroups; ++k) {
    const float4 v = s_o[k][c];
    sum += s_ml[k].y;
    o = make_float4(o.x + v.x, o.y + v.y, o.z + v.z, o.w + v.w);
  }
  store_result<kF16>(a, j.x, j.y + blockIdx.y, 4 * c, o.x, o.y, top, sum);
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  *reinterpret_cast<uint32_t*>(static_cast<char*>(a.out) + 2 * (j.x * a.out_token + (j.y + (int)blockIdx.y) * a.out_head + 4 * c + 2)) = pack_16x2<kF16>(o.z * inv, o.w * inv);
}

// Dynamic shared memory of a kernel, set once on a device (`known`: the devices that have it; half a microsecond a call otherwise)
inline int allow_smem(const void* kernel, int bytes, std::atomic<uint64_t>* known) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev < 64 && (known->load(std::memory_order_relaxed) >> dev & 1u)) return B200_LORA_OK;
  if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return fail(B200_LORA_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  if (dev < 64) known->fetch_or(1ull << dev, std::memory_order_relaxed);
  return B200_LORA_OK;
}

// How the items (row, kv head, chunk) meet the CTAs, by what the host knows: their number, and the blocks of keys of one at most
// (the table's width, the window). us, one CTA of four warps an item / of eight / clusters of 2, 4, 8 of eight / equal shares of four:
//   16 / 2 heads of 64: one request of 700 tokens (2 items, 22 blocks) 8.2 / 7.1 / 7.4, 6.6, 6.3 / 10.9; of 8000 48 / 33 / 22, 15, 10.9 /
//   15.9; of 32000 210 / 125 / 69, 39, 23.4 / 21.4; 64 of 1000 (128 items, 32 blocks) 11.9 / 10.0 / 16.5, 35, 66 / 16.7; 64 of 8000 64 / 48 /
//   53, 84, 128 / 52; 32 / 8 of 128: 8 of 300 (64, 19) 7.9 / 7.4 / 8.4, 12.5, 30 / 13.1; 8 of 2000 30 / 22 / 18.9, 24, 42 / 22;
//   16 / 2 of 128: 128 of 1000 (256, 63) 27.2 / 29.2 / 42, 97, 158 / 34
//   ragged, 48 of 500 to 8192 (384, 512) 203 / 179 / 166, 273, 368 / 138; 16 of 100 to 16000 (128, 1000) 208 / 138 / 147, 146, 210 / 109
struct PagedWay { int cluster, warps; bool shares; };
inline PagedWay paged_way(int T, int Hq, int Hk, int D, int64_t max_keys, int window, int sinks) {
  const int64_t keys = window > 0 ? std::min<int64_t>(max_keys, (int64_t)window + sinks) : max_keys, block = D == 64 ? paged_block_keys<64>() : paged_block_keys<128>();
  const int64_t units = (keys + block - 1) / block, items = (int64_t)T * Hk * ((Hq / Hk + 15) / 16);
  PagedWay w = {8, 8, false};
  while (w.cluster > 1 && items * w.cluster > 148) w.cluster /= 2;
  if (units < (w.cluster == 2 ? 64 : 20)) w.cluster = 1;
  if (items * w.cluster > 148) w.warps = 4;
  w.shares = (units > 32 * w.warps * w.cluster && items < 8 * kPagedCtas) || (w.cluster == 8 && units > 700);
  return w;
}

inline size_t paged_parts_bytes(int heads, int D) { return (size_t)2 * kPagedCtas * heads * D * 4; }
inline size_t paged_workspace_bytes(int T, int Hq, int Hk, int D, int64_t max_keys, int window, int sinks) {
  if (!paged_way(T, Hq, Hk, D, max_keys, window, sinks).shares) return 0;
  const int heads = std::min(Hq / Hk, 16);
  return paged_parts_bytes(heads, D) + (size_t)2 * kPagedCtas * heads * 8 + kPagedCtas * sizeof(int4);
}

template <int D, int NT, bool kF16, int kWay, int kWarps>
inline int paged_decode_launch_t(const PagedArgs& a, int ctas, int cluster, cudaStream_t stream) {
  const auto kernel = paged_decode_kernel<D, NT, kF16, kWay, kWarps>;
  static std::atomic<uint64_t> known{0};
  if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), paged_smem<D, NT>(kWarps), &known)) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(32 * kWarps);
  cfg.dynamicSmemBytes = paged_smem<D, NT>(kWarps);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = bgmv_options().pdl ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(B200_LORA_ECUDA, "paged_decode_kernel launch: %s", cudaGetErrorString(e));
  }
  if (kWay != kShares) return B200_LORA_OK;
  return launch_dependent(paged_join_kernel<D, kF16>, "paged_join_kernel", dim3((unsigned)ctas, (unsigned)a.heads), kJoinThreads, 0, stream, a);
}

template <int D, int NT, bool kF16>
inline int paged_decode_launch_by(const PagedArgs& a, cudaStream_t stream) {
  const PagedWay w = paged_way(a.T, a.Hq, a.Hk, D, (int64_t)a.table_width * a.cache.block_size, a.window, a.sinks);
  if (w.shares && a.part_o != nullptr) return paged_decode_launch_t<D, NT, kF16, kShares, 4>(a, kPagedCtas, 1, stream);
  const int64_t items = (int64_t)a.T * a.Hk * a.chunks;
  const int ctas = (int)std::min<int64_t>((w.warps == 8 ? 148 : kPagedCtas) / w.cluster, items) * w.cluster;
  if (w.cluster > 1) return paged_decode_launch_t<D, NT, kF16, kClusters, 8>(a, ctas, w.cluster, stream);
  if (w.warps == 8) return paged_decode_launch_t<D, NT, kF16, kWhole, 8>(a, ctas, 1, stream);
  return paged_decode_launch_t<D, NT, kF16, kWhole, 4>(a, ctas, 1, stream);
}

inline int paged_decode_launch(PagedArgs a, int D, int dtype, void* workspace, cudaStream_t stream) {
  const int group = a.Hq / a.Hk;
  a.heads = std::min(group, 16);
  a.chunks = ceil_div_i(group, a.heads);
  if (workspace != nullptr) {  // (null: no shares)
    char* ws = static_cast<char*>(workspace);
    a.part_o = reinterpret_cast<float*>(ws);
    a.part_ml = reinterpret_cast<float*>(ws + paged_parts_bytes(a.heads, D));
    a.joins = reinterpret_cast<int4*>(ws + paged_parts_bytes(a.heads, D) + (size_t)2 * kPagedCtas * a.heads * 8);
  }
  const bool f16 = dtype == B200_LORA_F16, wide = a.heads > 8;
  if (D == 64) {
    if (wide) return f16 ? paged_decode_launch_by<64, 2, true>(a, stream) : paged_decode_launch_by<64, 2, false>(a, stream);
    return f16 ? paged_decode_launch_by<64, 1, true>(a, stream) : paged_decode_launch_by<64, 1, false>(a, stream);
  }
  if (wide) return f16 ? paged_decode_launch_by<128, 2, true>(a, stream) : paged_decode_launch_by<128, 2, false>(a, stream);
  return f16 ? paged_decode_launch_by<128, 1, true>(a, stream) : paged_decode_launch_by<128, 1, false>(a, stream);
}

}  // namespace b200lora
