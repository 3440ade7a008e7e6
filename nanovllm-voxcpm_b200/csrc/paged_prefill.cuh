// Attention of packed new tokens over a paged key-value cache on the tensor cores: bf16 and fp16, causal, over everything or over
// a sliding window of the last keys plus a few first ones.
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t, h] . k_j - max),  over the keys j that token t sees
//
// A CTA takes two tiles of 128 rows of one sequence and kv head: a row is a (token, query head), heads of a group inside, so that
// a K / V tile brought in once serves them all and a tile spans few tokens (16 with eight heads: little masked work at the
// diagonal and at the window's edge). Tiles of 128 keys: S = Q K^T and O += P V by tcgen05.mma with fp32 accumulators in tensor
// memory, P (rounded to the type of V) in the columns of S; a warpgroup per tile does the softmax, a thread per row. While one
// tile's softmax runs, the other tile's products do.
#pragma once

#include "paged_attention.cuh"
#include "tc_common.cuh"

namespace b200lora {

constexpr int kPpRows = 128, kPpKeys = 128;       // of a tile
#ifndef B200_POLY
#define B200_POLY 16
#endif
constexpr int kPpPolyEvery = B200_POLY;
constexpr int kPpPanel = kPpKeys * 128;           // bytes of 128 rows of 64 columns
// One softmax warpgroup per tile; one more with the loading warp and the MMA warp, which leaves its registers to them. Two tiles: 168
// registers a thread at launch, 384 * 168 = 64512, and 2 * 208 + 88 = 3 * 168; one tile, two CTAs on an SM: 128, and 208 + 48 = 2 * 128.
__host__ __device__ constexpr int pp_threads(int tiles) { return 128 * (tiles + 1); }
constexpr int kPpSoftmaxRegs = 208;
__host__ __device__ constexpr int pp_other_regs(int tiles) { return tiles == 2 ? 88 : 48; }
template <int D>
__host__ __device__ constexpr int pp_stages(int tiles) { return (D == 64 ? 1 : 0) + tiles; }
template <int D>
__host__ __device__ constexpr int pp_tile() { return kPpKeys * D * 2; }
template <int D>
__host__ __device__ constexpr int pp_smem(int tiles) { return (2 * pp_stages<D>(tiles) + tiles) * pp_tile<D>() + 1024; }

struct PpMaps { CUtensorMap q, k, v; };
struct PpArgs {
  PagedArgs p;
  int h_shift, head_tiles;   // heads of a tile = 1 << h_shift; tiles over all heads
  int n_blocks;              // blocks of tokens that the launch has CTAs for
  int box;                   // cache rows of a copy: 8 .. 128, a power of two that divides the block size
  int k_heads_inner, v_heads_inner;  // order of the map's middle dimensions: (head, position) or (position, head)
};

__device__ __forceinline__ void tma_load_3d_at(uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst), "l"(m),
               "r"(c0), "r"(c1), "r"(c2), "r"(bar)
               : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst), "l"(m),
               "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
               : "memory");
}
// D (+)= A . B with A in tensor memory, where `leader`
__device__ __forceinline__ void umma_ts_elected(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate,
                                                uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\tsetp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(leader)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
      "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// mbar_wait_bounded with its polls in place: a call would set the registers of the roles to the launch's number
__device__ __forceinline__ void pp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  for (int it = 0; it < kSpinLimit; ++it) {
    if (mbar_try_wait(bar, parity)) return;
    if (*abort_flag != 0) return;
  }
  *abort_flag = 1;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (NaN where one of them is)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x for x <= 8 or so on the FMA units: x = n + f with n whole and f in [-0.5, 0.5] (adding and subtracting 1.5 * 2^23 rounds to n), 2^f
// by a polynomial with constant term 1, least in its largest relative error (1.7e-7 in fp32; weighted least squares until the
// extrema are even), n added to the exponent. From -127 down exactly 0.
__device__ __forceinline__ float2 exp2_poly(float2 x) {
  constexpr float kRound = 12582912.f;
  x = make_float2(fmaxf(x.x, -127.f), fmaxf(x.y, -127.f));
  const float2 t = add2(x, make_float2(kRound, kRound)), f = fma2(add2(t, make_float2(-kRound, -kRound)), make_float2(-1.f, -1.f), x);
  float2 y = fma2(f, make_float2(0x1.5bba14p-10f, 0x1.5bba14p-10f), make_float2(0x1.3cea88p-7f, 0x1.3cea88p-7f));
  y = fma2(f, y, make_float2(0x1.c6b752p-5f, 0x1.c6b752p-5f));
  y = fma2(f, y, make_float2(0x1.ebf9bcp-3f, 0x1.ebf9bcp-3f));
  y = fma2(f, y, make_float2(0x1.62e42ap-1f, 0x1.62e42ap-1f));
  y = fma2(f, y, make_float2(1.f, 1.f));
  return make_float2(__uint_as_float(__float_as_uint(y.x) + (__float_as_uint(t.x) << 23)), __uint_as_float(__float_as_uint(y.y) + (__float_as_uint(t.y) << 23)));
}
// bits [0, n) of a word, n of any sign and size
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }

template <int D, bool kF16, int kTiles>
__global__ void __launch_bounds__(pp_threads(kTiles), 3 - kTiles) paged_prefill_kernel(const __grid_constant__ PpMaps maps, const __grid_constant__ PpArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr int kSt = pp_stages<D>(kTiles), kTile = pp_tile<D>(), kPanels = D / 64;
  constexpr int kLoader = 4 * kTiles, kIssuer = kLoader + 1, kTmem = 256 * kTiles, kO = kTiles * kPpKeys;  // warps; columns: all, the first of O
  enum { Q_FULL, S_READY, P_READY = S_READY + 2, O_DONE = P_READY + 4, K_FULL = O_DONE + 2, K_FREE = K_FULL + kSt, V_FULL = K_FREE + kSt,
         V_FREE = V_FULL + kSt, N_BARS = V_FREE + kSt };
  __shared__ __align__(8) uint64_t bars[N_BARS];
  __shared__ uint32_t s_tmem, s_boxes[4];
  __shared__ volatile int abort_flag;
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const PagedArgs& p = a.p;
  // (V first: what a wrong stride of its descriptor could reach stays inside the allocation)
  const uint32_t v_u32 = (smem_u32(smem_raw) + 1023u) & ~1023u, k_u32 = v_u32 + kSt * kTile, q_u32 = k_u32 + kSt * kTile;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };

  if (tid == 0) {
    for (int i = 0; i < N_BARS; ++i) mbar_init(bar(i), i >= P_READY && i < O_DONE ? kPpRows : 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kIssuer) tmem_alloc(smem_u32(&s_tmem), kTmem);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  glue_enter();  // (dependents may start: every CTA of this launch holds its tensor memory by then)
  const uint32_t tmem = s_tmem;

  // ---- which tokens: the blocks of the sequences in order, the last ones first (their contexts are the longest)
  const int blk = a.n_blocks - 1 - (int)blockIdx.x / a.head_tiles, head0 = ((int)blockIdx.x % a.head_tiles) << a.h_shift;
  const int per_tile = kPpRows >> a.h_shift, span = kTiles * per_tile;
  int req = -1, begin = 0, len = 0, q0 = 0;
  for (int base = 0, run = 0; base < p.n_req && req < 0; base += 32) {
    const int i = base + lane;
    int b = 0, n = 0;
    if (i < p.n_req) {
      b = p.cu_seqlens[i];
      const int e = p.cu_seqlens[i + 1];
      n = b >= 0 && e <= p.T && e > b ? e - b : 0;
    }
    int upto = (n + span - 1) / span;
    const int mine = upto;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int v = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += v;
    }
    const uint32_t hit = __ballot_sync(0xffffffffu, run + upto > blk);
    if (hit != 0) {
      const int who = __ffs(hit) - 1;
      req = base + who;
      begin = __shfl_sync(0xffffffffu, b, who);
      len = __shfl_sync(0xffffffffu, n, who);
      q0 = (blk - run - __shfl_sync(0xffffffffu, upto - mine, who)) * span;
    }
    run += __shfl_sync(0xffffffffu, upto, 31);
  }
    const int n_here = req < 0 ? 0 : min(span, len - q0);                             // tokens of this CTA
    const int ctx = req < 0 ? 0 : max(p.context_lens[req], 0), pos0 = ctx - len + q0;  // position of the first
    const int held = (int)min((int64_t)min(ctx, INT32_MAX - 255), (int64_t)p.table_width * p.cache.block_size);
    const int key_end = min(pos0 + n_here, held);                                     // keys that any row sees: [0, sink_end) and
    const int lo_first = p.window > 0 ? max(0, max(pos0, 0) - (p.window - 1)) : 0;    // [lo_first, key_end)
    const int sink_end = max(0, min(min(p.sinks, lo_first), key_end));
    const int first_tile = lo_first / kPpKeys, sink_tiles = min((sink_end + kPpKeys - 1) / kPpKeys, first_tile);
    const int n_tiles = key_end <= 0 || n_here == 0 ? 0 : sink_tiles + max(0, (key_end + kPpKeys - 1) / kPpKeys - first_tile);
    auto key0_of = [&](int i) { return (i < sink_tiles ? i : i - sink_tiles + first_tile) * kPpKeys; };

    if (warp < kLoader) {  // ------------------------------------------------------------------- softmax
      asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPpSoftmaxRegs));
      const int t = warp >> 2, row = (warp & 3) * 32 + lane, tok = t * per_tile + (row >> a.h_shift), head = head0 + (row & ((1 << a.h_shift) - 1));
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t s_at = tmem + t * kPpKeys + lanes, o_at = tmem + kO + t * D + lanes;
      const int pos = pos0 + tok;
      const int lo = p.window > 0 ? max(pos, 0) - (p.window - 1) : 0;
      const int tile_lo = pos0 + t * per_tile, tile_hi = tile_lo + per_tile - 1;  // positions of the tile
      const uint32_t all_boxes = bits_below(kPpKeys / a.box);
      const int box_shift = 31 - __clz(a.box);
      float m = -INFINITY, l = 0.f;  // maximum that the probabilities refer to, in units of log2; their sum
      for (int i = 0; i < n_tiles; ++i) {
        const int key0 = key0_of(i);
        pp_wait(bar(S_READY + t), (uint32_t)(i & 1), &abort_flag);
        tc_fence_after_sync();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld_32x32(s_at + 32 * c, s[c]);
        const uint32_t boxes = s_boxes[i & 3];
        const bool masked = key0 + kPpKeys - 1 > tile_lo || (p.window > 0 && key0 < max(tile_hi, 0) - (p.window - 1) && key0 + kPpKeys > p.sinks) || boxes != all_boxes;
        float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          tmem_ld_wait();
          if (half == 0) {
#pragma unroll
            for (int c = 2; c < 4; ++c) tmem_ld_32x32(s_at + 32 * c, s[c]);
          }
#pragma unroll
          for (int c = 2 * half; c < 2 * half + 2; ++c) {
            if (masked) {
              const int at = key0 + 32 * c;
              uint32_t seen = bits_below(pos + 1 - at) & (~bits_below(lo - at) | bits_below(p.sinks - at));
              uint32_t there = 0;  // (a copy has 8 rows or more)
#pragma unroll
              for (int g = 0; g < 4; ++g) there |= (boxes >> ((32 * c + 8 * g) >> box_shift)) & 1u ? 0xffu << (8 * g) : 0u;
              seen &= there;
              asm volatile("" : "+r"(seen));  // (one word at a time: 128 tests at once cost 350 bytes of spills)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!((seen >> j) & 1u)) s[c][j] = 0xff800000u;  // -inf
            }
#pragma unroll
            for (int j = 0; j < 32; j += 2) top4[j / 2 % 4] = max3(top4[j / 2 % 4], __uint_as_float(s[c][j]), __uint_as_float(s[c][j + 1]));
          }
        }
        const float mx = max3(max3(top4[0], top4[1], top4[2]), top4[3], top4[3]);
        // The maximum moves only where it would grow by more than 2^8: until then probabilities stay below that, and O as it is.
        const float top = mx * p.sc;
        const bool grows = !(top <= m + 8.f);  // (a NaN among the scores makes the maximum and with it the whole row NaN)
        if (__any_sync(0xffffffffu, grows)) {
          const float f = grows ? ex2(m - top) : 1.f;
          if (grows) m = top;
          l *= f;
          if (i > 0) {  // (S of this tile came behind P V of the one before: O is complete)
#pragma unroll
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld_32x16(o_at + 16 * c, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st_32x16(o_at + 16 * c, o);
            }
          }
        }
        const float base = m == -INFINITY ? 0.f : fmaf(m, 0.f, -m);  // (an infinite score: NaN, as inf - inf)
        const float2 scale2 = make_float2(p.sc, p.sc), base2 = make_float2(base, base);
        float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t packed[16];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 x = fma2(make_float2(__uint_as_float(s[c][j]), __uint_as_float(s[c][j + 1])), scale2, base2);
            const float2 y = j % kPpPolyEvery == kPpPolyEvery - 2 ? exp2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
            sum[j / 2 % 2] = add2(sum[j / 2 % 2], y);
            packed[j / 2] = pack_16x2<kF16>(y.x, y.y);  // (rounded to the type of V; the sum is that of the unrounded ones)
          }
          tmem_st_32x16(s_at + 16 * c, packed);
          if (c & 1) {  // half of P: its products may begin
            tmem_st_wait();
            tc_fence_before_sync();
            mbar_arrive(bar(P_READY + 2 * t + (c >> 1)));
          }
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      const bool live = tok < n_here;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (no visible key: zeros; NaN stays)
      const int64_t token = begin + q0 + tok;
      char* dst = static_cast<char*>(p.out) + 2 * (token * p.out_token + head * p.out_head);
      if (n_tiles > 0) {
        pp_wait(bar(O_DONE + t), 0, &abort_flag);
        tc_fence_after_sync();
      }
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n_tiles > 0) {
          tmem_ld_32x32(o_at + 32 * c, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0;
        }
        if (live) {
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 v;
            v.x = pack_16x2<kF16>(__uint_as_float(o[j]) * inv, __uint_as_float(o[j + 1]) * inv);
            v.y = pack_16x2<kF16>(__uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv);
            v.z = pack_16x2<kF16>(__uint_as_float(o[j + 4]) * inv, __uint_as_float(o[j + 5]) * inv);
            v.w = pack_16x2<kF16>(__uint_as_float(o[j + 6]) * inv, __uint_as_float(o[j + 7]) * inv);
            stg128(dst + 2 * (32 * c + j), v);
          }
        }
      }
      if (live && p.lse != nullptr) p.lse[token * p.Hq + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      tc_fence_before_sync();
    } else {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(pp_other_regs(kTiles)));
      if (warp == kLoader) {  // ------------------------------------------------------------------ loads
        const uint32_t leader = elect_one();
        const int kvh = head0 / (p.Hq / p.Hk);
        const int32_t* table = p.tables + req * p.table_ld;
        if (n_tiles > 0) {
          if (leader) {
            mbar_arrive_expect_tx(bar(Q_FULL), kTiles * kTile);
            for (int t = 0; t < kTiles; ++t)
              for (int c = 0; c < kPanels; ++c)
                tma_load_3d_at(q_u32 + t * kTile + c * kPpPanel, &maps.q, 64 * c, head0, begin + q0 + t * per_tile, bar(Q_FULL));
          }
          const int n_boxes = kPpKeys / a.box;
          for (int i = 0; i < n_tiles; ++i) {
            const int st = i % kSt, key = key0_of(i) + lane * a.box;
            int block = -1, in_block = 0;
            if (lane < n_boxes && key < held) {
              const int page = key / p.cache.block_size;
              block = table[page];
              in_block = key - page * p.cache.block_size;
            }
            const bool there = (unsigned)block < (unsigned)p.cache.num_blocks;
            if (!there) { block = p.cache.num_blocks; in_block = 0; }  // outside the map: zeros
            const uint32_t boxes = __ballot_sync(0xffffffffu, there);
            for (int which = 0; which < 2; ++which) {
              const uint32_t full = bar((which ? V_FULL : K_FULL) + st);
              if (i >= kSt) pp_wait(bar((which ? V_FREE : K_FREE) + st), (uint32_t)((i / kSt - 1) & 1), &abort_flag);
              if (leader) {
                if (which == 0) s_boxes[i & 3] = boxes;  // (read up to kSt tiles later: fewer than four)
                mbar_arrive_expect_tx(full, kTile);
              }
              __syncwarp();
              if (lane < n_boxes) {
                const uint32_t dst = (which ? v_u32 : k_u32) + st * kTile + lane * a.box * 128;
                const bool inner = which ? a.v_heads_inner : a.k_heads_inner;
                for (int c = 0; c < kPanels; ++c)
                  tma_load_4d(dst + c * kPpPanel, which ? &maps.v : &maps.k, 64 * c, inner ? kvh : in_block, inner ? in_block : kvh, block, full);
              }
            }
          }
        }
      } else if (warp == kIssuer) {  // ---------------------------------------------------------- products
        const uint32_t leader = elect_one();
        const uint32_t type = kF16 ? 0u : (1u << 7) | (1u << 10);
        const uint32_t idesc_s = (1u << 4) | type | ((uint32_t)(kPpKeys >> 3) << 17) | ((uint32_t)(kPpRows >> 4) << 24);
        const uint32_t idesc_o = (1u << 4) | type | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kPpRows >> 4) << 24);  // V: keys are its rows
        const uint32_t hi_k = (uint32_t)(umma_smem_desc(0, 128) >> 32);
        auto lo_k = [](uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | (1u << 16); };
        auto lo_v = [](uint32_t addr) { return ((addr & 0x3FFFF) >> 4) | ((uint32_t)(kPpPanel >> 4) << 16); };  // 64-column panels
        auto scores = [&](int t, int st) {
  #pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t at = (k >> 2) * kPpPanel + (k & 3) * 32;
            umma_elected(tmem + t * kPpKeys, lo_k(q_u32 + t * kTile + at), lo_k(k_u32 + st * kTile + at), hi_k, idesc_s, k > 0, leader);
          }
          umma_commit_elected(bar(S_READY + t), leader);
        };
        if (n_tiles > 0) {
          pp_wait(bar(Q_FULL), 0, &abort_flag);
          pp_wait(bar(K_FULL), 0, &abort_flag);
          for (int t = 0; t < kTiles; ++t) scores(t, 0);
          umma_commit_elected(bar(K_FREE), leader);
          for (int i = 0; i < n_tiles; ++i) {
            const int st = i % kSt, next = (i + 1) % kSt;
            pp_wait(bar(V_FULL + st), (uint32_t)((i / kSt) & 1), &abort_flag);
            // Rows of V that no token of this CTA sees may hold anything (a block's stale rows): they become zero, as 0 * V must.
            const int key0 = key0_of(i);
            if (!(key0 + kPpKeys <= sink_end || (key0 >= lo_first && key0 + kPpKeys <= key_end))) {
              for (int x = lane; x < kPpKeys * kPanels * 8; x += 32) {
                const int row = x / (kPanels * 8), key = key0 + row, c = x % (kPanels * 8);
                if (!(key < sink_end || (key >= lo_first && key < key_end)))
                  sts128(v_u32 + st * kTile + (c >> 3) * kPpPanel + row * 128 + (c & 7) * 16, make_uint4(0, 0, 0, 0));
              }
              fence_proxy_async_smem();
              __syncwarp();
            }
            for (int t = 0; t < kTiles; ++t) {
#pragma unroll
              for (int k = 0; k < kPpKeys / 16; ++k) {
                if (k % 4 == 0) {
                  pp_wait(bar(P_READY + 2 * t + k / 4), (uint32_t)(i & 1), &abort_flag);
                  tc_fence_after_sync();
                }
                umma_ts_elected(tmem + kO + t * D, tmem + t * kPpKeys + 8 * k, lo_v(v_u32 + st * kTile + k * 2048), hi_k, idesc_o,
                                i > 0 || k > 0, leader);
              }
              if (i + 1 < n_tiles) {
                // (behind P V of this tile in the same thread: P has been read when S is written over it)
                if (t == 0) pp_wait(bar(K_FULL + next), (uint32_t)(((i + 1) / kSt) & 1), &abort_flag);
                scores(t, next);
              } else {
                umma_commit_elected(bar(O_DONE + t), leader);
              }
            }
            if (i + 1 < n_tiles) {
              umma_commit_elected(bar(V_FREE + st), leader);
              umma_commit_elected(bar(K_FREE + next), leader);
            }
          }
        }
      }
    }
  __syncthreads();
  if (warp == kIssuer) {
    tc_fence_after_sync();
    tmem_dealloc(tmem, kTmem);
  }
  if (tid == 0 && abort_flag != 0) atomicOr(&g_b200_status, kStatusWaitGaveUp);
}

// ------------------------------------------------------------------ host
inline bool pp_map(CUtensorMap* out, const void* base, bool f16, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const EncodeTiledFn fn = encode_tiled_fn();
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  return fn != nullptr && fn(out, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), dims,
                             strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Map of K or V: columns, then heads and positions of a block by stride, then blocks
inline bool pp_cache_map(CUtensorMap* out, const lora_b200_paged_cache& c, bool v, int Hk, int D, int box, bool f16, int* heads_inner) {
  const int64_t head = v ? c.v_head : c.k_head, token = v ? c.v_token : c.k_token, block = v ? c.v_block : c.k_block;
  const bool inner = Hk == 1 || (c.block_size > 1 && head <= token);
  *heads_inner = inner ? 1 : 0;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)(inner ? Hk : c.block_size), (cuuint64_t)(inner ? c.block_size : Hk), (cuuint64_t)c.num_blocks};
  // (the stride of a dimension of one entry means nothing; any will do)
  const cuuint64_t strides[3] = {(cuuint64_t)(inner ? (Hk == 1 ? D : head) : token) * 2, (cuuint64_t)(inner ? token : head) * 2,
                                 (cuuint64_t)(c.num_blocks == 1 ? (int64_t)c.block_size * Hk * D : block) * 2};
  const cuuint32_t b[4] = {64, (cuuint32_t)(inner ? 1 : box), (cuuint32_t)(inner ? box : 1), 1};
  return head >= 0 && token >= 0 && block >= 0 && pp_map(out, v ? c.v : c.k, f16, 4, dims, strides, b);
}

// Whether the tensor-core kernel takes a call: copies of 8 cache rows or more that lie in one block, and strides that its maps take.
inline bool paged_prefill_plan(const PagedArgs& p, int D, bool f16, int tiles, PpMaps* maps, PpArgs* a) {
  if (p.cache.block_size % 8 != 0) return false;
  a->p = p;
  a->box = 8;
  while (a->box < kPpKeys && p.cache.block_size % (2 * a->box) == 0) a->box *= 2;
  const int group = p.Hq / p.Hk;
  a->h_shift = 0;
  while (a->h_shift < 4 && group % (2 << a->h_shift) == 0) ++a->h_shift;
  a->head_tiles = p.Hq >> a->h_shift;
  const int per_tile = kPpRows >> a->h_shift;
  const int64_t blocks = (int64_t)p.T / (tiles * per_tile) + p.n_req;
  if (blocks * a->head_tiles > INT32_MAX) return false;
  a->n_blocks = (int)blocks;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.Hq, (cuuint64_t)p.T};
  const cuuint64_t strides[2] = {(cuuint64_t)(p.Hq == 1 ? D : p.q_head) * 2, (cuuint64_t)(p.T == 1 ? (int64_t)p.Hq * D : p.q_token) * 2};
  const cuuint32_t box[3] = {64, 1u << a->h_shift, (cuuint32_t)per_tile};
  return p.q_head >= 0 && p.q_token >= 0 && pp_map(&maps->q, p.q, f16, 3, dims, strides, box) &&
         pp_cache_map(&maps->k, p.cache, false, p.Hk, D, a->box, f16, &a->k_heads_inner) &&
         pp_cache_map(&maps->v, p.cache, true, p.Hk, D, a->box, f16, &a->v_heads_inner);
}

template <int D, bool kF16, int kTiles>
inline int paged_prefill_launch_t(const PpMaps& maps, const PpArgs& a, cudaStream_t stream) {
  const auto kernel = paged_prefill_kernel<D, kF16, kTiles>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, pp_smem<D>(kTiles));
  if (e != cudaSuccess) return fail(B200_LORA_ECUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  return launch_dependent(kernel, "paged_prefill_kernel", dim3((unsigned)(a.n_blocks * a.head_tiles)), pp_threads(kTiles), pp_smem<D>(kTiles), stream, maps, a);
}

#ifndef B200_TILES64
#define B200_TILES64 1
#define B200_TILES128 2
#endif
inline int paged_prefill_launch(const PagedArgs& p, int D, int dtype, void* workspace, cudaStream_t stream) {
  PpMaps maps;
  PpArgs a = {};
  const bool f16 = dtype == B200_LORA_F16;
  const int tiles = D == 64 ? B200_TILES64 : B200_TILES128;
  if (!paged_prefill_plan(p, D, f16, tiles, &maps, &a)) return paged_decode_launch(p, D, dtype, workspace, stream);
  if (D == 64) return f16 ? paged_prefill_launch_t<64, true, B200_TILES64>(maps, a, stream) : paged_prefill_launch_t<64, false, B200_TILES64>(maps, a, stream);
  return f16 ? paged_prefill_launch_t<128, true, B200_TILES128>(maps, a, stream) : paged_prefill_launch_t<128, false, B200_TILES128>(maps, a, stream);
}

}  // namespace b200lora
