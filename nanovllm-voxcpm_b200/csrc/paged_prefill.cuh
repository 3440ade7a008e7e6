// Attention of packed new tokens over a paged key-value cache on the tensor cores: bf16 and fp16, causal, over everything or over
// a sliding window of the last keys plus a few first ones.
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t, h] . k_j - max),  over the keys j that token t sees
//
// A CTA takes two tiles of 128 rows of one sequence and kv head: a row is a (token, query head), heads of a group inside, so that
// a K / V tile brought in once serves them all and a tile spans few tokens (16 with eight heads: little masked work at the
// diagonal and at the window's edge). Tiles of 128 keys: S = Q K^T and O += P V by tcgen05.mma with fp32 accumulators in tensor
// memory, P (rounded to the type of V) in the columns of S; a warpgroup per tile does the softmax, a thread per row. While one
// tile's softmax runs, the other tile's products do. Heads of 64 leave columns for P: there a CTA has one tile and an SM two CTAs.
//
// Bound: the products where contexts are long, else the chain S - softmax - P V of a tile. A pair of tiles of heads of 128 takes 3000
// cycles where its products take 2048, of which a row's softmax is 2000 (128 exponentials, latency of tensor memory, one warp to a
// scheduler at a time). Measured: 8192 tokens, 16 / 2 heads of 128, 228 us = 1.20 PFLOP/s (0.73 of the measured GEMM rate), heads of 64
// 190 to 205 us (0.44); 4096 behind 12288, 32 / 8 of 128, 875 us = 1.10 PFLOP/s one after another, at the clock that the power cap leaves
// (760 us, 1.27 PFLOP/s, alone); 8001 tokens with a window of 1024, 16 / 2 of 128, 90 us = 0.70 PFLOP/s: 22.6 us for a wave of 148 items
// behind 6.3 us (2368, 4736 and 7104 tokens are one to three waves: 28.9, 51.5 and 74.1 us), and of 3.4 waves the last costs 17; 12
// prompts of 100 to 1200, heads of 64, 37 us: 3.3 us, then 1.8 us a tile (the other CTA of the SM at work too; 1.4 alone) and 2.7 us an
// item, of which the fullest CTA has 13 tiles in 3 items (960 items of 3.4 tiles; 12 equal prompts of 16 to 1200 tokens fit within 2 us).
#pragma once

#include "paged_attention.cuh"
#include "tc_common.cuh"

namespace b200lora {

constexpr int kPpRows = 128, kPpKeys = 128;       // of a tile
constexpr int kPpSinkBox = 32;
constexpr int kPpOutPitch = 80;      // bytes of 32 columns of a row in shared memory, and 16 to spread the banks
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
__host__ __device__ constexpr int pp_smem(int tiles) { return (2 * pp_stages<D>(tiles) + tiles) * pp_tile<D>() + tiles * kPpRows * kPpOutPitch + 1024; }

// Items that do not fill a wave of CTAs may be cut into parts along the keys, joined by a second launch: us, whole / cut, 16 / 2 heads,
// 16 tokens behind 8192 keys (heads of 128) 112 / 29, behind 65536 844 / 56, 500 behind 3000 (64) 42 / 25; 32 / 8 of 128, 4096 behind
// 12288 (3.5 waves of items of even length) 905 / 868. Not where every item is short, nor whole prompts of more than half a
// wave: their last items are their shortest (8192 tokens 223 / 239).
constexpr int kPpSplitTiles = 8;     // tiles of an item, at least
constexpr int kPpSplitWaves = 6;     // waves of CTAs at most
constexpr int kPpShare = 2, kPpParts = 32;  // tiles of a part at least, parts at most (the join reads them one after another)

struct PpMaps { CUtensorMap q, k, v; };
struct PpArgs {
  PagedArgs p;
  int h_shift, head_tiles;   // heads of a tile = 1 << h_shift; tiles over all heads
  int n_blocks;              // blocks of tokens that the launch has CTAs for
  int box, box_shift;        // cache rows of a copy: 8 .. 128, a power of two that divides the block size; its logarithm
  float* parts; void* joins;  // split: partial results and what there is to join
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
// (NaN where one of them is)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// 2^x for x up to 2^7 on the FMA units: x = n + f with n whole and f in [-0.5, 0.5] (adding and subtracting 1.5 * 2^23 rounds to n), 2^f
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

// Keys of a block table at most: indexes of keys, rounded up to tiles and with the columns of one added, are ints.
constexpr int kPpMaxKeys = INT32_MAX - 255;
// (positions that are not ints are those of rows behind the last token)
__device__ __forceinline__ int pp_position(int first, int n) { return (int)min((int64_t)first + n, (int64_t)INT32_MAX - 1); }

// A piece of work: tiles [i0, i1) of the keys that a block of tokens sees, for one set of heads.
struct PpPiece {
  int head0, begin, q0, n_here;                // first head; first row of the sequence; first token and tokens of the block
  int req, pos0, held, key_end, lo_first, sink_end;  // position of the first token; keys that a row sees: [0, sink_end), [lo_first, key_end)
  int first_box, sink_boxes, i0, i1;           // the keys in boxes: those of the first tokens, then from first_box on, side by side
  int parts;                                   // 0: no more pieces; 1: the whole item; else the item is in that many parts
  // first key of box b of tile i, with 1 << shift keys in a box
  __device__ __forceinline__ int key_of(int i, int b, int shift) const {
    const int c = i * (kPpKeys >> shift) + b;
    return (c < sink_boxes ? c : c - sink_boxes + first_box) << shift;
  }
};

// New rows of request i, and its first one; a range that leaves the rows of q counts as none
__device__ __forceinline__ int pp_rows(const PagedArgs& p, int i, int* begin) {
  *begin = p.cu_seqlens[i];
  const int e = p.cu_seqlens[i + 1];
  return *begin >= 0 && e <= p.T && e > *begin ? e - *begin : 0;
}
// Sum of the lanes up to this one
__device__ __forceinline__ int warp_upto(int v) {
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int u = __shfl_up_sync(0xffffffffu, v, d);
    if ((int)(threadIdx.x & 31) >= d) v += u;
  }
  return v;
}

// 32 requests, one per lane: new rows, the first of them, context; blocks of the requests up to this one
struct PpLane { int begin, len, ctx, mine, upto; };
__device__ __forceinline__ PpLane pp_lane(const PpArgs& a, int span, int i) {
  PpLane q = {0, 0, 0, 0, 0};
  if (i < a.p.n_req) {
    q.ctx = max(a.p.context_lens[i], 0);
    q.len = pp_rows(a.p, i, &q.begin);
  }
  q.mine = (q.len + span - 1) / span;
  q.upto = warp_upto(q.mine);
  return q;
}
__device__ __forceinline__ int pp_items(const PpArgs& a, int span, const PpLane& lanes0) {
  int blocks = __shfl_sync(0xffffffffu, lanes0.upto, 31);
  for (int base = 32; base < a.p.n_req; base += 32) blocks += __shfl_sync(0xffffffffu, pp_lane(a, span, base + (threadIdx.x & 31)).upto, 31);
  return min(blocks, a.n_blocks) * a.head_tiles;  // (overlapping ranges could have more)
}

// Item `item` of the n_items, longest contexts first as far as one warp can tell (up to 32 requests: blocks by the position that
// they end at; more: the last block of the last sequence first; 32 requests of 30 to 400 tokens, heads of 64, 27.2 us, 33 of them 33.3;
// of 100 each 13.9 and 14.5), the sets of heads of a block one after another. A whole warp calls
// it, with the first 32 requests in hand.
__device__ __forceinline__ void pp_find(const PpArgs& a, int span, int item, int n_items, const PpLane& lanes0, PpPiece* w) {
  const PagedArgs& p = a.p;
  const int lane = threadIdx.x & 31, back = item / a.head_tiles;
  w->head0 = (item - back * a.head_tiles) << a.h_shift;
  PpLane q = lanes0;
  int base = 0, who, block;
  if (p.n_req <= 32) {
    const int from = max(q.ctx - q.len, 0) / span, to = from + q.mine;  // levels of the request: its blocks, counted from position 0
    auto at_or_above = [&](int level) { return (int)__reduce_add_sync(0xffffffffu, (unsigned)max(0, to - max(level, from))); };
    int level = 0, above = (int)__reduce_max_sync(0xffffffffu, (unsigned)to);
    while (above - level > 1) {  // the highest level with more than `back` blocks at or above it
      const int mid = (level + above) >> 1;
      if (at_or_above(mid) > back) level = mid;
      else above = mid;
    }
    const bool has = from <= level && level < to;
    const int nth = back - at_or_above(level + 1);
    const uint32_t mask = __ballot_sync(0xffffffffu, has);
    who = max(0, __ffs(__ballot_sync(0xffffffffu, has && __popc(mask & ((1u << lane) - 1u)) == nth)) - 1);
    block = level - __shfl_sync(0xffffffffu, from, who);
  } else {
    const int blk = n_items / a.head_tiles - 1 - back;
    for (int run = 0;; base += 32, q = pp_lane(a, span, base + lane)) {
      const uint32_t hit = __ballot_sync(0xffffffffu, run + q.upto > blk);
      if (hit != 0) {
        who = __ffs(hit) - 1;
        block = blk - run - __shfl_sync(0xffffffffu, q.upto - q.mine, who);
        break;
      }
      run += __shfl_sync(0xffffffffu, q.upto, 31);
    }
  }
  const int len = __shfl_sync(0xffffffffu, q.len, who);
  w->req = base + who;
  w->begin = __shfl_sync(0xffffffffu, q.begin, who);
  w->q0 = block * span;
  w->n_here = min(span, len - w->q0);
  w->pos0 = __shfl_sync(0xffffffffu, q.ctx, who) - len + w->q0;
  w->held = (int)min((int64_t)w->pos0 + w->n_here, (int64_t)p.table_width * p.cache.block_size);
  w->key_end = w->held;
  w->lo_first = p.window > 0 ? max(0, max(w->pos0, 0) - (p.window - 1)) : 0;
  w->sink_end = max(0, min(min(p.sinks, w->lo_first), w->key_end));
  // (a window behind the table's end has no box; its first one is at the end, since a key next to 2^31 and its tile need not fit an int)
  w->first_box = min(w->lo_first, max(w->held, 0) + a.box - 1) >> a.box_shift;
  w->sink_boxes = min((w->sink_end + a.box - 1) >> a.box_shift, w->first_box);
  w->i0 = 0;
  const int boxes = w->key_end <= 0 ? 0 : w->sink_boxes + max(0, ((w->key_end + a.box - 1) >> a.box_shift) - w->first_box);
  w->i1 = (boxes + (kPpKeys >> a.box_shift) - 1) / (kPpKeys >> a.box_shift);
  w->parts = 1;
}

// The part of an item that CTA c leaves for the join (slot c): numerators [row / 128][column / 4][row % 128] of four columns, then
// maximum and sum of every row.
template <int D>
__host__ __device__ constexpr int pp_slot_floats(int tiles) { return tiles * kPpRows * (D + 2); }
// Of the item whose parts the CTAs c, c + stride, ... (`parts` of them) hold; parts < 2: none
struct PpJoin { int head0, token0, n_here, parts, stride, pad[3]; };

template <int D, bool kF16, int kTiles, bool kSplit>
__global__ void __launch_bounds__(pp_threads(kTiles), 3 - kTiles) paged_prefill_kernel(const __grid_constant__ PpMaps maps, const __grid_constant__ PpArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr int kSt = pp_stages<D>(kTiles), kTile = pp_tile<D>(), kPanels = D / 64;
  // Where the columns allow it P has its own, and S of the next tile is made while this one's softmax runs; the softmax is then all
  // there is to wait for, and an eighth of the exponentials on the FMA units pays. (8192 tokens, 16 / 2 heads of 64: 208 us with P in
  // S, 198 with columns of its own, 190 with an eighth, 197 with a quarter, 233 with half; heads of 128 gain from neither.)
  constexpr bool kOwnP = kTiles == 1 && D == 64;
  constexpr int kLoader = 4 * kTiles, kIssuer = kLoader + 1, kTmem = 256 * kTiles, kO = kTiles * kPpKeys;  // warps; columns: all, the first of O
  enum { Q_FULL, Q_FREE, S_READY, P_READY = S_READY + 2, O_DONE = P_READY + 4, K_FULL = O_DONE + 2, K_FREE = K_FULL + kSt, V_FULL = K_FREE + kSt,
         V_FREE = V_FULL + kSt, PIECE = V_FREE + kSt, TAKEN = PIECE + 2, S_TAKEN = TAKEN + 2, PV_DONE, N_BARS };
  __shared__ __align__(8) uint64_t bars[N_BARS];
  __shared__ uint32_t s_tmem, s_boxes[4];
  __shared__ PpPiece s_piece[2];
  __shared__ volatile int abort_flag;
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const PagedArgs& p = a.p;
  // (V first: what a wrong stride of its descriptor could reach stays inside the allocation)
  const uint32_t raw = smem_u32(smem_raw), v_u32 = (raw + 1023u) & ~1023u, k_u32 = v_u32 + kSt * kTile, q_u32 = k_u32 + kSt * kTile, out_u32 = q_u32 + kTiles * kTile;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };

  if (tid == 0) {
    for (int i = 0; i < N_BARS; ++i) mbar_init(bar(i), (i >= P_READY && i < O_DONE) || i == S_TAKEN ? kPpRows : i == TAKEN || i == TAKEN + 1 ? 4 * kTiles + 1 : 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kIssuer) tmem_alloc(smem_u32(&s_tmem), kTmem);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  glue_enter();  // (dependents may start: every CTA of this launch holds its tensor memory by then)
  const uint32_t tmem = s_tmem;
  const int per_tile = kPpRows >> a.h_shift, span = kTiles * per_tile;

  // Pieces come from the loading warp through two places in shared memory.
  auto take = [&](int k, PpPiece* w) {
    pp_wait(bar(PIECE + (k & 1)), (uint32_t)(k >> 1) & 1, &abort_flag);
    *w = s_piece[k & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(TAKEN + (k & 1)));
    return w->parts > 0 && abort_flag == 0;
  };
  if (warp < kLoader) {  // ------------------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPpSoftmaxRegs));
    const int t = warp >> 2, row = (warp & 3) * 32 + lane, tok = t * per_tile + (row >> a.h_shift);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + t * kPpKeys + lanes, o_at = tmem + kO + t * D + lanes, p_at = kOwnP ? tmem + kO + D + lanes : s_at;
    const uint32_t all_boxes = bits_below(kPpKeys / a.box);
    const int tile_shift = 7 - a.box_shift, step = min(a.box, 32);  // boxes of a tile, as a logarithm; columns of 32 that lie in one box
    const uint32_t stage = out_u32 + warp * (32 * kPpOutPitch);  // 32 columns of the warp's rows on their way out
    uint32_t n = 0, pieces = 0;  // tiles and pieces with tiles so far: phases of the barriers
    PpPiece w;
    for (int k = 0; take(k, &w); ++k) {
      const int pos = pp_position(w.pos0, tok);
      const int lo = p.window > 0 ? max(pos, 0) - (p.window - 1) : 0;
      const int tile_lo = pp_position(w.pos0, t * per_tile), tile_hi = pp_position(tile_lo, per_tile - 1);  // positions of the tile
      // tiles [clear0, clear1) need no mask: behind the first tokens, from where every row's window has begun, up to the first row
      const int w_lo = p.window > 0 ? max(tile_hi, 0) - (p.window - 1) : 0;
      const int clear0 = (w.sink_boxes + max(0, (int)(((uint32_t)max(w_lo, 0) + a.box - 1u) >> a.box_shift) - w.first_box) + (1 << tile_shift) - 1) >> tile_shift;
      const int clear1 = (((tile_lo + 1) >> a.box_shift) + w.sink_boxes - w.first_box) >> tile_shift;
      float m = -INFINITY, l = 0.f;  // what the probabilities refer to, in units of log2; their sum
      for (int i = w.i0; i < w.i1; ++i, ++n) {
        pp_wait(bar(S_READY + t), n & 1, &abort_flag);
        tc_fence_after_sync();
        uint32_t s[4][32];
#pragma unroll
        for (int c = 0; c < 2; ++c) tmem_ld_32x32(s_at + 32 * c, s[c]);
        const uint32_t boxes = s_boxes[n & 3];
        const bool masked = i < clear0 || i >= clear1 || boxes != all_boxes;
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
              uint32_t seen = 0;
#pragma unroll 1
              for (int g = 0; g < 32; g += step) {
                const int col = 32 * c + g, b = col >> a.box_shift, at = w.key_of(i, b, a.box_shift) + (col & (a.box - 1));
                const uint32_t bits = bits_below(pos + 1 - at) & (~bits_below(lo - at) | bits_below(p.sinks - at));
                if ((boxes >> b) & 1u) seen |= (bits & bits_below(step)) << g;
              }
              asm volatile("" : "+r"(seen));  // (one word at a time: 128 tests at once cost 350 bytes of spills)
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!((seen >> j) & 1u)) s[c][j] = 0xff800000u;  // -inf
            }
#pragma unroll
            for (int j = 0; j < 32; j += 2) top4[j / 2 % 4] = max3(top4[j / 2 % 4], __uint_as_float(s[c][j]), __uint_as_float(s[c][j + 1]));
          }
        }
        if (kOwnP) {
          tc_fence_before_sync();
          mbar_arrive(bar(S_TAKEN));
        }
        const float mx = max3(max3(top4[0], top4[1], top4[2]), top4[3], top4[3]);
        const float top = mx * p.sc;
        const bool grows = !(top <= m + (kProbSlack + kProbUp<kF16>));  // (a NaN among the scores makes the maximum and with it the whole row NaN)
        if (kOwnP && n > 0) {  // P and O of the tile before are done with
          pp_wait(bar(PV_DONE), (n - 1) & 1, &abort_flag);
          tc_fence_after_sync();
        }
        if (__any_sync(0xffffffffu, grows)) {
          const float up = top - kProbUp<kF16>, f = grows ? ex2(m - up) : 1.f;
          if (grows) m = up;
          l *= f;
          if (i > w.i0) {  // (if P lies in S: S of this tile came behind P V of the one before, O is complete)
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
            const float2 y = kOwnP && j % 16 == 14 ? exp2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
            sum[j / 2 % 2] = add2(sum[j / 2 % 2], y);
            packed[j / 2] = pack_16x2<kF16>(y.x, y.y);  // (rounded to the type of V; the sum is that of the unrounded ones)
          }
          tmem_st_32x16(p_at + 16 * c, packed);
          if (c & 1) {  // half of P: its products may begin
            tmem_st_wait();
            tc_fence_before_sync();
            mbar_arrive(bar(P_READY + 2 * t + (c >> 1)));
          }
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      const bool live = tok < w.n_here, any = w.i1 > w.i0, whole = !kSplit || w.parts == 1;
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (no visible key: zeros; NaN stays)
      const int64_t token0 = (int64_t)w.begin + w.q0;
      if (any) {
        if (kOwnP) pp_wait(bar(PV_DONE), (n - 1) & 1, &abort_flag);
        else pp_wait(bar(O_DONE + t), pieces & 1, &abort_flag);
        ++pieces;
        tc_fence_after_sync();
      }
      if (whole) {
        // Through shared memory, so that four lanes write 64 adjacent bytes of a row. (A row's pieces straight from its thread: 32
        // half-used sectors a store, 3200 cycles for a tile of 128 columns.)
        char* dst[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int of = (warp & 3) * 32 + 8 * r + (lane >> 2), its = t * per_tile + (of >> a.h_shift);
          dst[r] = its < w.n_here ? static_cast<char*>(p.out) + 2 * ((token0 + its) * p.out_token + (w.head0 + (of & ((1 << a.h_shift) - 1))) * p.out_head) + 16 * (lane & 3) : nullptr;
        }
        uint32_t all[D / 32][32];
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          if (any) {
            tmem_ld_32x32(o_at + 32 * c, all[c]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) all[c][j] = 0;
          }
        }
        tmem_ld_wait();
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          const uint32_t(&o)[32] = all[c];
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            uint4 v;
            v.x = pack_16x2<kF16>(__uint_as_float(o[j]) * inv, __uint_as_float(o[j + 1]) * inv);
            v.y = pack_16x2<kF16>(__uint_as_float(o[j + 2]) * inv, __uint_as_float(o[j + 3]) * inv);
            v.z = pack_16x2<kF16>(__uint_as_float(o[j + 4]) * inv, __uint_as_float(o[j + 5]) * inv);
            v.w = pack_16x2<kF16>(__uint_as_float(o[j + 6]) * inv, __uint_as_float(o[j + 7]) * inv);
            sts128(stage + lane * kPpOutPitch + 2 * j, v);
          }
          __syncwarp();
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (dst[r] != nullptr) stg128(dst[r] + 64 * c, lds128(stage + (8 * r + (lane >> 2)) * kPpOutPitch + 16 * (lane & 3)));
          __syncwarp();
        }
        if (live && p.lse != nullptr) p.lse[(token0 + tok) * p.Hq + w.head0 + (row & ((1 << a.h_shift) - 1))] = l == 0.f ? -INFINITY : (m + log2f(l)) * 0.6931471805599453f;
      } else {
        float* const part = a.parts + (int64_t)blockIdx.x * pp_slot_floats<D>(kTiles);
        float4* const at = reinterpret_cast<float4*>(part) + t * (D / 4) * kPpRows + row;
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld_32x32(o_at + 32 * c, o);
          tmem_ld_wait();
          if (live) {
#pragma unroll
            for (int j = 0; j < 32; j += 4) stg128(at + (8 * c + j / 4) * kPpRows, make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]));
          }
        }
        if (live) reinterpret_cast<float2*>(part + kTiles * kPpRows * D)[t * kPpRows + row] = make_float2(m, l);
      }
      tc_fence_before_sync();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(pp_other_regs(kTiles)));
    if (warp == kLoader) {  // ------------------------------------------------------------------ loads
      const uint32_t leader = elect_one();
      const int n_boxes = kPpKeys / a.box;
      uint32_t n = 0, pieces = 0;
      const PpLane lanes0 = pp_lane(a, span, lane);
      const int n_items = pp_items(a, span, lanes0), G = gridDim.x, waves = n_items / G, rest = n_items - waves * G;
      // Split: the items that do not fill a wave are cut into parts, CTA i + s * rest has part s of item i.
      const int most = kSplit && rest > 0 ? G / rest : 1;
      if (kSplit && leader) static_cast<PpJoin*>(a.joins)[blockIdx.x].parts = 0;
      PpPiece w;
      bool more_pieces = true;
      for (int k = 0; more_pieces; ++k) {
        w.parts = 0;
        // (every other wave backwards: contexts get shorter from item to item)
        const int c = k & 1 ? G - 1 - (int)blockIdx.x : (int)blockIdx.x;
        if (k < waves) {
          pp_find(a, span, k * G + c, n_items, lanes0, &w);
        } else if (k == waves && most >= 2) {
          const int i = blockIdx.x % rest, s = blockIdx.x / rest;
          if (s < most) {
            pp_find(a, span, k * G + i, n_items, lanes0, &w);
            const int tiles = w.i1;
            w.parts = max(1, min(min(most, kPpParts), tiles / kPpShare));
            if (s >= w.parts) w.parts = 0;
            if (w.parts > 1) {
              w.i0 = (int)((int64_t)tiles * s / w.parts);
              w.i1 = (int)((int64_t)tiles * (s + 1) / w.parts);
              if (s == 0 && leader) static_cast<PpJoin*>(a.joins)[i] = {w.head0, w.begin + w.q0, w.n_here, w.parts, rest, {0, 0, 0}};
            }
          }
        } else if (k == waves && c < rest) {
          pp_find(a, span, k * G + c, n_items, lanes0, &w);
        }
        more_pieces = w.parts > 0;
        if (k >= 2) pp_wait(bar(TAKEN + (k & 1)), (uint32_t)((k >> 1) - 1) & 1, &abort_flag);
        if (abort_flag != 0) { w.parts = 0; more_pieces = false; }
        if (leader) {
          s_piece[k & 1] = w;
          mbar_arrive(bar(PIECE + (k & 1)));
        }
        if (!more_pieces || w.i1 <= w.i0) continue;
        const int kvh = w.head0 / (p.Hq / p.Hk);
        const int32_t* table = p.tables + w.req * p.table_ld;
        for (int i = w.i0; i < w.i1; ++i, ++n) {
          const int st = n % kSt, key = w.key_of(i, lane, a.box_shift);
          int block = -1, in_block = 0;
          if (lane < n_boxes && key < w.held) {
            const int page = key / p.cache.block_size;
            block = table[page];
            in_block = key - page * p.cache.block_size;
          }
          if (i == w.i0) {
            if (pieces > 0) pp_wait(bar(Q_FREE), (pieces - 1) & 1, &abort_flag);
            ++pieces;
            if (leader) {
              mbar_arrive_expect_tx(bar(Q_FULL), kTiles * kTile);
              for (int t = 0; t < kTiles; ++t)
                for (int c = 0; c < kPanels; ++c)
                  tma_load_3d_at(q_u32 + t * kTile + c * kPpPanel, &maps.q, 64 * c, w.head0, w.begin + w.q0 + t * per_tile, bar(Q_FULL));
            }
          }
          const bool there = (unsigned)block < (unsigned)p.cache.num_blocks;
          if (!there) { block = p.cache.num_blocks; in_block = 0; }  // outside the map: zeros
          const uint32_t boxes = __ballot_sync(0xffffffffu, there);
          for (int which = 0; which < 2; ++which) {
            const uint32_t full = bar((which ? V_FULL : K_FULL) + st);
            if (n >= kSt) pp_wait(bar((which ? V_FREE : K_FREE) + st), (n / kSt - 1) & 1, &abort_flag);
            if (leader) {
              if (which == 0) s_boxes[n & 3] = boxes;  // (read up to kSt tiles later: fewer than four)
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
      uint32_t n = 0, pieces = 0;
      PpPiece w;
      for (int k = 0; take(k, &w); ++k) {
        if (w.i1 <= w.i0) continue;
        pp_wait(bar(Q_FULL), pieces & 1, &abort_flag);
        ++pieces;
        pp_wait(bar(K_FULL + n % kSt), (n / kSt) & 1, &abort_flag);
        if (kOwnP && n > 0) {
          pp_wait(bar(S_TAKEN), (n - 1) & 1, &abort_flag);
          tc_fence_after_sync();
        }
        for (int t = 0; t < kTiles; ++t) scores(t, n % kSt);
        umma_commit_elected(bar(K_FREE + n % kSt), leader);
        if (w.i1 == w.i0 + 1) umma_commit_elected(bar(Q_FREE), leader);
        for (int i = w.i0; i < w.i1; ++i, ++n) {
          const int st = n % kSt, next = (n + 1) % kSt;
          const bool more = i + 1 < w.i1;
          if (kOwnP && more) {
            pp_wait(bar(K_FULL + next), ((n + 1) / kSt) & 1, &abort_flag);
            pp_wait(bar(S_TAKEN), n & 1, &abort_flag);
            tc_fence_after_sync();
            scores(0, next);
            umma_commit_elected(bar(K_FREE + next), leader);
            if (i + 2 == w.i1) umma_commit_elected(bar(Q_FREE), leader);
          }
          pp_wait(bar(V_FULL + st), (n / kSt) & 1, &abort_flag);
          // Rows of V that no token of this CTA sees may hold anything (a block's stale rows): they become zero, as 0 * V must.
          const int first_key = w.key_of(i, 0, a.box_shift), last_key = w.key_of(i, (kPpKeys >> a.box_shift) - 1, a.box_shift) + a.box - 1;
          if (!(last_key < w.sink_end || (first_key >= w.lo_first && last_key < w.key_end))) {
            for (int x = lane; x < kPpKeys * kPanels * 8; x += 32) {
              const int row = x / (kPanels * 8), key = w.key_of(i, row >> a.box_shift, a.box_shift) + (row & (a.box - 1)), c = x % (kPanels * 8);
              if (!(key < w.sink_end || (key >= w.lo_first && key < w.key_end)))
                sts128(v_u32 + st * kTile + (c >> 3) * kPpPanel + row * 128 + (c & 7) * 16, make_uint4(0, 0, 0, 0));
            }
            fence_proxy_async_smem();
            __syncwarp();
          }
          for (int t = 0; t < kTiles; ++t) {
#pragma unroll
            for (int k = 0; k < kPpKeys / 16; ++k) {
              if (k % 4 == 0) {
                pp_wait(bar(P_READY + 2 * t + k / 4), n & 1, &abort_flag);
                tc_fence_after_sync();
              }
              umma_ts_elected(tmem + kO + t * D, tmem + (kOwnP ? kO + D : t * kPpKeys) + 8 * k, lo_v(v_u32 + st * kTile + k * 2048), hi_k, idesc_o,
                              i > w.i0 || k > 0, leader);
            }
            if (kOwnP) {
              umma_commit_elected(bar(PV_DONE), leader);
            } else if (more) {
              // (behind P V of this tile in the same thread: P has been read when S is written over it)
              if (t == 0) pp_wait(bar(K_FULL + next), ((n + 1) / kSt) & 1, &abort_flag);
              scores(t, next);
            } else {
              umma_commit_elected(bar(O_DONE + t), leader);
            }
          }
          umma_commit_elected(bar(V_FREE + st), leader);
          if (!kOwnP && more) umma_commit_elected(bar(K_FREE + next), leader);
          if (!kOwnP && i + 2 == w.i1) umma_commit_elected(bar(Q_FREE), leader);
        }
      }
      // the last commits must have arrived before this CTA's shared memory is given up
      if (n > 0) {
        pp_wait(bar(V_FREE + (n - 1) % kSt), ((n - 1) / kSt) & 1, &abort_flag);
        pp_wait(bar(Q_FREE), (pieces - 1) & 1, &abort_flag);
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

// Joins the parts of the item that CTA blockIdx.x has the first part of. A thread per row of the item, 16 columns (blockIdx.y): eight
// parts' worth of them are under way at a time.
template <int D, bool kF16, int kTiles>
__global__ void __launch_bounds__(kTiles * kPpRows) paged_prefill_join_kernel(const __grid_constant__ PpArgs a) {
  glue_enter();
  const PpJoin j = static_cast<const PpJoin*>(a.joins)[blockIdx.x];
  if (j.parts < 2) return;
  const PagedArgs& p = a.p;
  const int t = threadIdx.x / kPpRows, row = threadIdx.x % kPpRows, tok = t * (kPpRows >> a.h_shift) + (row >> a.h_shift);
  if (tok >= j.n_here) return;
  const int head = j.head0 + (row & ((1 << a.h_shift) - 1)), c0 = 4 * blockIdx.y;
  const float* const first = a.parts + (int64_t)blockIdx.x * pp_slot_floats<D>(kTiles);
  const int64_t step = (int64_t)j.stride * pp_slot_floats<D>(kTiles);
  auto stats = [&](int k) { return reinterpret_cast<const float2*>(first + k * step + kTiles * kPpRows * D)[t * kPpRows + row]; };
  float top = -INFINITY, sum = 0.f;
#pragma unroll 8
  for (int k = 0; k < j.parts; ++k) top = fmaxf(top, stats(k).x);
  float4 o[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int k = 0; k < j.parts; ++k) {
    const float2 ml = stats(k);
    const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);  // (a row of NaN has NaN for its maximum)
    sum += f * ml.y;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float4 v = reinterpret_cast<const float4*>(first + k * step)[(t * (D / 4) + c0 + c) * kPpRows + row];
      o[c] = make_float4(o[c].x + f * v.x, o[c].y + f * v.y, o[c].z + f * v.z, o[c].w + f * v.w);
    }
  }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  const int64_t token = (int64_t)j.token0 + tok;
  char* const dst = static_cast<char*>(p.out) + 2 * (token * p.out_token + head * p.out_head + 4 * c0);
#pragma unroll
  for (int c = 0; c < 4; c += 2) {
    uint4 v;
    v.x = pack_16x2<kF16>(o[c].x * inv, o[c].y * inv);
    v.y = pack_16x2<kF16>(o[c].z * inv, o[c].w * inv);
    v.z = pack_16x2<kF16>(o[c + 1].x * inv, o[c + 1].y * inv);
    v.w = pack_16x2<kF16>(o[c + 1].z * inv, o[c + 1].w * inv);
    stg128(dst + 8 * c, v);
  }
  if (c0 == 0 && p.lse != nullptr) p.lse[token * p.Hq + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
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
  return (Hk == 1 || head > 0) && (c.block_size == 1 || token > 0) && (c.num_blocks == 1 || block > 0) && pp_map(out, v ? c.v : c.k, f16, 4, dims, strides, b);
}

// Heads of a tile, as a power of two: they divide a group
inline int pp_h_shift(int group) {
  int s = 0;
  while (s < 4 && group % (2 << s) == 0) ++s;
  return s;
}

// Whether the tensor-core kernel takes a call: copies of 8 cache rows or more that lie in one block, a table of which every key has an
// int, and strides that its maps take (not 0, as of heads that are expanded from one).
inline bool paged_prefill_plan(const PagedArgs& p, int D, bool f16, int tiles, PpMaps* maps, PpArgs* a) {
  if (p.cache.block_size % 8 != 0 || (int64_t)p.table_width * p.cache.block_size > kPpMaxKeys) return false;
  a->p = p;
  a->box = 8;
  // Short boxes where first tokens stay visible: they share a tile with the window's begin (8001 tokens, window of 1024 and 4 first
  // ones: 95 -> 89 us; without first ones whole tiles have the faster masks: window of 512 62 us, in short boxes 66).
  while (a->box < (p.sinks > 0 ? kPpSinkBox : kPpKeys) && p.cache.block_size % (2 * a->box) == 0) a->box *= 2;
  a->box_shift = 0;
  while ((1 << a->box_shift) < a->box) ++a->box_shift;
  a->h_shift = pp_h_shift(p.Hq / p.Hk);
  a->head_tiles = p.Hq >> a->h_shift;
  const int per_tile = kPpRows >> a->h_shift;
  const int64_t blocks = (int64_t)p.T / (tiles * per_tile) + p.n_req;
  if (blocks * a->head_tiles > INT32_MAX) return false;
  a->n_blocks = (int)blocks;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)p.Hq, (cuuint64_t)p.T};
  const cuuint64_t strides[2] = {(cuuint64_t)(p.Hq == 1 ? D : p.q_head) * 2, (cuuint64_t)(p.T == 1 ? (int64_t)p.Hq * D : p.q_token) * 2};
  const cuuint32_t box[3] = {64, 1u << a->h_shift, (cuuint32_t)per_tile};
  return (p.Hq == 1 || p.q_head > 0) && (p.T == 1 || p.q_token > 0) && pp_map(&maps->q, p.q, f16, 3, dims, strides, box) &&
         pp_cache_map(&maps->k, p.cache, false, p.Hk, D, a->box, f16, &a->k_heads_inner) &&
         pp_cache_map(&maps->v, p.cache, true, p.Hk, D, a->box, f16, &a->v_heads_inner);
}

// Whether a launch cuts the items that do not fill a wave of CTAs into parts, as told by what the host knows: items at most, and
// tiles of an item at most.
inline bool pp_splits(int T, int n_req, int Hq, int h_shift, int tiles, int64_t max_context, int window) {
  const int span = tiles * (kPpRows >> h_shift);
  const int64_t items = ((int64_t)T / span + n_req) * (Hq >> h_shift);
  const int64_t keys = window > 0 ? std::min<int64_t>(max_context, (int64_t)window + span) : max_context;
  const int wave = 148 * (3 - tiles);
  return keys / kPpKeys >= kPpSplitTiles && (2 * items <= wave || (items <= kPpSplitWaves * wave && keys >= 2 * (int64_t)T));
}
constexpr int pp_tiles(int D) { return D == 64 ? 1 : 2; }
inline size_t pp_split_bytes(int D) {
  const int tiles = pp_tiles(D), ctas = 148 * (3 - tiles);
  return (size_t)ctas * tiles * kPpRows * (D + 2) * 4 + ctas * sizeof(PpJoin);
}
// (blocks that the tile kernel does not take: what the decode kernel needs for as many rows)
inline size_t paged_prefill_workspace_bytes(int T, int n_req, int Hq, int Hk, int D, int block_size, int64_t max_context, int window) {
  if (block_size % 8 != 0) return paged_workspace_bytes(T, Hq, Hk, D, max_context, window, 0);
  return pp_splits(T, n_req, Hq, pp_h_shift(Hq / Hk), pp_tiles(D), max_context, window) ? pp_split_bytes(D) : 0;
}

template <int D, bool kF16, bool kSplit>
inline int paged_prefill_launch_t(const PpMaps& maps, const PpArgs& a, cudaStream_t stream) {
  constexpr int kTiles = pp_tiles(D), kCtas = 148 * (3 - kTiles);
  const auto kernel = paged_prefill_kernel<D, kF16, kTiles, kSplit>;
  constexpr int smem = pp_smem<D>(kTiles);
  static std::atomic<uint64_t> known{0};
  if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), smem, &known)) return rc;
  const int ctas = kSplit ? kCtas : (int)std::min<int64_t>(kCtas, (int64_t)a.n_blocks * a.head_tiles);
  const int rc = launch_dependent(kernel, "paged_prefill_kernel", dim3((unsigned)ctas), pp_threads(kTiles), (size_t)smem, stream, maps, a);
  if (rc != B200_LORA_OK || !kSplit) return rc;
  return launch_dependent(paged_prefill_join_kernel<D, kF16, kTiles>, "paged_prefill_join_kernel", dim3((unsigned)ctas, D / 16), kTiles * kPpRows, 0, stream, a);
}

inline int paged_prefill_launch(const PagedArgs& p, int D, int dtype, void* workspace, cudaStream_t stream) {
  PpMaps maps;
  PpArgs a = {};
  const bool f16 = dtype == B200_LORA_F16;
  if (!paged_prefill_plan(p, D, f16, pp_tiles(D), &maps, &a)) return paged_decode_launch(p, D, dtype, p.cache.block_size % 8 != 0 ? workspace : nullptr, stream);
  if (pp_splits(p.T, p.n_req, p.Hq, a.h_shift, pp_tiles(D), (int64_t)p.table_width * p.cache.block_size, p.window)) {
    a.parts = static_cast<float*>(workspace);
    a.joins = static_cast<char*>(workspace) + pp_split_bytes(D) - 148 * (3 - pp_tiles(D)) * sizeof(PpJoin);
    if (D == 64) return f16 ? paged_prefill_launch_t<64, true, true>(maps, a, stream) : paged_prefill_launch_t<64, false, true>(maps, a, stream);
    return f16 ? paged_prefill_launch_t<128, true, true>(maps, a, stream) : paged_prefill_launch_t<128, false, true>(maps, a, stream);
  }
  if (D == 64) return f16 ? paged_prefill_launch_t<64, true, false>(maps, a, stream) : paged_prefill_launch_t<64, false, false>(maps, a, stream);
  return f16 ? paged_prefill_launch_t<128, true, false>(maps, a, stream) : paged_prefill_launch_t<128, false, false>(maps, a, stream);
}

}  // namespace b200lora
