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
//
// Two more forms of it. Differential heads: the tiles of a CTA are the two maps of the same rows, which share K and V; a map's scores take
// half of the columns, its O all of those of V, and the warpgroups trade sums, then take the difference and the norm of half of the columns
// each. 2048 tokens behind 8192, 32 / 8 heads of 128, 675 us = 0.69 PFLOP/s (1.14 with the second terms of the probabilities): the
// products, at the clock that the power cap leaves; 12 prompts of 100 to 1200, 16 / 2 of 64, 69 us: twice the exponentials of one map (37 us).
// Prefixes that requests share: the rows of all requests of a group side by side, cut along the keys so that the parts fill the GPU; a part
// leaves its sums as they are, for the launch over the keys behind the prefix (paged_attention.cuh). 96 requests behind four prefixes of
// 3000 to 9000 keys, 32 / 8 of 128: 30 us of 100, a tile of keys in 4000 cycles (two CTAs an SM): S and P V in turn with a softmax of
// 2000 and the look-ups and loads of the next tile.
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
// Tiles of a CTA, and how many of them have rows of their own: the two maps of differential heads are two tiles of the same rows.
static_assert(kPpKeys == kPrefixTile, "parts of a prefix are whole tiles");
// (The rows over a prefix seldom fill two, and one leaves an SM room for a CTA of the launch over the keys behind it.)
__host__ __device__ constexpr int pp_tiles(int D, int form) { return (D == 128 && form == kPlain) || form == kDiff ? 2 : 1; }
__host__ __device__ constexpr int pp_row_tiles(int D, int form) { return form == kDiff ? 1 : pp_tiles(D, form); }
template <int D>
__host__ __device__ constexpr int pp_smem(int tiles, int row_tiles) { return (2 * pp_stages<D>(tiles) + row_tiles) * pp_tile<D>() + tiles * kPpRows * kPpOutPitch + 1024; }

// Items that do not fill a wave of CTAs may be cut into parts along the keys, joined by a second launch: us, whole / cut, 16 / 2 heads,
// 16 tokens behind 8192 keys (heads of 128) 112 / 29, behind 65536 844 / 56, 500 behind 3000 (64) 42 / 25; 32 / 8 of 128, 4096 behind
// 12288 (3.5 waves of items of even length) 905 / 868. Not where every item is short, nor whole prompts of more than half a
// wave: their last items are their shortest (8192 tokens 223 / 239).
constexpr int kPpSplitTiles = 8;     // tiles of an item, at least
constexpr int kPpSplitWaves = 6;     // waves of CTAs at most
constexpr int kPxChunk = 2;          // tiles of a part of a prefix, at least
constexpr int kPpShare = 2, kPpParts = 32;  // tiles of a part at least, parts at most (the join reads them one after another)

struct PpMaps { CUtensorMap q, k, v; };
struct PpArgs {
  PagedArgs p;
  int h_shift, head_tiles;   // heads of a tile = 1 << h_shift; tiles over all heads
  int n_blocks;              // blocks of tokens that the launch has CTAs for
  int box, box_shift;        // cache rows of a copy: 8 .. 128, a power of two that divides the block size; its logarithm
  float* parts; void* joins;  // split: partial results and what there is to join
  int px_ctas;               // CTAs that the parts of prefixes are to fill
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
  int part, r1, keys;                          // of a prefix: which part of it, the request behind the group's, its keys
  // first key of box b of tile i, with 1 << shift keys in a box
  __device__ __forceinline__ int key_of(int i, int b, int shift) const {
    const int c = i * (kPpKeys >> shift) + b;
    return (c < sink_boxes ? c : c - sink_boxes + first_box) << shift;
  }
};

// Of the requests [r0, r1), the one that begins at or before the row last
__device__ __forceinline__ int px_request(const PagedArgs& p, int row, int r0, int r1) {
  while (r1 - r0 > 1) {
    const int mid = (r0 + r1) >> 1;
    if (p.cu_seqlens[mid] <= row) r0 = mid;
    else r1 = mid;
  }
  return r0;
}
// Position of a row of the group that begins with request r0; -1 if its request's rows leave those of q
__device__ __forceinline__ int px_position(const PagedArgs& p, int row, int r0, int r1) {
  if (p.cu_seqlens == nullptr) return max(p.context_lens[row], 0) - 1;  // (less than none is none, the least int too)
  const int r = px_request(p, row, r0, r1), end = p.cu_seqlens[r + 1];
  if (p.cu_seqlens[r] < 0 || end > p.T || row >= end) return -1;
  return (int)max((int64_t)p.context_lens[r] - (end - row), (int64_t)-1);
}

// The order of the rows by their keys behind the prefix, most first, by one CTA; `keys`: room for one of each in shared memory
__device__ __forceinline__ void px_order(const PagedArgs& p, int* keys) {
  const int n = p.T <= kPxOrder ? p.T : 0;
  for (int row = threadIdx.x; row < n; row += blockDim.x) {
    const int r = p.cu_seqlens == nullptr ? row : px_request(p, row, 0, p.n_req);
    int lo = 0, hi = p.n_groups;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (p.cu_groups[mid] <= r) lo = mid;
      else hi = mid;
    }
    const PxGroup g = px_group(p, lo);
    const int ctx = p.context_lens[r];
    keys[row] = max(0, max(ctx, 0) - (g.r0 <= r && r < g.r1 ? g.keys : 0));
  }
  __syncthreads();
  for (int row = threadIdx.x; row < n; row += blockDim.x) {
    const int mine = keys[row];
    int rank = 0;
#pragma unroll 8
    for (int k = 0; k < n; ++k) rank += keys[k] > mine || (keys[k] == mine && k < row) ? 1 : 0;
    p.px_head->order[rank] = row;
  }
  __syncthreads();
  if (threadIdx.x == 0) st_release_gpu(&p.px_head->next_item, 0);  // (with the order, and with what this CTA has waited for)
  __syncthreads();
}

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

// Of a prefix launch: tiles of a part, so that the parts of all prefixes are as many as the CTAs that the launch is to fill, or more; items
// over all groups (a block of rows, a set of heads, a part). 32 groups, one a lane, at a time.
struct PxLane { PxGroup g; int blocks, tiles; };
__device__ __forceinline__ PxLane px_lane(const PpArgs& a, int span, int g) {
  PxLane q;
  q.g = px_group(a.p, g);
  q.tiles = (int)(((unsigned)q.g.keys + kPpKeys - 1u) / kPpKeys);
  q.blocks = q.tiles == 0 ? 0 : (q.g.end - q.g.begin + span - 1) / span;
  return q;
}
// A part of `chunk` tiles each: one wave of CTAs where that is possible, since ceil(t / c) <= t / c + 1, so that with R items of one part
// each and W tiles over them W / c + R <= CTAs; then the least c near it that still fits.
__device__ __forceinline__ int px_chunk_tiles(const PpArgs& a, int span, const PxLane& lanes0) {
  constexpr unsigned kMost = 1u << 25;  // (of a lane's 32: what more there may be changes nothing in the outcome that matters)
  unsigned work = 0, rows = 0, longest = 0;
  for (int base = 0; base < a.p.n_groups; base += 32) {
    const PxLane q = base == 0 ? lanes0 : px_lane(a, span, base + (int)(threadIdx.x & 31));
    const unsigned mine = (unsigned)q.blocks * (unsigned)a.head_tiles;  // (fits: the host's items do)
    rows = min(kMost, rows + min(kMost, mine));
    work = min(kMost, work + (unsigned)min((unsigned long long)kMost, (unsigned long long)mine * (unsigned)q.tiles));
    longest = max(longest, (unsigned)q.tiles);
  }
  work = __reduce_add_sync(0xffffffffu, work);
  rows = __reduce_add_sync(0xffffffffu, rows);
  longest = __reduce_max_sync(0xffffffffu, longest);
  const unsigned once = (unsigned)a.px_ctas / 2;  // (a CTA an SM leaves room beside it; two where that is long, too)
  const unsigned one = work > 8u * once ? (unsigned)a.px_ctas : once;
  const unsigned ctas = one * max(1u, (2 * rows + one - 1) / one);  // (as many waves as leave half of the places to cuts)
  const unsigned least = max((unsigned)kPxChunk, (longest + a.p.px_most - 1) / a.p.px_most), room = max(1u, ctas - rows);
  unsigned chunk = max(1u, (work + room - 1) / room);
  if (a.p.n_groups <= 32) {
    const unsigned mine = (unsigned)lanes0.blocks * (unsigned)a.head_tiles;
    for (int k = 0; k < 4 && chunk > least; ++k) {
      const unsigned parts = ((unsigned)lanes0.tiles + chunk - 2) / (chunk - 1);
      if (__reduce_add_sync(0xffffffffu, (unsigned)min((unsigned long long)kMost, (unsigned long long)mine * parts)) > ctas) break;
      --chunk;
    }
  }
  return (int)max(chunk, least);
}
// Items of a group, at most INT32_MAX over all (the host sees to that for groups that do not overlap)
__device__ __forceinline__ int px_items_of(const PpArgs& a, const PxLane& q, int chunk) {
  return (int)min((long long)q.blocks * a.head_tiles * ((q.tiles + chunk - 1) / chunk), (long long)(INT32_MAX >> 6));
}
// Item `item` of the launch, or parts = 0
__device__ __forceinline__ void px_find(const PpArgs& a, int span, int chunk, int item, const PxLane& lanes0, PpPiece* w) {
  const PagedArgs& p = a.p;
  const int lane = threadIdx.x & 31;
  w->parts = 0;
  for (int base = 0; base < p.n_groups; base += 32) {
    const PxLane q = base == 0 ? lanes0 : px_lane(a, span, base + lane);
    const int mine = px_items_of(a, q, chunk), upto = warp_upto(mine);
    const uint32_t hit = __ballot_sync(0xffffffffu, upto > item);
    if (hit == 0) {
      item -= __shfl_sync(0xffffffffu, upto, 31);
      continue;
    }
    const int who = __ffs(hit) - 1;
    const int at = item - __shfl_sync(0xffffffffu, upto - mine, who), blocks = __shfl_sync(0xffffffffu, q.blocks, who);
    const int r0 = __shfl_sync(0xffffffffu, q.g.r0, who), r1 = __shfl_sync(0xffffffffu, q.g.r1, who);
    const int begin = __shfl_sync(0xffffffffu, q.g.begin, who), end = __shfl_sync(0xffffffffu, q.g.end, who);
    w->keys = __shfl_sync(0xffffffffu, q.g.keys, who);
    // (the blocks of rows over one part and set of heads side by side: they read the same keys)
    const int block = at % blocks, rest = at / blocks, set = rest % a.head_tiles;
    w->part = rest / a.head_tiles;
    w->head0 = set << a.h_shift;
    w->req = r0;
    w->r1 = r1;
    w->begin = begin;
    w->q0 = block * span;
    w->n_here = min(span, end - begin - w->q0);
    // No key behind the contexts of the block's requests: rows there may hold anything.
    int first = begin + w->q0, last = first + w->n_here - 1, most = 0;  // requests of the block
    if (p.cu_seqlens != nullptr) {
      first = px_request(p, first, r0, r1);
      last = px_request(p, last, r0, r1);
    }
    for (int r = first + lane; r <= last; r += 32) most = max(most, p.context_lens[r]);
    most = __reduce_max_sync(0xffffffffu, most);
    w->pos0 = 0;
    w->held = w->key_end = min(w->keys, most);
    w->lo_first = w->sink_end = w->first_box = w->sink_boxes = 0;
    w->i0 = w->part * chunk;
    w->i1 = min(w->i0 + chunk, (w->key_end + kPpKeys - 1) / kPpKeys);
    w->parts = 1;
    return;
  }
}

// The part of an item that CTA c leaves for the join (slot c): numerators [row / 128][column / 4][row % 128] of four columns, then
// maximum and sum of every row.
template <int D>
__host__ __device__ constexpr int pp_slot_floats(int tiles) { return tiles * kPpRows * (D + 2); }
// Of the item whose parts the CTAs c, c + stride, ... (`parts` of them) hold; parts < 2: none
struct PpJoin { int head0, token0, n_here, parts, stride, pad[3]; };

// kForm kDiff: the tiles are the two maps of the same rows, over the same K and V: scores take half of the columns each, a warpgroup
// ends with half of the columns of both maps' O.
template <int D, bool kF16, bool kSplit, int kForm>
__global__ void __launch_bounds__(pp_threads(pp_tiles(D, kForm)), 3 - pp_tiles(D, kForm)) paged_prefill_kernel(const __grid_constant__ PpMaps maps, const __grid_constant__ PpArgs a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  constexpr int kTiles = pp_tiles(D, kForm), kRowTiles = pp_row_tiles(D, kForm), kSt = pp_stages<D>(kTiles), kTile = pp_tile<D>(), kPanels = D / 64;
  // Where the columns allow it P has its own, and S of the next tile is made while this one's softmax runs; the softmax is then all
  // there is to wait for, and an eighth of the exponentials on the FMA units pays. (8192 tokens, 16 / 2 heads of 64: 208 us with P in
  // S, 198 with columns of its own, 190 with an eighth, 197 with a quarter, 233 with half; heads of 128 gain from neither.)
  constexpr bool kOwnP = kTiles == 1 && D == 64;
  // Differential: probabilities are two 16-bit numbers each in the product with V (bf16: both truncated, 2^-15 of a probability at most),
  // since what the maps have in common leaves with the difference and what rounding did to it stays. Scores of spread 1, lam of 0.5,
  // against 64 bits where the rounding of the result alone has 1: one number 1.55, second terms for half of the keys 1.31, for all 1.
  // 2048 tokens behind 8192, 32 / 8 heads of 128, 474, 580, 662 us (P V is what bounds it); 12 prompts of 101 to 1200, 16 / 2 heads of
  // 64, 66, 67, 69. (For half of them a key would count with the more bits the earlier it lies in its tile, and with other ones than a decode
  // step gives it.)
  constexpr bool kFine = kForm == kDiff;
  constexpr int kLoader = 4 * kTiles, kIssuer = kLoader + 1, kTmem = 256 * kTiles, kO = kTiles * kPpKeys;  // warps; columns: all, the first of O
  enum { Q_FULL, Q_FREE, S_READY, P_READY = S_READY + 2, O_DONE = P_READY + 4, K_FULL = O_DONE + 2, K_FREE = K_FULL + kSt, V_FULL = K_FREE + kSt,
         V_FREE = V_FULL + kSt, PIECE = V_FREE + kSt, TAKEN = PIECE + 2, S_TAKEN = TAKEN + 2, PV_DONE, SHARED, N_BARS };
  __shared__ __align__(8) uint64_t bars[N_BARS];
  __shared__ uint32_t s_tmem, s_boxes[4];
  __shared__ PpPiece s_piece[2];
  __shared__ volatile int abort_flag;
  __shared__ __align__(16) float s_weight[kForm == kDiff ? D : 4];   // of the norm
  __shared__ float s_sums[kForm == kDiff ? 2 : 1][kTiles][kPpRows];  // what the maps tell each other: sums, sums of squares
  const int tid = threadIdx.x, warp = uniform(tid >> 5), lane = tid & 31;
  const PagedArgs& p = a.p;
  // (V first: what a wrong stride of its descriptor could reach stays inside the allocation)
  const uint32_t raw = smem_u32(smem_raw), v_u32 = (raw + 1023u) & ~1023u, k_u32 = v_u32 + kSt * kTile, q_u32 = k_u32 + kSt * kTile, out_u32 = q_u32 + kRowTiles * kTile;
  auto bar = [&](int i) { return smem_u32(&bars[i]); };

  if (kForm == kPrefix) {
    // The launch behind this one may start once all CTAs have let it (it has no use for tensor memory). CTA 0 has no part of a
    // prefix; it leaves the counter that the other's items come from, and their order.
    griddep_wait();
    if (blockIdx.x == 0) {
      px_order(p, reinterpret_cast<int*>(smem_raw));
      griddep_launch_dependents();
      return;
    }
    griddep_launch_dependents();
  }
  if (tid == 0) {
    for (int i = 0; i < N_BARS; ++i) mbar_init(bar(i), (i >= P_READY && i < O_DONE) || i == S_TAKEN ? kPpRows : i == SHARED ? 2 * kPpRows : i == TAKEN || i == TAKEN + 1 ? 4 * kTiles + 1 : 1);
    abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == kIssuer) tmem_alloc(smem_u32(&s_tmem), kTmem);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  if (kForm != kPrefix) glue_enter();  // (dependents may start: every CTA of this launch holds its tensor memory by then)
  if (kForm == kDiff) {
    for (int i = tid; i < D; i += pp_threads(kTiles)) {
      float w = 1.f;
      if (p.norm_weight != nullptr) {
        const float2 pair = unpack_16x2<kF16>(reinterpret_cast<const uint32_t*>(p.norm_weight)[i >> 1]);
        w = i & 1 ? pair.y : pair.x;
      }
      s_weight[i] = w;
    }
    __syncthreads();
  }
  const uint32_t tmem = s_tmem;
  const int per_tile = kPpRows >> a.h_shift, span = kRowTiles * per_tile;

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
    const int t = warp >> 2, row = (warp & 3) * 32 + lane, tok0 = (kForm == kDiff ? 0 : t) * per_tile, tok = tok0 + (row >> a.h_shift);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_at = tmem + t * kPpKeys + lanes, o_at = tmem + kO + t * D + lanes, p_at = kOwnP ? tmem + kO + D + lanes : s_at;
    const uint32_t all_boxes = bits_below(kPpKeys / a.box);
    const int tile_shift = 7 - a.box_shift, step = min(a.box, 32);  // boxes of a tile, as a logarithm; columns of 32 that lie in one box
    const uint32_t stage = out_u32 + warp * (32 * kPpOutPitch);  // 32 columns of the warp's rows on their way out
    uint32_t n = 0, pieces = 0, exchanges = 0;  // tiles and pieces with tiles so far: phases of the barriers
    PpPiece w;
    for (int k = 0; take(k, &w); ++k) {
      int pos = pp_position(w.pos0, tok);
      const int lo = p.window > 0 ? max(pos, 0) - (p.window - 1) : 0;
      int tile_lo = pp_position(w.pos0, tok0);
      if (kForm == kPrefix) {  // (rows have positions of their own, most of them behind the prefix; the first key that some row of the warp does not see)
        pos = tok < w.n_here && w.i1 > w.i0 ? min(px_position(p, w.begin + w.q0 + tok, w.req, w.r1), w.keys - 1) : w.keys - 1;
        tile_lo = __reduce_min_sync(0xffffffffu, pos);
      }
      const int tile_hi = pp_position(tile_lo, per_tile - 1);  // positions of the tile
      // tiles [clear0, clear1) need no mask: behind the first tokens, from where every row's window has begun, up to the first row
      const int w_lo = p.window > 0 ? max(tile_hi, 0) - (p.window - 1) : 0;
      const int clear0 = (w.sink_boxes + max(0, (int)(((uint32_t)max(w_lo, 0) + a.box - 1u) >> a.box_shift) - w.first_box) + (1 << tile_shift) - 1) >> tile_shift;
      const int clear1 = (((tile_lo + 1) >> a.box_shift) + w.sink_boxes - w.first_box) >> tile_shift;
      float lam = 0.f;  // (asked for ahead of the tiles)
      if (kForm == kDiff && tok < w.n_here)
        lam = p.lam[((int64_t)w.begin + w.q0 + tok) * p.lam_token + (w.head0 + (row & ((1 << a.h_shift) - 1))) * p.lam_head];
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
          uint32_t packed[16], rest[16];
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float2 x = fma2(make_float2(__uint_as_float(s[c][j]), __uint_as_float(s[c][j + 1])), scale2, base2);
            const float2 y = kOwnP && j % 16 == 14 ? exp2_poly(x) : make_float2(ex2(x.x), ex2(x.y));
            sum[j / 2 % 2] = add2(sum[j / 2 % 2], y);
            if (kFine && !kF16) {  // (the upper halves as they are, and what they leave)
              packed[j / 2] = __byte_perm(__float_as_uint(y.x), __float_as_uint(y.y), 0x7632);
              const float2 low = fma2(make_float2(__uint_as_float(__float_as_uint(y.x) & 0xffff0000u), __uint_as_float(__float_as_uint(y.y) & 0xffff0000u)), make_float2(-1.f, -1.f), y);
              rest[j / 2] = __byte_perm(__float_as_uint(low.x), __float_as_uint(low.y), 0x7632);
            } else {
              packed[j / 2] = pack_16x2<kF16>(y.x, y.y);  // (rounded to the type of V; the sum is that of the unrounded ones)
              if (kFine) rest[j / 2] = rest_16x2<kF16>(y, packed[j / 2]);
            }
          }
          tmem_st_32x16(p_at + 16 * c, packed);
          if (kFine) tmem_st_32x16(p_at + kPpKeys / 2 + 16 * c, rest);
          if (c & 1) {  // half of P: its products may begin
            tmem_st_wait();
            tc_fence_before_sync();
            mbar_arrive(bar(P_READY + 2 * t + (c >> 1)));
          }
        }
        l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      }
      const bool live = tok < w.n_here, any = w.i1 > w.i0, whole = kForm != kPrefix && (!kSplit || w.parts == 1);
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);  // (no visible key: zeros; NaN stays)
      const int64_t token0 = (int64_t)w.begin + w.q0;
      if (any) {
        if (kOwnP) pp_wait(bar(PV_DONE), (n - 1) & 1, &abort_flag);
        else pp_wait(bar(O_DONE + t), pieces & 1, &abort_flag);
        if (kForm == kDiff && whole) pp_wait(bar(O_DONE + (t ^ 1)), pieces & 1, &abort_flag);
        ++pieces;
        tc_fence_after_sync();
      }
      auto whose = [&](int r) { return (warp & 3) * 32 + 8 * r + (lane >> 2); };  // row that the lane stores in round r
      auto stored = [&](int r, int col) {  // its columns from `col` on in out, null: not there
        const int of = whose(r), its = tok0 + (of >> a.h_shift);
        return its < w.n_here ? static_cast<char*>(p.out) + 2 * ((token0 + its) * p.out_token + (w.head0 + (of & ((1 << a.h_shift) - 1))) * p.out_head + col) + 16 * (lane & 3) : nullptr;
      };
      if (kForm == kDiff && whole) {
        // Half of the columns of both maps: their sums go through shared memory, then the sums of squares of the halves. Behind the
        // second exchange every thread has its columns of O, which the next piece may then overwrite.
        auto exchange = [&](int which, float v) {
          s_sums[which][t][row] = v;
          tc_fence_before_sync();
          mbar_arrive(bar(SHARED));
          pp_wait(bar(SHARED), exchanges & 1, &abort_flag);
          ++exchanges;
          tc_fence_after_sync();
          return s_sums[which][t ^ 1][row];
        };
        const float other = over(exchange(0, l));
        const float one = t == 0 ? inv : other, two = lam * (t == 0 ? other : inv);
        float y[D / 2], ss = 0.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          uint32_t o1[32], o2[32];
          const uint32_t at = tmem + kO + t * (D / 2) + 32 * c + lanes;
          if (any) {
            tmem_ld_32x32(at, o1);
            tmem_ld_32x32(at + D, o2);
            tmem_ld_wait();
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) {  // (both products rounded: equal maps cancel)
            y[32 * c + j] = any ? __fmul_rn(__uint_as_float(o1[j]), one) - __fmul_rn(__uint_as_float(o2[j]), two) : 0.f;
            ss += y[32 * c + j] * y[32 * c + j];
          }
        }
        ss += exchange(1, ss);
        const float r = p.norm_weight != nullptr ? rsqrtf(ss * (1.f / D) + p.eps) : 1.f;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
          const int col = t * (D / 2) + 32 * c;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
              const float4 w4 = *reinterpret_cast<const float4*>(s_weight + col + j + i);
              f[i] = r * w4.x;
              f[i + 1] = r * w4.y;
              f[i + 2] = r * w4.z;
              f[i + 3] = r * w4.w;
            }
            const float* const x = y + 32 * c + j;
            uint4 v;
            v.x = pack_16x2<kF16>(x[0] * f[0], x[1] * f[1]);
            v.y = pack_16x2<kF16>(x[2] * f[2], x[3] * f[3]);
            v.z = pack_16x2<kF16>(x[4] * f[4], x[5] * f[5]);
            v.w = pack_16x2<kF16>(x[6] * f[6], x[7] * f[7]);
            sts128(stage + lane * kPpOutPitch + 2 * j, v);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            char* const dst = stored(i, col);
            if (dst != nullptr) stg128(dst, lds128(stage + (8 * i + (lane >> 2)) * kPpOutPitch + 16 * (lane & 3)));
          }
          __syncwarp();
        }
      } else if (kForm == kPrefix) {
        // The part's sums as they are, through shared memory for the same reason as below, 16 columns of fp32 at a time.
        const int64_t part_at = ((int64_t)w.part * p.T + token0) * p.Hq;
#pragma unroll
        for (int c = 0; any && c < D / 16; ++c) {
          uint32_t o[16];
          tmem_ld_32x16(o_at + 16 * c, o);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 16; j += 4) sts128(stage + lane * kPpOutPitch + 4 * j, make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]));
          __syncwarp();
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int of = whose(r), its = tok0 + (of >> a.h_shift);
            if (its < w.n_here)
              stg128(p.px_o + (part_at + (int64_t)its * p.Hq + w.head0 + (of & ((1 << a.h_shift) - 1))) * D + 16 * c + 4 * (lane & 3),
                     lds128(stage + (8 * r + (lane >> 2)) * kPpOutPitch + 16 * (lane & 3)));
          }
          __syncwarp();
        }
        if (live) p.px_ml[part_at + (int64_t)tok * p.Hq + w.head0 + (row & ((1 << a.h_shift) - 1))] = make_float2(m, l);
      } else if (whole) {
        // Through shared memory, so that four lanes write 64 adjacent bytes of a row. (A row's pieces straight from its thread: 32
        // half-used sectors a store, 3200 cycles for a tile of 128 columns.)
        char* dst[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) dst[r] = stored(r, 0);
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
      const int G = (int)gridDim.x - (kForm == kPrefix ? 1 : 0);
      PpLane lanes0 = {0, 0, 0, 0, 0};
      PxLane groups0 = {{0, 0, 0, 0, 0}, 0, 0};
      int n_items = 0, chunk = 1;
      if constexpr (kForm == kPrefix) {
        groups0 = px_lane(a, span, lane);
        chunk = px_chunk_tiles(a, span, groups0);
        if (blockIdx.x == 1 && leader) p.px_head->chunk = chunk;
      } else {
        lanes0 = pp_lane(a, span, lane);
        n_items = pp_items(a, span, lanes0);
      }
      const int waves = n_items / G, rest = n_items - waves * G;
      // Split: the items that do not fill a wave are cut into parts, CTA i + s * rest has part s of item i.
      const int most = kSplit && rest > 0 ? G / rest : 1;
      if (kSplit && leader) static_cast<PpJoin*>(a.joins)[blockIdx.x].parts = 0;
      PpPiece w;
      bool more_pieces = true;
      for (int k = 0; more_pieces; ++k) {
        w.parts = 0;
        // (every other wave backwards: contexts get shorter from item to item)
        const int c = k & 1 ? G - 1 - (int)blockIdx.x : (int)blockIdx.x;
        if constexpr (kForm == kPrefix) {
          px_find(a, span, chunk, k * G + (int)blockIdx.x - 1, groups0, &w);
        } else if (k < waves) {
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
              mbar_arrive_expect_tx(bar(Q_FULL), kRowTiles * kTile);
              for (int t = 0; t < kRowTiles; ++t)
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
        constexpr int kSteps = D / 16 / kMaps<kForm>;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int k = (kForm == kDiff ? t * kSteps : 0) + i;
          const uint32_t at = (k >> 2) * kPpPanel + (k & 3) * 32;
          umma_elected(tmem + t * kPpKeys, lo_k(q_u32 + (kForm == kDiff ? 0 : t * kTile) + at), lo_k(k_u32 + st * kTile + at), hi_k, idesc_s, i > 0, leader);
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
              if (kFine)
                umma_ts_elected(tmem + kO + t * D, tmem + t * kPpKeys + kPpKeys / 2 + 8 * k, lo_v(v_u32 + st * kTile + k * 2048), hi_k, idesc_o, 1, leader);
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
  const int64_t token = (int64_t)j.token0 + tok;
  const float inv = over(sum);
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

// The same for differential heads: 32 rows of the item (blockIdx.y), a warp per 16 columns, of both maps (the tiles of a part); the sums
// of squares of a row meet in shared memory.
template <int D, bool kF16>
__global__ void __launch_bounds__(2 * D) paged_prefill_join_maps_kernel(const __grid_constant__ PpArgs a) {
  __shared__ float s_squares[D / 16][32];
  glue_enter();
  const PpJoin j = static_cast<const PpJoin*>(a.joins)[blockIdx.x];
  if (j.parts < 2) return;
  const PagedArgs& p = a.p;
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5, row = 32 * blockIdx.y + lane, tok = row >> a.h_shift, c0 = 4 * group;
  const bool live = tok < j.n_here;
  const int head = j.head0 + (row & ((1 << a.h_shift) - 1));
  const int64_t token = (int64_t)j.token0 + tok;
  const float* const first = a.parts + (int64_t)blockIdx.x * pp_slot_floats<D>(2);
  const int64_t step = (int64_t)j.stride * pp_slot_floats<D>(2);
  float y[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) y[i] = 0.f;
  for (int map = 0; live && map < 2; ++map) {
    auto stats = [&](int k) { return reinterpret_cast<const float2*>(first + k * step + 2 * kPpRows * D)[map * kPpRows + row]; };
    float top = -INFINITY, sum = 0.f;
#pragma unroll 8
    for (int k = 0; k < j.parts; ++k) top = fmaxf(top, stats(k).x);
    float4 o[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < j.parts; ++k) {
      const float2 ml = stats(k);
      const float f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
      sum += f * ml.y;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 v = reinterpret_cast<const float4*>(first + k * step)[(map * (D / 4) + c0 + c) * kPpRows + row];
        o[c] = make_float4(o[c].x + f * v.x, o[c].y + f * v.y, o[c].z + f * v.z, o[c].w + f * v.w);
      }
    }
    const float f = map == 0 ? over(sum) : p.lam[token * p.lam_token + head * p.lam_head] * over(sum);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float x[4] = {o[c].x, o[c].y, o[c].z, o[c].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) y[4 * c + i] = map == 0 ? __fmul_rn(x[i], f) : y[4 * c + i] - __fmul_rn(x[i], f);
    }
  }
  if (p.norm_weight != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) ss += y[i] * y[i];
    s_squares[group][lane] = ss;
    __syncthreads();
    ss = 0.f;
#pragma unroll
    for (int g = 0; g < D / 16; ++g) ss += s_squares[g][lane];
    const float r = rsqrtf(ss * (1.f / D) + p.eps);
#pragma unroll
    for (int i = 0; i < 16; i += 2) {
      const float2 w = unpack_16x2<kF16>(*reinterpret_cast<const uint32_t*>(static_cast<const char*>(p.norm_weight) + 2 * (4 * c0 + i)));
      y[i] *= r * w.x;
      y[i + 1] *= r * w.y;
    }
  }
  if (!live) return;
  char* const dst = static_cast<char*>(p.out) + 2 * (token * p.out_token + head * p.out_head + 4 * c0);
#pragma unroll
  for (int i = 0; i < 16; i += 8)
    stg128(dst + 2 * i, make_uint4(pack_16x2<kF16>(y[i], y[i + 1]), pack_16x2<kF16>(y[i + 2], y[i + 3]), pack_16x2<kF16>(y[i + 4], y[i + 5]),
                                   pack_16x2<kF16>(y[i + 6], y[i + 7])));
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
inline bool paged_prefill_plan(const PagedArgs& p, int D, bool f16, int row_tiles, PpMaps* maps, PpArgs* a) {
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
  const int64_t blocks = (int64_t)p.T / (row_tiles * per_tile) + p.n_req;
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
inline bool pp_splits(int T, int n_req, int Hq, int h_shift, int row_tiles, int ctas, int64_t max_context, int window) {
  const int span = row_tiles * (kPpRows >> h_shift);
  const int64_t items = ((int64_t)T / span + n_req) * (Hq >> h_shift);
  const int64_t keys = window > 0 ? std::min<int64_t>(max_context, (int64_t)window + span) : max_context;
  return keys / kPpKeys >= kPpSplitTiles && (2 * items <= ctas || (items <= kPpSplitWaves * ctas && keys >= 2 * (int64_t)T));
}
constexpr int pp_ctas(int D, int form) { return 148 * (3 - pp_tiles(D, form)); }
inline size_t pp_split_bytes(int D, int form) {
  return (size_t)pp_ctas(D, form) * pp_tiles(D, form) * kPpRows * (D + 2) * 4 + pp_ctas(D, form) * sizeof(PpJoin);
}
// (blocks that the tile kernel does not take: what the decode kernel needs for as many rows)
template <int kForm = kPlain>
inline size_t paged_prefill_workspace_bytes(int T, int n_req, int Hq, int Hk, int D, int block_size, int64_t max_context, int window) {
  if (block_size % 8 != 0) return paged_workspace_bytes<kForm>(T, Hq, Hk, D, max_context, window, 0);
  return pp_splits(T, n_req, Hq, pp_h_shift(Hq / Hk), pp_row_tiles(D, kForm), pp_ctas(D, kForm), max_context, window) ? pp_split_bytes(D, kForm) : 0;
}

template <int D, bool kF16, bool kSplit, int kForm>
inline int paged_prefill_launch_t(const PpMaps& maps, const PpArgs& a, cudaStream_t stream) {
  constexpr int kTiles = pp_tiles(D, kForm), kCtas = pp_ctas(D, kForm);
  const auto kernel = paged_prefill_kernel<D, kF16, kSplit, kForm>;
  constexpr int smem = pp_smem<D>(kTiles, pp_row_tiles(D, kForm));
  static std::atomic<uint64_t> known{0};
  if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), smem, &known, kForm == kPrefix)) return rc;
  const int ctas = kForm == kPrefix ? a.px_ctas + 1 : kSplit ? kCtas : (int)std::min<int64_t>(kCtas, (int64_t)a.n_blocks * a.head_tiles);
  const int rc = launch_dependent(kernel, "paged_prefill_kernel", dim3((unsigned)ctas), pp_threads(kTiles), (size_t)smem, stream, maps, a);
  if (rc != B200_LORA_OK || !kSplit) return rc;
  if constexpr (kForm == kDiff)
    return launch_dependent(paged_prefill_join_maps_kernel<D, kF16>, "paged_prefill_join_maps_kernel", dim3((unsigned)ctas, kPpRows / 32), 2 * D, 0, stream, a);
  else
    return launch_dependent(paged_prefill_join_kernel<D, kF16, kTiles>, "paged_prefill_join_kernel", dim3((unsigned)ctas, D / 16), kTiles * kPpRows, 0, stream, a);
}

template <int kForm = kPlain>
inline int paged_prefill_launch(const PagedArgs& p, int D, int dtype, void* workspace, cudaStream_t stream) {
  PpMaps maps;
  PpArgs a = {};
  const bool f16 = dtype == B200_LORA_F16;
  if (!paged_prefill_plan(p, D, f16, pp_row_tiles(D, kForm), &maps, &a))
    return paged_decode_launch<kForm>(p, D, dtype, p.cache.block_size % 8 != 0 ? workspace : nullptr, stream);
  if (pp_splits(p.T, p.n_req, p.Hq, a.h_shift, pp_row_tiles(D, kForm), pp_ctas(D, kForm), (int64_t)p.table_width * p.cache.block_size, p.window)) {
    a.parts = static_cast<float*>(workspace);
    a.joins = static_cast<char*>(workspace) + pp_split_bytes(D, kForm) - pp_ctas(D, kForm) * sizeof(PpJoin);
    if (D == 64) return f16 ? paged_prefill_launch_t<64, true, true, kForm>(maps, a, stream) : paged_prefill_launch_t<64, false, true, kForm>(maps, a, stream);
    return f16 ? paged_prefill_launch_t<128, true, true, kForm>(maps, a, stream) : paged_prefill_launch_t<128, false, true, kForm>(maps, a, stream);
  }
  if (D == 64) return f16 ? paged_prefill_launch_t<64, true, false, kForm>(maps, a, stream) : paged_prefill_launch_t<64, false, false, kForm>(maps, a, stream);
  return f16 ? paged_prefill_launch_t<128, true, false, kForm>(maps, a, stream) : paged_prefill_launch_t<128, false, false, kForm>(maps, a, stream);
}

// Requests with common prefixes: a launch over the prefixes, the requests of a group side by side, and one over the keys behind them, a row
// at a time, that joins. Host code; what the device makes of the lengths is at px_chunk_tiles.
struct PxPlan { int most, ctas; size_t ml_bytes, o_bytes; };  // parts of a prefix at most; CTAs that they are to fill; bytes of workspace
inline PxPlan px_plan(int T, int Hq, int Hk, int D) {
  PxPlan x;
  const int h_shift = pp_h_shift(Hq / Hk), span = kPpRows >> h_shift;
  x.ctas = pp_ctas(D, kPrefix);
  const int64_t blocks = (int64_t)ceil_div_i(T, span) * (Hq >> h_shift);
  x.most = (int)std::max<int64_t>(1, std::min<int64_t>(kPpParts, (2 * x.ctas + blocks - 1) / blocks));
  const size_t sums = (size_t)x.most * T * Hq;
  x.ml_bytes = (sums * 8 + 15) / 16 * 16;
  x.o_bytes = sums * D * 4;
  return x;
}
// Whether requests are attended by group, as told by what the host knows: where a group has more than one, copies of the cache's rows take
// tiles of them, and the keys that the tables hold at most are worth a second launch.
// Decode: 100 MB of keys and values a call, each request's its own. us, request by request / by group, prefixes with 100 keys behind them:
//   16 / 2 heads of 64: 16 requests of 8000 (67 MB) 15.5 / 20.7, 64 of 1500 (55 MB) 11.6 / 14.9, of 3000 (105 MB) 17.7 / 16.4, 192 of 1500
//   33.6 / 20.9; 8 / 8 of 64: 16 of 3000 (105 MB) 17.8 / 15.8, 64 of 300 (59 MB) 13.1 / 18.6, of 1500 32 / 19.5; 32 / 8 of 128: 4 of 8000
//   (134 MB) 23.9 / 24.6, 16 of 1500 (109 MB) 17.7 / 16.3, of 3000 29.5 / 17.6; 16 / 2 of 128: 64 of 700 (59 MB) 12.0 / 16.9, of 3000 30 / 19.2
//   On the wrong side of that line: many keys behind the prefixes (the host knows their sum alone: 16 requests, 32 / 8 of 128, of 3000 behind 1000
//   45 / 83, 48 of them 112 / 139), and groups of one to three requests (96 of 2100, 16 / 2 of 64, in 95, 48, 32, 24 and 8 groups 22 / 43,
//   28, 26, 23, 19; 32 / 8 of 128 144 to 99 / 173, 113, 80, 68, 50).
// Packed: tiles of rows over the whole contexts against those over the prefix and an item for every new token and kv head, by formulas
// that tell which is less rather than how much (at 4 of 120 points the slower way, by more than 15 %). us, 32 requests with 2, 6, 12, 24 new
// tokens behind 4000 keys: 16 / 2 heads of 64 25, 25, 26, 39 / 17, 27, 33, 53; 32 / 8 of 128 123, 123, 125, 127 / 32, 55, 88, 165
inline bool px_shares(int T, int n_req, int n_groups, int Hq, int Hk, int D, int block_size, int64_t max_keys, bool packed) {
  if (n_groups < 1 || n_req <= n_groups || block_size % 8 != 0 || max_keys < 1 || max_keys > kPpMaxKeys || T >= (1 << 24)) return false;
  if (!packed) return (double)T * max_keys * Hk * D * 4 >= 100e6;
  const int h_shift = pp_h_shift(Hq / Hk), per_tile = kPpRows >> h_shift, sets = Hq >> h_shift;
  const double tiles = (double)max_keys / kPpKeys, each = ceil_div_i(ceil_div_i(T, n_req), per_tile * pp_row_tiles(D, kPlain));
  const double alone = 8 + n_req * each * sets * tiles * 1.8 / pp_ctas(D, kPlain);
  const double items = (double)T * Hk * ceil_div_i(Hq / Hk, kItemHeads<kSuffix>), blocks = ceil_div_i(T, per_tile) + n_groups - 1;
  return 12 + 4.5 * items / kPagedCtas + blocks * sets * tiles * 1.2 / pp_ctas(D, kPrefix) < alone;
}
inline size_t shared_prefix_workspace_bytes(int T, int n_req, int n_groups, int Hq, int Hk, int D, int block_size, int64_t max_keys, bool packed) {
  // (a call whose strides a map refuses goes without sharing)
  const size_t plain = packed ? paged_prefill_workspace_bytes(T, n_req, Hq, Hk, D, block_size, max_keys, 0) : paged_workspace_bytes(T, Hq, Hk, D, max_keys, 0, 0);
  if (!px_shares(T, n_req, n_groups, Hq, Hk, D, block_size, max_keys, packed)) return plain;
  const PxPlan x = px_plan(T, Hq, Hk, D);
  return std::max(plain, sizeof(PxHead) + x.ml_bytes + x.o_bytes);
}

template <int D, bool kF16>
inline int shared_prefix_launch_t(PagedArgs p, bool packed, void* workspace, cudaStream_t stream) {
  const int dtype = kF16 ? B200_LORA_F16 : B200_LORA_BF16;
  PpMaps maps;
  PpArgs a = {};
  if (!px_shares(p.T, p.n_req, p.n_groups, p.Hq, p.Hk, D, p.cache.block_size, (int64_t)p.table_width * p.cache.block_size, packed) ||
      !paged_prefill_plan(p, D, kF16, pp_row_tiles(D, kPrefix), &maps, &a))
    return packed ? paged_prefill_launch(p, D, dtype, workspace, stream) : paged_decode_launch(p, D, dtype, workspace, stream);
  const PxPlan x = px_plan(p.T, p.Hq, p.Hk, D);
  char* const parts = static_cast<char*>(workspace) + sizeof(PxHead);
  p.px_most = x.most;
  p.px_head = static_cast<PxHead*>(workspace);
  p.px_ml = reinterpret_cast<float2*>(parts);
  p.px_o = reinterpret_cast<float*>(parts + x.ml_bytes);
  a.p = p;
  a.px_ctas = x.ctas;
  const int rc = paged_prefill_launch_t<D, kF16, false, kPrefix>(maps, a, stream);
  return rc != B200_LORA_OK ? rc : paged_decode_launch<kSuffix>(p, D, dtype, nullptr, stream);
}
inline int shared_prefix_launch(const PagedArgs& p, int D, int dtype, bool packed, void* workspace, cudaStream_t stream) {
  const bool f16 = dtype == B200_LORA_F16;
  if (D == 64) return f16 ? shared_prefix_launch_t<64, true>(p, packed, workspace, stream) : shared_prefix_launch_t<64, false>(p, packed, workspace, stream);
  return f16 ? shared_prefix_launch_t<128, true>(p, packed, workspace, stream) : shared_prefix_launch_t<128, false>(p, packed, workspace, stream);
}

}  // namespace b200lora
