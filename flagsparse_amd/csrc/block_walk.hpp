// block_walk.hpp — a workgroup's walk over the blocks that its queries select: the
// kernels of many queries, forward and gradient of the queries
// (block_attention.hip, block_attention_grad.hip).
//
// A workgroup takes consecutive tokens of a sequence, all heads of one group, 16
// rows a wave.  Tokens near each other select many of the same
// blocks: a table in LDS holds, for each block of a window of the sequence, a bit
// for each token that selects it.  The blocks with a bit are walked in order, keys
// and values loaded once for the workgroup, and a wave takes part with the tiles
// that have a token of the block.
#pragma once

#include "block_tile.hpp"

namespace fs {
namespace {

constexpr int kMaskWords = 2048;

template <int WAVES>
struct WalkMemory {
  uint32_t mask[kMaskWords];
  uint16_t list[kMaskWords];
  uint32_t total[WAVES];
};

// What a workgroup works on.
struct WalkTile {
  Sequence sq;
  int seq, head;
  int token0, tokens;  // of all tokens; how many
  int pos0;            // position of the first
  int per;             // tokens a full tile
};

template <int WAVES>
__host__ __device__ inline int tokens_of(int group) { return WAVES * 16 / group; }

// Head by head over the XCDs (each has its keys and values in a cache of its own), a
// head's last tiles first: they have the most blocks to choose from.
template <int WAVES>
__device__ inline bool walk_tile(const BlockArgs& p, int lane, WalkTile& t) {
  const int64_t at = xcd_range_block(blockIdx.x, gridDim.x);
  t.head = (int)(at / p.tiles);
  t.per = tokens_of<WAVES>(p.group);
  int tile;
  if (!find_tile(p.seqs, t.per, p.tiles - 1 - at % p.tiles, lane, t.seq, tile)) return false;
  t.sq = sequence_of(p.seqs, t.seq);
  const int first = tile * t.per;
  t.token0 = t.sq.first + first;
  t.tokens = t.sq.count - first < t.per ? t.sq.count - first : t.per;
  t.pos0 = t.sq.keys - t.sq.count + first;
  return true;
}

// A lane's row.
__device__ inline RowOf row_of(const BlockArgs& p, const WalkTile& t, int w, int lane) {
  RowOf o;
  const int r = w * 16 + (lane & 15);
  o.token = r / p.group;
  o.head = r - o.token * p.group;
  o.in = o.token < t.tokens;
  if (!o.in) o.token = 0;
  o.pos = o.in ? t.pos0 + o.token : -1;
  return o;
}

// A lane's selection in a step has a bit for each half.
template <class T, int DP, int WAVES, class Body>
__device__ inline void walk_blocks(const BlockArgs& p, const WalkTile& t, const RowOf& row,
                                   WalkMemory<WAVES>& mem, uint8_t (&kv)[2][2][Rows<T, DP>::kBytes], int tid, int w,
                                   int lane, Body body) {
  using R = Rows<T, DP>;
  constexpr int THREADS = 64 * WAVES, kHalf = R::kKeys / 2;
  const int lg_block = p.lg_groups + 4;
  const int lg_halves = lg_block - (kHalf == 32 ? 5 : 4);  // of a block's halves of a step
  const int words = (t.per + 31) / 32, window = kMaskWords / words;
  const int last = t.pos0 + t.tokens - 1;
  const int n_blocks = last < 0 ? 0 : (last >> lg_block) + 1;
  const int entries = t.tokens * p.top;
  const int32_t* ids = p.blocks + (int64_t)t.token0 * p.b_token + (int64_t)t.head * p.b_head;
  KeySource<T, DP, WAVES> src;
  src.init(p, t.sq, t.seq, t.head, w, lane);
  const uint32_t kv0 = lds_address(kv);

  for (int w0 = 0; w0 < n_blocks; w0 += window) {
    __syncthreads();
    const int here = n_blocks - w0 < window ? n_blocks - w0 : window;
    for (int i = tid; i < here * words; i += THREADS) mem.mask[i] = 0u;
    __syncthreads();
    for (int e = tid; e < entries; e += THREADS) {
      const int tok = e / p.top;
      const int64_t id = ids[(int64_t)tok * p.b_token + (e - tok * p.top)];
      // (a block behind the token's own has none of its keys)
      if (id >= w0 && id < w0 + here && id <= ((t.pos0 + tok) >> lg_block))
        atomicOr(&mem.mask[((int)id - w0) * words + (tok >> 5)], 1u << (tok & 31));
    }
    __syncthreads();
    // the blocks with a bit, in order
    const int each = (here + THREADS - 1) / THREADS;
    auto named = [&](int b) {
      uint32_t any = 0;
      if (b < here)
        for (int k = 0; k < words; ++k) any |= mem.mask[b * words + k];
      return any != 0;
    };
    uint32_t mine = 0;
    for (int i = 0; i < each; ++i) mine += named(tid * each + i);
    const uint32_t upto = wave_sum_scan(mine);
    if (lane == 63) mem.total[w] = upto;
    __syncthreads();
    uint32_t at = upto - mine;
    int count = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      if (i < w) at += mem.total[i];
      count += (int)mem.total[i];
    }
    count = alike(count);
    for (int i = 0; i < each; ++i)
      if (named(tid * each + i)) mem.list[at++] = (uint16_t)(tid * each + i);
    __syncthreads();

    const int steps = ((count << lg_halves) + 1) / 2;
    Halves next;
    int next_slot[2];
    uint32_t next_missing;
    auto prepare = [&](int s) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int q = 2 * s + h, e = q >> lg_halves;
        const int slot = alike((int)mem.list[e < count ? e : 0]);
        next_slot[h] = slot;
        next.first[h] = e < count ? ((w0 + slot) << lg_block) + (q & ((1 << lg_halves) - 1)) * kHalf : -1;
      }
      auto first = [&](int gr) { return next.of<T, DP>(gr); };
      next_missing = src.missing(first);
      const uint32_t to = kv0 + (uint32_t)((s & 1) * 2 * R::kBytes);
      src.load(to, to + R::kBytes, w, first);
    };
    prepare(0);
    for (int s = 0; s < steps; ++s) {
      const Halves now = next;
      const int slot[2] = {next_slot[0], next_slot[1]};
      const uint32_t missing = next_missing;
      wait_loads<0>();
      wait_reads();
      barrier();  // the step's rows are there, and nobody reads the other slot any more
      if (s + 1 < steps) prepare(s + 1);
      uint32_t sel = 0;
      bool edge = missing != 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t bits = mem.mask[slot[h] * words + (row.token >> 5)];
        const bool in = (now.first[h] >= 0) & row.in & (((bits >> (row.token & 31)) & 1u) != 0u);
        sel |= in ? 1u << h : 0u;
        // keys behind a row's own position
        edge |= in & (now.first[h] + kHalf - 1 > row.pos);
      }
      if (__ballot(sel != 0u) == 0) continue;
      const bool some = __ballot(sel != 3u) != 0;  // not all
      const uint32_t kb = kv0 + (uint32_t)((s & 1) * 2 * R::kBytes);
      body(now, sel, some, __ballot(edge) != 0, missing, kb, kb + R::kBytes);
    }
    wait_loads<0>();
  }
}

}  // namespace
}  // namespace fs
