// block_walk.hpp — a workgroup's walk over the blocks that its queries select: the
// kernels of many queries, forward and gradient of the queries
// (block_attention.hip, block_attention_grad.hip).
//
// A workgroup takes consecutive tokens of a sequence, all heads of one group, 16
// rows a tile and two tiles a wave.  Tokens near each other select many of the same
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
__host__ __device__ inline int tokens_of(int group) { return WAVES * 32 / group; }

// Head by head over the XCDs (each has its keys and values in a cache of its own), a
// head's last tiles first: they have the most blocks to choose from.
template <int WAVES>
__device__ inline bool walk_tile(const BlockArgs& p, int lane, WalkTile& t) {
  const int64_t at = xcd_range_block(blockIdx.x, gridDim.x);
  t.head = (int)(at / p.tiles);
  t.per = tokens_of<WAVES>(p.group);
  int tile;
  if (!find_tile(p.seqs, t.per, p.tiles - 1 - at % p.tiles, lane, t.seq, tile)) return false;
  t.sq = sequence_at(p.seqs, t.seq);
  const int first = tile * t.per;
  t.token0 = t.sq.first + first;
  t.tokens = t.sq.count - first < t.per ? t.sq.count - first : t.per;
  t.pos0 = t.sq.keys - t.sq.count + first;
  return true;
}

// The rows of a wave's two tiles.
template <int WAVES>
__device__ inline void rows_of(const BlockArgs& p, const WalkTile& t, int w, int lane, RowOf (&row)[2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = w * 32 + i * 16 + (lane & 15);
    row[i].token = r / p.group;
    row[i].head = r % p.group;
    row[i].in = row[i].token < t.tokens;
    if (!row[i].in) row[i].token = 0;
    row[i].pos = row[i].in ? t.pos0 + row[i].token : -1;
  }
}

// One step's groups of 16 keys: the position of each one's first key (negative:
// none), and its block's place in the window.
template <class T, int DP>
struct Step {
  static constexpr int kGroups = Rows<T, DP>::kGroups;
  int first[kGroups], slot[kGroups];
  uint32_t missing;
};

template <class T, int DP, int WAVES, class Body>
__device__ inline void walk_blocks(const BlockArgs& p, const WalkTile& t, const RowOf (&row)[2],
                                   WalkMemory<WAVES>& mem, uint8_t (&kv)[2][2][Rows<T, DP>::kBytes], int tid, int w,
                                   int lane, Body body) {
  using R = Rows<T, DP>;
  constexpr int THREADS = 64 * WAVES, G = R::kGroups;
  const int block = p.seqs.block, lg_block = p.lg_groups + 4;
  const int words = (t.per + 31) / 32, window = kMaskWords / words;
  const int last = t.pos0 + t.tokens - 1;
  const int n_blocks = last < 0 ? 0 : (last >> lg_block) + 1;
  const int entries = t.tokens * p.top;
  const int32_t* ids = p.blocks + (int64_t)t.token0 * p.b_token + (int64_t)t.head * p.b_head;

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
    uint32_t mine = 0;
    for (int i = 0; i < each; ++i) {
      const int b = tid * each + i;
      uint32_t any = 0;
      if (b < here)
        for (int k = 0; k < words; ++k) any |= mem.mask[b * words + k];
      mine += any != 0;
    }
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
    for (int i = 0; i < each; ++i) {
      const int b = tid * each + i;
      uint32_t any = 0;
      if (b < here)
        for (int k = 0; k < words; ++k) any |= mem.mask[b * words + k];
      if (any != 0) mem.list[at++] = (uint16_t)b;
    }
    __syncthreads();

    const int steps = ((count << p.lg_groups) + G - 1) / G;
    Step<T, DP> next;
    auto prepare = [&](int s) {
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        const int q = s * G + gr, e = q >> p.lg_groups;
        const bool in = e < count;
        const int slot = __builtin_amdgcn_readfirstlane(in ? (int)mem.list[e] : 0);
        next.slot[gr] = slot;
        next.first[gr] = in ? (w0 + slot) * block + (q & ((1 << p.lg_groups) - 1)) * 16 : -1;
      }
      auto entry = [&](int gr) {
        int f = next.first[0];
#pragma unroll
        for (int i = 1; i < G; ++i) f = gr == i ? next.first[i] : f;
        return f;
      };
      next.missing = missing_pages<T, DP>(p, t.sq, t.seq, entry);
      load_rows<T, DP, WAVES>(p, p.k, t.sq, t.seq, t.head, lds_address(kv[s & 1][0]), w, lane, entry);
      load_rows<T, DP, WAVES>(p, p.v, t.sq, t.seq, t.head, lds_address(kv[s & 1][1]), w, lane, entry);
    };
    prepare(0);
    for (int s = 0; s < steps; ++s) {
      const Step<T, DP> now = next;
      wait_loads<0>();
      wait_reads();
      barrier();  // the step's rows are there, and nobody reads the other slot any more
      if (s + 1 < steps) prepare(s + 1);
      bool sel[2][G];
      bool any[2] = {false, false};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
          if (gr > 0 && p.lg_groups >= (G == 4 ? 2 : 1)) {
            sel[i][gr] = sel[i][0];
            continue;
          }
          const uint32_t bits = mem.mask[now.slot[gr] * words + (row[i].token >> 5)];
          sel[i][gr] = now.first[gr] >= 0 && row[i].in && ((bits >> (row[i].token & 31)) & 1u);
          any[i] |= sel[i][gr];
        }
      const bool a = __ballot(any[0]) != 0, b = __ballot(any[1]) != 0;
      if (!a && !b) continue;
      // keys behind a row's own position, or in no page of the cache
      bool edge = now.missing != 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int gr = 0; gr < G; ++gr) edge |= sel[i][gr] && now.first[gr] + 15 > row[i].pos;
      body(now, sel, a, b, __ballot(edge) != 0, lds_address(kv[s & 1][0]), lds_address(kv[s & 1][1]));
    }
    wait_loads<0>();
  }
}

}  // namespace
}  // namespace fs
