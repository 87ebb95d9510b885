// block_walk.hpp — a workgroup's walk over the blocks that its queries select: the
// kernels of many queries, forward and gradient of the queries
// (block_attention.hip, block_attention_grad.hip).
//
// A workgroup takes consecutive tokens of a sequence, all heads of one group, 16
// rows a wave.  Tokens near each other select many of the same blocks: a table in LDS
// holds, for each block of a window of the sequence, a bit for each token that selects
// it.  The blocks with a bit are walked in order, keys and values loaded once for the
// workgroup, and a wave takes part where one of its tokens selects the block.
//
// Which waves take part differs from block to block, so the waves do not meet at a
// barrier: some waves load, a step each in turn, into a ring of slots, and the others
// follow each at its own pace.  A loader says in LDS which step a slot holds; a wave that
// has read it adds one to the slot's count, and a slot is loaded again when all that take
// part have.  Every wait ends: each wave goes through its steps in order, and the first
// step that is not yet read by all waits for its loader alone, which waits for the
// readers of the step that had its slot before, an earlier one.
// A loader is one wave, which issues an instruction in some cycles: what it needs is laid
// out 64 blocks at a time, a lane each.  It announces a step before it goes on to its
// next: with two or three steps of a loader under way 16384 tokens of 4 x 16 heads took 3%
// and 5% longer, chunks of 4 x 512 tokens 3% and 7% (of two pairs of loaders, one for the
// keys and one for the values).
#pragma once

#include <cstddef>

#include "block_tile.hpp"

namespace fs {
namespace {

constexpr int kMaskWords = 2048;

// Waves that read and that load, and slots by what LDS holds.
template <class T, int DP, int READERS, int LOADERS>
struct WalkShape {
  static constexpr int kReaders = READERS, kLoaders = LOADERS, kWaves = READERS + LOADERS, kThreads = 64 * kWaves;
  static constexpr int kBytes = Rows<T, DP>::kBytes;
  static constexpr int kSlots = kBytes > 8192 ? 4 : 8;
  static_assert(kSlots % LOADERS == 0, "a slot is one loader's");
  struct alignas(1024) Memory {
    uint8_t kv[kSlots][2][kBytes];  // (first: kv0 in what follows is its address)
    uint32_t mask[kMaskWords];
    uint64_t part[READERS][kMaskWords / 64];  // listed blocks that a wave takes part in
    uint16_t list[kMaskWords];
    uint32_t total[kWaves];
    uint32_t ready[2][kSlots];  // 1 + the step that a slot holds; of the keys, of the values
    uint32_t missing[kSlots];
    uint32_t done[kSlots];
  };
};

// What a workgroup works on.
struct WalkTile {
  Sequence sq;
  int seq, head;
  int token0, tokens;  // of all tokens; how many
  int pos0;            // position of the first
};

// Head by head over the XCDs (each has its keys and values in a cache of its own), a
// head's last tiles first: they have the most blocks to choose from.
__device__ inline bool walk_tile(const BlockArgs& p, uint32_t block, int lane, WalkTile& t) {
  const int64_t at = xcd_range_block(block, (uint32_t)(p.tiles * p.heads));
  t.head = (int)(at / p.tiles);
  int tile;
  if (!find_tile(p.seqs, p.per, p.tiles - 1 - at % p.tiles, lane, t.seq, tile)) return false;
  t.sq = sequence_of(p.seqs, t.seq);
  const int first = alike(tile) * p.per;
  t.token0 = t.sq.first + first;
  t.tokens = t.sq.count - first < p.per ? t.sq.count - first : p.per;
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

// Words in LDS that other waves of the workgroup write, by their addresses.
__device__ inline uint32_t look(uint32_t at) { return (uint32_t)alike((int)*(volatile lds_word*)(uintptr_t)at); }
__device__ inline void tell(uint32_t at, uint32_t v) { *(volatile lds_word*)(uintptr_t)at = v; }
__device__ inline void in_order() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <class Shape>
__device__ inline void walk_start(typename Shape::Memory& mem, int tid) {
  if (tid < Shape::kSlots) mem.ready[0][tid] = mem.ready[1][tid] = mem.done[tid] = 0u;
}

// The walk of a wave that loads (LOADS) or reads: body(...) takes a step, calls values()
// before it reads the values and done() once, when it has read all.  Both kinds
// meet at the same barriers; each has code of its own, so that a loader's holds no rows.
template <class T, int DP, class Shape, bool LOADS, class Body>
__device__ inline void walk_blocks(const BlockArgs& p, const WalkTile& t, const RowOf& row, typename Shape::Memory& mem,
                                   uint32_t kv0, int tid, int w, int lane, Body body) {
  using R = Rows<T, DP>;
  constexpr int THREADS = Shape::kThreads, READERS = Shape::kReaders, S = Shape::kSlots;
  constexpr int kLoads = KeySource<T, DP>::kLoads;
  const int lg_block = p.lg_groups + 4, lg_steps = lg_block - 5;  // of a block
  const int words = (p.per + 31) / 32, window = kMaskWords / words;
  const int last = t.pos0 + t.tokens - 1;
  const int n_blocks = last < 0 ? 0 : (last >> lg_block) + 1;
  const int entries = t.tokens * p.top;
  const int32_t* ids = p.blocks + (int64_t)t.token0 * p.b_token + (int64_t)t.head * p.b_head;
  // the words that hold the wave's tokens, and their bits
  const int t_lo = w * 16 / p.group, t_hi = (w * 16 + 15) / p.group;
  const int word_lo = t_lo >> 5, word_hi = t_hi >> 5;
  const uint32_t bits_lo = word_lo == word_hi ? (uint32_t)(((uint64_t)1 << (t_hi - t_lo + 1)) - 1) << (t_lo & 31)
                                              : ~0u << (t_lo & 31);
  const uint32_t bits_hi = word_lo == word_hi ? 0u : (uint32_t)(((uint64_t)1 << ((t_hi & 31) + 1)) - 1);
  const uint32_t ready0 = kv0 + (uint32_t)offsetof(typename Shape::Memory, ready);
  const uint32_t missing0 = kv0 + (uint32_t)offsetof(typename Shape::Memory, missing);
  const uint32_t done0 = kv0 + (uint32_t)offsetof(typename Shape::Memory, done);
  uint32_t base = 0;  // steps of the windows before
  uint32_t expected[S / Shape::kLoaders];  // readings of a loader's slots so far
#pragma unroll
  for (int i = 0; i < S / Shape::kLoaders; ++i) expected[i] = 0u;

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
    for (int i = 0; i < Shape::kWaves; ++i) {
      if (i < w) at += mem.total[i];
      count += (int)mem.total[i];
    }
    count = alike(count);
    for (int i = 0; i < each; ++i)
      if (named(tid * each + i)) mem.list[at++] = (uint16_t)(tid * each + i);
    __syncthreads();
    if constexpr (!LOADS) {
      for (int u0 = 0; u0 < count; u0 += 64) {
        uint32_t any = 0;
        if (u0 + lane < count) {
          const uint32_t* m = &mem.mask[mem.list[u0 + lane] * words];
          if (word_lo < words) any |= m[word_lo] & bits_lo;
          if (word_hi < words) any |= m[word_hi] & bits_hi;
        }
        const uint64_t m = __ballot(any != 0);
        if (lane == 0) mem.part[w][u0 >> 6] = m;
      }
    }
    __syncthreads();

    const uint32_t steps = (uint32_t)count << lg_steps;
    if constexpr (LOADS) {
      constexpr uint32_t LOADERS = Shape::kLoaders, OWN = S / LOADERS;  // slots of this one
      const uint32_t nth = (uint32_t)(w - READERS);
      KeySource<T, DP> k, v;
      k.init(p, p.k, t.sq, t.seq, t.head, lane);
      v.init(p, p.v, t.sq, t.seq, t.head, lane);
      // a block's rows are one behind the other in packed rows and in a page that holds it
      const bool together = k.table == nullptr || k.shift >= lg_block;
      uint32_t readers = 0;  // of 64 blocks, a lane each
      int first = 0;         // their first keys
      uint64_t k_at = 0, v_at = 0;
      uint64_t here = 0;     // those whose page is in the cache
      int chunk = -1;
      for (uint32_t x = (nth + LOADERS - base % LOADERS) % LOADERS; x < steps; x += LOADERS) {
        const uint32_t step = base + x;
        const int u = (int)(x >> lg_steps), ss = (int)(x & ((1u << lg_steps) - 1u)), uu = u & 63;
        if (u >> 6 != chunk) {
          chunk = u >> 6;
          readers = 0;
#pragma unroll
          for (int r = 0; r < READERS; ++r) readers += (uint32_t)(mem.part[r][chunk] >> lane) & 1u;
          const int mine = chunk * 64 + lane;
          first = mine < count ? (w0 + (int)mem.list[mine]) << lg_block : 0;
          int64_t page = 0;
          if (together && k.table != nullptr) {
            const int at = first >> k.shift;
            page = at < k.per_seq ? p.seqs.pages[(int64_t)t.seq * p.seqs.ld_pages + at] : -1;
            if (page >= k.n_pages) page = -1;
          }
          k_at = (uint64_t)(uintptr_t)k.rows_at(page < 0 ? 0 : page, first);
          v_at = (uint64_t)(uintptr_t)v.rows_at(page < 0 ? 0 : page, first);
          here = __ballot(page >= 0);
        }
        typename KeySource<T, DP>::Place k_place, v_place;
        const int j = __builtin_amdgcn_readlane(first, uu) + ss * R::kKeys;
        k_place.missing = 0;
        k_place.whole = v_place.whole = together && j + R::kKeys <= k.keys && ((here >> uu) & 1u);
        if (k_place.whole) {
          auto at = [&](uint64_t a, uint32_t row) {
            const uint64_t bytes = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(a >> 32), uu) << 32 |
                                   (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)a, uu);
            return (const char*)(uintptr_t)(bytes + (uint64_t)((uint32_t)(ss * R::kKeys)) * row);
          };
          k_place.at[0] = at(k_at, k.row);
          v_place.at[0] = at(v_at, v.row);
        } else {
          k.find(j, k_place);
          v.find(j, v_place);
        }
        const uint32_t i = step % S, own = i / LOADERS;
        uint32_t want = 0;
#pragma unroll
        for (uint32_t n = 0; n < OWN; ++n)
          if (n == own) want = expected[n];
        while (look(done0 + 4 * i) != want) __builtin_amdgcn_s_sleep(1);
        in_order();
        if (lane == 0) tell(missing0 + 4 * i, k_place.missing);
        const uint32_t to = kv0 + 2 * i * Shape::kBytes;
        k.load(to, k_place, lane);
        v.load(to + Shape::kBytes, v_place, lane);
        const uint32_t n_readers = (uint32_t)__builtin_amdgcn_readlane((int)readers, uu);
#pragma unroll
        for (uint32_t n = 0; n < OWN; ++n)
          if (n == own) expected[n] += n_readers;
        wait_loads<kLoads>();  // the keys' are done
        if (lane == 0) tell(ready0 + 4 * i, step + 1);
        wait_loads<0>();
        if (lane == 0) tell(ready0 + 4 * (S + i), step + 1);
      }
    } else {
      // (a wave of one token takes part with all its rows)
      const bool alone = t_lo == t_hi;
      for (int u0 = 0; u0 < count; u0 += 64) {
        uint64_t left = mem.part[w][u0 >> 6];
        left = (uint64_t)(uint32_t)alike((int)(uint32_t)left) | (uint64_t)(uint32_t)alike((int)(uint32_t)(left >> 32)) << 32;
        const int mine = u0 + lane < count ? (int)mem.list[u0 + lane] : 0;  // 64 blocks
        for (; left != 0; left &= left - 1) {
          const int uu = __builtin_ctzll(left), u = u0 + uu, nth = __builtin_amdgcn_readlane(mine, uu);
          bool sel = row.in;
          if (!alone) sel &= ((mem.mask[nth * words + (row.token >> 5)] >> (row.token & 31)) & 1u) != 0u;
          const bool some = __ballot(sel) != ~0ull;  // not all
          for (int ss = 0; ss < 1 << lg_steps; ++ss) {
            const int now = ((w0 + nth) << lg_block) + ss * R::kKeys;
            const bool edge = __ballot(sel & (now + R::kKeys - 1 > row.pos)) != 0;  // keys behind a row's position
            const uint32_t step = base + ((uint32_t)u << lg_steps) + (uint32_t)ss;
            const uint32_t i = step % S;
            while (look(ready0 + 4 * i) != step + 1) __builtin_amdgcn_s_sleep(1);
            in_order();
            const uint32_t missing = p.seqs.pages != nullptr ? look(missing0 + 4 * i) : 0u;
            body(
                now, sel, some, edge || missing != 0, missing, kv0 + 2 * i * Shape::kBytes,
                kv0 + (2 * i + 1) * Shape::kBytes,
                [&] {
                  while (look(ready0 + 4 * (S + i)) != step + 1) __builtin_amdgcn_s_sleep(1);
                  in_order();
                },
                [&] {
                  wait_reads();
                  if (lane == 0)
                    __hip_atomic_fetch_add((lds_word*)(uintptr_t)(done0 + 4 * i), 1u, __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_WORKGROUP);
                  in_order();
                });
          }
        }
      }
    }
    base += steps;
  }
}

template <class T, int DP, class Shape>
__device__ inline void walk_loads(const BlockArgs& p, const WalkTile& t, typename Shape::Memory& mem, uint32_t kv0,
                                  int tid, int w, int lane) {
  walk_blocks<T, DP, Shape, true>(p, t, RowOf{}, mem, kv0, tid, w, lane, [] {});
}

}  // namespace
}  // namespace fs
