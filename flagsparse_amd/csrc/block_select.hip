// block_select.hip — the blocks that a query attends to: by a score of each block,
//   score[t, h, b] = < sum over the group's heads of q[t], mean[b, h] >
// the largest ones of the blocks before the query's own, with the first and the most
// recent blocks in any case.
//
// Two scores near each other decide which block is read, so they are computed in 64
// bits (products of 32-bit values are exact there) on the 64-bit matrix
// instructions, 16 blocks by 16 tokens; a single token's by 64-bit multiply-adds.
// A workgroup takes 16 tokens of a sequence and one key-value head: scores of some
// hundred blocks at a time go to LDS as ordered integers, behind the best of the
// blocks before, and a wave finds a token's limit by counting, the power of two
// first, then bit by bit.  Of single tokens each wave takes a part of the blocks, and
// one the best of all parts.  Ties go to the lower block.
//
// 16384 tokens of 4 x 16 heads of 128, 256 blocks, bf16 151 us (the queries alone are 268
// MB, 52 us at a copy's rate; the rest is the limits, a wave's two tokens one after the
// other); 32 single tokens of 8 x 4 heads over 1024 blocks 33 us, bound by the latency of
// a wave's loads of means, its search, and up to seven searches more of the wave that
// joins the parts.  Widths of 256: 32 single tokens over 1024 blocks 67 us.
#include "block_tile.hpp"

namespace fs {
namespace {

constexpr int kTokens = 16, kSelectWaves = 8;
constexpr int kChunk = 256;
constexpr int kKeysRow = kMostTop + kChunk + 1;  // (odd: tokens' rows on different banks)

typedef double f64x4 __attribute__((ext_vector_type(4)));

struct SelectArgs {
  fs_block_seqs seqs;
  const void* q;
  int64_t q_token, q_head;
  const void* means;
  int64_t m_seq, m_block, m_head;
  int32_t* out;
  int heads, group, width, most, top, first, recent;
  int lg_block;
  int64_t tiles;
};

// An integer that is ordered as the value is; not-a-numbers come lowest, and above
// the zero of places without a block.
__device__ inline uint64_t ordered(double x) {
  x += 0.0;  // (one zero)
  if (x != x) return 1;
  const uint64_t b = (uint64_t)__double_as_longlong(x);
  return b >> 63 ? ~b : b | (1ull << 63);
}

constexpr int kKeptRegs = kMostTop / 64, kRegs = (kMostTop + kChunk) / 64;

// Of the keys that a wave holds, lane by lane and register by register in the order of
// their blocks (0: none), the `want` largest, to the front of a row of LDS; returns how
// many.  Registers outside `used` hold none.
__device__ inline int keep_best(const uint64_t (&key)[kRegs], const int32_t (&id)[kRegs], uint32_t used, int want,
                                uint64_t* keys, int32_t* ids, int lane) {
  auto count = [&](auto test) {
    int n = 0;
#pragma unroll
    for (int k = 0; k < kRegs; ++k)
      if ((used >> k) & 1u) n += __builtin_popcountll(__ballot(test(key[k])));
    return n;
  };
  uint64_t least = 1;  // all above it are taken, and of those at it the first `ties`
  int ties = 0;
  const int have = count([](uint64_t x) { return x != 0; });
  if (have > want) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < kRegs; ++k)
      if ((used >> k) & 1u) most = most > (uint32_t)(key[k] >> 32) ? most : (uint32_t)(key[k] >> 32);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
      const uint32_t other = (uint32_t)__shfl_xor((int)most, off);
      most = most > other ? most : other;
    }
    most = (uint32_t)alike((int)most);
    // the limit's upper half: within a few powers of two of the largest, mostly
    uint32_t high = 0;
    int bit = 31, n = 0;
    for (uint32_t j = 0; j < 6; ++j) {
      const uint32_t next = (most & 0xfff00000u) - (j << 20);
      n = count([&](uint64_t x) { return (uint32_t)(x >> 32) >= next; });
      if (n >= want) {
        high = next;
        bit = 19;
        break;
      }
    }
    if (n != want || high == 0) {
      for (; bit >= 0; --bit) {
        const uint32_t next = high | 1u << bit;
        n = count([&](uint64_t x) { return (uint32_t)(x >> 32) >= next; });
        if (n >= want) high = next;
        if (n == want) break;
      }
    }
    uint32_t low = 0;
    if (n != want && count([&](uint64_t x) { return (uint32_t)(x >> 32) >= high; }) != want) {
      const int above = count([&](uint64_t x) { return (uint32_t)(x >> 32) > high; });
      for (bit = 31; bit >= 0; --bit) {
        const uint32_t next = low | 1u << bit;
        n = above + count([&](uint64_t x) { return (uint32_t)(x >> 32) == high && (uint32_t)x >= next; });
        if (n >= want) low = next;
        if (n == want) break;
      }
    }
    least = (uint64_t)high << 32 | low;
    ties = want - count([&](uint64_t x) { return x > least; });
  } else {
    ties = have;
  }
  int done = 0;
  const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
  for (int k = 0; k < kRegs; ++k) {
    if (!((used >> k) & 1u)) continue;
    const uint64_t same = __ballot(key[k] == least);
    const bool take = key[k] > least || (key[k] == least && __builtin_popcountll(same & below) < ties);
    const uint64_t m = __ballot(take);
    ties -= __builtin_popcountll(same);
    if (take) {
      const int to = done + __builtin_popcountll(m & below);
      keys[to] = key[k];
      ids[to] = id[k];
    }
    done += __builtin_popcountll(m);
  }
  return done;
}

// The best of a row's `kept` and of the keys of blocks c0 + i, i < here, behind them, as
// far as the blocks are within [from, to).
__device__ inline int keep_best_of_row(uint64_t* keys, int32_t* ids, int kept, int c0, int here, int from, int to,
                                       int want, int lane) {
  uint64_t key[kRegs];
  int32_t id[kRegs];
  uint32_t used = 0;
#pragma unroll
  for (int k = 0; k < kRegs; ++k) {
    key[k] = 0;
    id[k] = 0;
    const int place = k * 64 + lane;
    if (k < kKeptRegs) {
      if (k * 64 >= kept) continue;
      used |= 1u << k;
      if (place < kept) {
        key[k] = keys[place];
        id[k] = ids[place];
      }
    } else {
      if ((k - kKeptRegs) * 64 >= here) continue;
      used |= 1u << k;
      const int b = c0 + place - kMostTop;
      if (place - kMostTop < here && b >= from && b < to) key[k] = keys[place];
      id[k] = b;
    }
  }
  return keep_best(key, id, used, want, keys, ids, lane);
}

// SINGLE: a workgroup takes one token, where few have many blocks.
template <class T, int DP, bool SINGLE>
__global__ __launch_bounds__((64 * kSelectWaves), (SINGLE || DP > 128 ? 2 : 4)) void block_select_kernel(const SelectArgs p) {
  constexpr int E = 16 / (int)sizeof(T), J = DP * (int)sizeof(T) / 64, W = kSelectWaves, kEach = kTokens / W;
  __shared__ uint64_t s_key[kTokens][kKeysRow];
  __shared__ int32_t s_id[kTokens][kMostTop];
  __shared__ int s_kept[W];
  constexpr int kSumRow = DP + 2;  // (16 rows on different banks)
  __shared__ alignas(16) double s_sum[kTokens][kSumRow];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int64_t at = xcd_range_block(blockIdx.x, gridDim.x);
  const int head = (int)(at / p.tiles);
  int seq, tile;
  constexpr int kPer = SINGLE ? 1 : kTokens;
  if (!find_tile(p.seqs, kPer, at % p.tiles, lane, seq, tile)) return;
  const Sequence sq = sequence_of(p.seqs, seq);
  const int t0 = alike(tile) * kPer, n = sq.count - t0 < kPer ? sq.count - t0 : kPer;
  const int64_t token0 = (int64_t)sq.first + t0;
  const int pos0 = seq < p.seqs.n_seqs ? sq.keys - sq.count + t0 : INT32_MIN / 2;
  // blocks that the tile's last token chooses from
  const int last_own = pos0 + n - 1 < 0 ? -1 : (pos0 + n - 1) >> p.lg_block;
  const int limit = last_own - p.recent + 1 < p.most ? last_own - p.recent + 1 : p.most;
  const int want = p.top - p.first - p.recent;  // of a token whose own block is behind both
  const T* means = static_cast<const T*>(p.means) + (seq < p.seqs.n_seqs ? seq * p.m_seq : 0) + head * p.m_head;

  auto load_means = [&](int b, int end, Slice<T> (&m)[J]) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int e = 0; e < E; ++e) m[j].v[e] = (T)0.0f;
      if (b < end && (4 * j + g) * E < p.width) m[j] = load_slice(means + (int64_t)b * p.m_block + (4 * j + g) * E);
    }
  };
  // sums of the group's queries, four columns of a token a thread
  Slice<T> ahead[J];  // the wave's first means
  if (limit > p.first && want > 0) {
    load_means(SINGLE ? limit : w * 16 + i, limit, ahead);
    const int fours = DP / 4;
    for (int x = tid; x < kTokens * fours; x += 64 * W) {
      const int t = x / fours, c = (x - t * fours) * 4;
      double sum[4] = {0.0, 0.0, 0.0, 0.0};
      if (t < n && c < p.width) {
        const T* q = static_cast<const T*>(p.q) + (token0 + t) * p.q_token + (int64_t)head * p.group * p.q_head + c;
#pragma unroll 8
        for (int h = 0; h < p.group; ++h) {
          T v[4];
          __builtin_memcpy(v, q + h * p.q_head, sizeof v);
#pragma unroll
          for (int y = 0; y < 4; ++y) sum[y] += (double)(float)v[y];
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) s_sum[t][c + y] = sum[y];
    }
    __syncthreads();
  }
  int kept[kEach];
#pragma unroll
  for (int x = 0; x < kEach; ++x) kept[x] = 0;

  if constexpr (SINGLE) {
    // a part of the blocks a wave
    const int each = limit > p.first && want > 0 ? ((limit - p.first + W - 1) / W + 15) / 16 * 16 : 0;
    const int from = p.first + w * each, to = each == 0 ? from : from + each < limit ? from + each : limit;
    int mine = 0;
    for (int c0 = from; c0 < to; c0 += kChunk) {
      const int here = to - c0 < kChunk ? to - c0 : kChunk;
      for (int b0 = 0; b0 < here; b0 += 32) {
        Slice<T> m[2][J];
        load_means(c0 + b0 + i, to, m[0]);
        load_means(c0 + b0 + 16 + i, to, m[1]);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          double s = 0.0;
#pragma unroll
          for (int j = 0; j < J; ++j) {
#pragma unroll
            for (int e = 0; e < E; ++e)
              s = __builtin_fma((double)(float)m[x][j].v[e], s_sum[0][(4 * j + g) * E + e], s);
            fence();
          }
          s += __shfl_xor(s, 16);
          s += __shfl_xor(s, 32);
          const int b = b0 + x * 16 + i;
          if (g == 0 && b < here) s_key[w][kMostTop + b] = ordered(s);
        }
      }
      mine = keep_best_of_row(s_key[w], s_id[w], mine, c0, here, from, to, want, lane);
    }
    if (lane == 0) s_kept[w] = mine;
    __syncthreads();
    if (w == 0) {
      // the best of all parts, a register or two of each at a time
      kept[0] = mine;
      for (int x = 1; x < W; ++x) {
        uint64_t key[kRegs];
        int32_t id[kRegs];
        uint32_t used = 0;
        const int other = alike(s_kept[x]);
#pragma unroll
        for (int k = 0; k < kRegs; ++k) {
          key[k] = 0;
          id[k] = 0;
          if (k >= 2 * kKeptRegs) continue;
          const int row = k < kKeptRegs ? 0 : x, place = (k % kKeptRegs) * 64 + lane, have = row == 0 ? kept[0] : other;
          if (have > (k % kKeptRegs) * 64) used |= 1u << k;
          if (place < have) {
            key[k] = s_key[row][place];
            id[k] = s_id[row][place];
          }
        }
        if (other > 0) kept[0] = keep_best(key, id, used, want, s_key[0], s_id[0], lane);
      }
    }
  } else {
    for (int c0 = 0; c0 < limit && want > 0; c0 += kChunk) {
      const int here = limit - c0 < kChunk ? limit - c0 : kChunk;
      if (c0 > 0) __syncthreads();
      for (int b0 = w * 16; b0 < here; b0 += 16 * W) {
        Slice<T> m[J];
        if (c0 + b0 == w * 16) {
#pragma unroll
          for (int j = 0; j < J; ++j) m[j] = ahead[j];
        } else {
          load_means(c0 + b0 + i, limit, m);
        }
        f64x4 s = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (4 * j * E >= p.width) continue;
#pragma unroll
          for (int e = 0; e < E; ++e)
            s = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)m[j].v[e], s_sum[i][(4 * j + g) * E + e], s, 0, 0, 0);
          fence();
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = r * 4 + g;  // of the 64-bit results
          if (b0 + row < here) s_key[i][kMostTop + b0 + row] = ordered(s[r]);
        }
      }
      __syncthreads();
#pragma unroll
      for (int x = 0; x < kEach; ++x) {
        const int t = w * kEach + x;
        if (t >= n) continue;
        const int own = pos0 + t < 0 ? -1 : (pos0 + t) >> p.lg_block;
        const int end = own - p.recent + 1 < p.most ? own - p.recent + 1 : p.most;
        if (end > c0 && end > p.first)
          kept[x] = keep_best_of_row(s_key[t], s_id[t], kept[x], c0, here, p.first, end, want, lane);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < kEach; ++x) {
    const int t = w * kEach + x;
    if (t >= n) continue;
    const int own = pos0 + t < 0 ? -1 : (pos0 + t) >> p.lg_block;
    const int front = own + 1 < p.first ? own + 1 : p.first;
    const int back = own - p.recent + 1 > front ? own - p.recent + 1 : front;  // the first recent one
    int32_t* out = p.out + ((token0 + t) * p.heads + head) * p.top;
    for (int e = lane; e < p.top; e += 64) {
      int id = -1;
      if (e < front) id = e;
      else if (e < front + kept[x]) id = s_id[t][e - front];
      else if (e - front - kept[x] <= own - back) id = back + e - front - kept[x];
      out[e] = id;
    }
  }
}

}  // namespace
}  // namespace fs

extern "C" int fs_block_select(int val_t, const fs_block_seqs* seqs, int heads, int group, int width, const void* q,
                               int64_t q_token, int64_t q_head, const void* means, int64_t most, int64_t m_seq,
                               int64_t m_block, int64_t m_head, int top, int first, int recent, int32_t* out,
                               hipStream_t stream) {
  using namespace fs;
  const char* who = "fs_block_select";
  if (const int rc = block_sizes_fault(who, val_t, seqs, heads, group, width)) return rc;
  if (most < 0 || most > INT32_MAX) return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
  if (top < 1 || top > kMostTop || first < 0 || recent < 1 || first + (int64_t)recent > top)
    return fail(FS_E_INVALID, std::string(who) + ": top, first or recent out of range");
  if (seqs->n_tokens == 0) return FS_OK;
  if (!q || (!means && most > 0) || !out || q_token < 0 || q_head < 0 || m_seq < 0 || m_block < 0 || m_head < 0)
    return fail(FS_E_INVALID, std::string(who) + ": bad pointer or stride");
  SelectArgs p{};
  p.seqs = *seqs;
  p.q = q;
  p.q_token = q_token;
  p.q_head = q_head;
  p.means = means;
  p.m_seq = m_seq;
  p.m_block = m_block;
  p.m_head = m_head;
  p.out = out;
  p.heads = heads;
  p.group = group;
  p.width = width;
  p.most = (int)most;
  p.top = top;
  p.first = first;
  p.recent = recent;
  p.lg_block = __builtin_ctz((unsigned)seqs->block);
  // One token a workgroup, its blocks over the waves, where they are many and the tokens
  // few (or alone in their tile of 16 in any case).  us of both (single, tiles), bf16, 8
  // heads of 128:
  //   256 blocks   1 token 20, 13; 32 sequences of one 22, 13, of two 28, 16
  //   512 blocks   1 token 22, 21; of 16 sequences two 23, 27
  //   768 blocks   1 token 24, 30; of 16 sequences four 38, 38
  //   1024 blocks  1 token 27, 38; 32 sequences of one 32, 41, of two 47, 50, of four 77, 52
  // Widths above 128, whose means fill a wave's registers: 1024 blocks, 1 token 56, 59; 16
  // sequences of one 75, 61, of four 133, 70, so tiles always.
  const bool single = most >= 640 && width <= 128 &&
                      (seqs->n_tokens <= seqs->n_seqs || seqs->n_tokens * heads <= 512);
  p.tiles = block_tiles(*seqs, single ? 1 : kTokens);
  if (p.tiles * heads > kMostWorkgroups) return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
  return with_block_width(val_t, width, who, [&](auto val, auto dp) -> int {
    using T = decltype(val);
    constexpr int DP = decltype(dp)::value;
    const dim3 grid((uint32_t)(p.tiles * heads)), threads(64 * kSelectWaves);
    if constexpr (DP <= 128) {
      if (single) {
        hipLaunchKernelGGL((block_select_kernel<T, DP, true>), grid, threads, 0, stream, p);
        FS_CHECK_MAIN_LAUNCH("block_select_single_kernel");
        return FS_OK;
      }
    }
    hipLaunchKernelGGL((block_select_kernel<T, DP, false>), grid, threads, 0, stream, p);
    FS_CHECK_MAIN_LAUNCH("block_select_kernel");
    return FS_OK;
  });
}
