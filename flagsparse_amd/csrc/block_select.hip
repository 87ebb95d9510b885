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
// blocks before, and a wave finds a token's limit bit by bit, by counting.  Ties go
// to the lower block.
#include "block_tile.hpp"

namespace fs {
namespace {

constexpr int kTokens = 16, kSelectWaves = 4;
constexpr int kChunk = 384;
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

template <class T, int DP>
__global__ __launch_bounds__(64 * kSelectWaves) void block_select_kernel(const SelectArgs p) {
  constexpr int E = 16 / (int)sizeof(T), J = DP * (int)sizeof(T) / 64;
  __shared__ uint64_t s_key[kTokens][kKeysRow];
  __shared__ int32_t s_id[kTokens][kMostTop];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i = lane & 15, g = lane >> 4;
  const int64_t at = xcd_range_block(blockIdx.x, gridDim.x);
  const int head = (int)(at / p.tiles);
  int seq, tile;
  if (!find_tile(p.seqs, kTokens, at % p.tiles, lane, seq, tile)) return;
  const Sequence sq = sequence_at(p.seqs, seq);
  const int t0 = tile * kTokens, n = sq.count - t0 < kTokens ? sq.count - t0 : kTokens;
  const int64_t token0 = (int64_t)sq.first + t0;
  const int pos0 = seq < p.seqs.n_seqs ? sq.keys - sq.count + t0 : INT32_MIN / 2;

  // sums of the group's queries: the lane's pieces 4 j + g of its token (of a single
  // token, the same in all lanes of g)
  double qs[J * E];
#pragma unroll
  for (int x = 0; x < J * E; ++x) qs[x] = 0.0;
  const int mine = n == 1 ? 0 : i;
  if (mine < n) {
    for (int h = 0; h < p.group; ++h) {
      const T* q = static_cast<const T*>(p.q) + (token0 + mine) * p.q_token + (int64_t)(head * p.group + h) * p.q_head;
#pragma unroll
      for (int j = 0; j < J; ++j)
        if ((4 * j + g) * E < p.width) {
          const Slice<T> v = load_slice(q + (4 * j + g) * E);
#pragma unroll
          for (int e = 0; e < E; ++e) qs[j * E + e] += (double)(float)v.v[e];
        }
    }
  }

  // blocks that the tile's last token chooses from
  const int last_own = pos0 + n - 1 < 0 ? -1 : (pos0 + n - 1) >> p.lg_block;
  const int limit = last_own - p.recent + 1 < p.most ? last_own - p.recent + 1 : p.most;
  const T* means = static_cast<const T*>(p.means) + (seq < p.seqs.n_seqs ? seq * p.m_seq : 0) + head * p.m_head;
  int kept[kTokens / kSelectWaves];
#pragma unroll
  for (int x = 0; x < kTokens / kSelectWaves; ++x) kept[x] = 0;

  for (int c0 = 0; c0 < limit; c0 += kChunk) {
    const int here = limit - c0 < kChunk ? limit - c0 : kChunk;
    __syncthreads();
    for (int b0 = w * 16; b0 < here; b0 += 16 * kSelectWaves) {
      Slice<T> m[J];
      const int b = c0 + b0 + i;
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int e = 0; e < E; ++e) m[j].v[e] = (T)0.0f;
        if (b < limit && (4 * j + g) * E < p.width) m[j] = load_slice(means + (int64_t)b * p.m_block + (4 * j + g) * E);
      }
      if (n == 1) {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int e = 0; e < E; ++e) s = __builtin_fma((double)(float)m[j].v[e], qs[j * E + e], s);
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (g == 0 && b0 + i < here) s_key[0][kMostTop + b0 + i] = ordered(s);
      } else {
        f64x4 s = {0.0, 0.0, 0.0, 0.0};
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int e = 0; e < E; ++e)
            s = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)m[j].v[e], qs[j * E + e], s, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = r * 4 + g;  // of the 64-bit results
          if (b0 + row < here) s_key[i][kMostTop + b0 + row] = ordered(s[r]);
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kTokens / kSelectWaves; ++x) {
      const int t = w * (kTokens / kSelectWaves) + x;
      if (t >= n) continue;
      const int own = pos0 + t < 0 ? -1 : (pos0 + t) >> p.lg_block;
      const int end = own - p.recent + 1 < p.most ? own - p.recent + 1 : p.most;
      if (end <= c0 || end <= p.first) continue;
      const int want = p.top - p.first - p.recent;  // (own >= first + recent here)
      constexpr int K = (kMostTop + kChunk) / 64;
      uint64_t key[K];
      int32_t id[kMostTop / 64];
      int have = 0;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int place = k * 64 + lane;
        bool in;
        if (k < kMostTop / 64) {
          in = place < kept[x];
          id[k] = in ? s_id[t][place] : 0;
        } else {
          const int b = c0 + place - kMostTop;
          in = b >= p.first && b < end && place - kMostTop < here;
        }
        key[k] = in ? s_key[t][place] : 0ull;
        have += __builtin_popcountll(__ballot(key[k] != 0));
      }
      // the limit: all above it are taken, and of those at it the first `ties`
      uint64_t least = 1;
      int ties = 0;
      if (have > want) {
        least = 0;
        for (int bit = 63; bit >= 0; --bit) {
          const uint64_t next = least | 1ull << bit;
          int count = 0;
#pragma unroll
          for (int k = 0; k < K; ++k) count += __builtin_popcountll(__ballot(key[k] >= next));
          if (count >= want) least = next;
          if (count == want) break;
        }
        int above = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) above += __builtin_popcountll(__ballot(key[k] > least));
        ties = want - above;
      } else {
        ties = have;
      }
      int done = 0;
      const uint64_t below = ((uint64_t)1 << lane) - 1;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const uint64_t same = __ballot(key[k] == least);
        const bool take = key[k] > least || (key[k] == least && __builtin_popcountll(same & below) < ties);
        const uint64_t m = __ballot(take);
        ties -= __builtin_popcountll(same);
        if (take) {
          const int to = done + __builtin_popcountll(m & below);
          s_key[t][to] = key[k];
          s_id[t][to] = k < kMostTop / 64 ? id[k < kMostTop / 64 ? k : 0] : c0 + k * 64 + lane - kMostTop;
        }
        done += __builtin_popcountll(m);
      }
      kept[x] = done;
    }
  }
#pragma unroll
  for (int x = 0; x < kTokens / kSelectWaves; ++x) {
    const int t = w * (kTokens / kSelectWaves) + x;
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
  p.tiles = block_tiles(*seqs, kTokens);
  if (p.tiles * heads > kMostWorkgroups) return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
  return with_block_width(val_t, width, who, [&](auto val, auto dp) -> int {
    using T = decltype(val);
    constexpr int DP = decltype(dp)::value;
    hipLaunchKernelGGL((block_select_kernel<T, DP>), dim3((uint32_t)(p.tiles * heads)), dim3(64 * kSelectWaves), 0,
                       stream, p);
    FS_CHECK_MAIN_LAUNCH("block_select_kernel");
    return FS_OK;
  });
}
