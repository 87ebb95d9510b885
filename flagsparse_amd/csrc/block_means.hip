// block_means.hip — the mean of each block's keys, what a query's score of the block
// is taken with.
//
// One pass over the keys: a wave takes one head of a block, as many rows at a time
// as its 64 lanes have 16-byte slices for, sums in 32 bits and adds its rows' sums at
// the end, in a fixed order.  216 MB of f16 keys 47 us, 4.6 TB/s (36 us where they lie in
// the 256 MB cache).  The blocks of 64 new keys 10 us: a lane looks up the page of each
// of its 16 rows and loads the row, one after the other, and waits for both.
#include "block_tile.hpp"

namespace fs {
namespace {

struct MeansArgs {
  fs_block_seqs seqs;
  RowLayout k;
  const int32_t* start;
  void* out;
  int64_t m_seq, m_block, m_head;
  int heads, width, most;
  int lg_block;
};

// Blocks of sequence b that are written, and the first of them.
__device__ inline int blocks_of(const MeansArgs& p, int b, int& first, int& keys) {
  const Sequence q = sequence_at(p.seqs, b);
  keys = q.keys;
  first = 0;
  if (p.start != nullptr) {
    const int from = p.start[b];
    if (from >= q.keys) return 0;
    first = from > 0 ? from >> p.lg_block : 0;
  }
  int last = (int)(((int64_t)q.keys + p.seqs.block - 1) >> p.lg_block);
  last = last < p.most ? last : p.most;
  return last > first ? last - first : 0;
}

template <class T>
__global__ __launch_bounds__(256) void block_means_kernel(const MeansArgs p) {
  constexpr int E = Slice<T>::n;
  const int lane = threadIdx.x & 63;
  const int slices = p.width / E, groups = 64 / slices;  // lanes a row, rows at a time
  const int mine = lane / slices, slice = lane - mine * slices;
  const int64_t waves = (int64_t)gridDim.x * 4;
  for (int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);; item += waves) {
    const int64_t at = item / p.heads;
    const int head = (int)(item - at * p.heads);
    int seq = -1, block = 0;
    int64_t before = 0;
    for (int64_t b0 = 0; b0 < p.seqs.n_seqs; b0 += 64) {
      int first = 0, keys, own = 0;
      if (b0 + lane < p.seqs.n_seqs) own = blocks_of(p, (int)b0 + lane, first, keys);
      const uint32_t upto = wave_sum_scan((uint32_t)own);
      const uint64_t m = __ballot(before + upto > at);
      if (m != 0) {
        const int l = __builtin_ctzll(m);
        seq = (int)b0 + l;
        block = (int)(at - before) - (int)(__builtin_amdgcn_readlane((int)upto, l) - __builtin_amdgcn_readlane(own, l)) +
                __builtin_amdgcn_readlane(first, l);
        break;
      }
      before += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63);
    }
    if (seq < 0) return;
    const Sequence q = sequence_at(p.seqs, seq);
    const int j0 = block << p.lg_block;
    const int rows = q.keys - j0 < p.seqs.block ? q.keys - j0 : p.seqs.block;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.0f;
    int held = 0;  // rows that are in the cache
    if (mine < groups) {
      for (int r = mine; r < rows; r += groups) {
        const T* row = key_rows<T>(p.seqs, q, seq, p.k, head, (j0 + r) & ~15);
        if (row != nullptr) {
          const Slice<T> x = load_slice(row + (int64_t)((j0 + r) & 15) * p.k.row + slice * E);
#pragma unroll
          for (int e = 0; e < E; ++e) sum[e] += (float)x.v[e];
          ++held;
        }
      }
    }
    float total[E];
    int n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) total[e] = 0.0f;
    for (int g = 0; g < groups; ++g) {
#pragma unroll
      for (int e = 0; e < E; ++e) total[e] += __shfl(sum[e], g * slices + slice);
      n += __shfl(held, g * slices + slice);
    }
    if (mine == 0) {
      Slice<T> y;
#pragma unroll
      for (int e = 0; e < E; ++e) y.v[e] = (T)(n > 0 ? total[e] / (float)n : 0.0f);
      store_slice(static_cast<T*>(p.out) + seq * p.m_seq + block * p.m_block + head * p.m_head + slice * E, y);
    }
  }
}

}  // namespace
}  // namespace fs

extern "C" int fs_block_means(int val_t, const fs_block_seqs* seqs, int heads, int width, const void* k, int64_t k_page,
                              int64_t k_row, int64_t k_head, const int32_t* start, int64_t most, void* out,
                              int64_t m_seq, int64_t m_block, int64_t m_head, hipStream_t stream) {
  using namespace fs;
  const char* who = "fs_block_means";
  if (const int rc = block_sizes_fault(who, val_t, seqs, heads, 1, width)) return rc;
  if (most < 0 || most > INT32_MAX) return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
  if (seqs->n_seqs == 0 || most == 0) return FS_OK;
  if (!k || !out || k_page < 0 || k_row < 0 || k_head < 0 || m_seq < 0 || m_block < 0 || m_head < 0)
    return fail(FS_E_INVALID, std::string(who) + ": bad pointer or stride");
  MeansArgs p{};
  p.seqs = *seqs;
  p.k = RowLayout{k, k_page, k_row, k_head};
  p.start = start;
  p.out = out;
  p.m_seq = m_seq;
  p.m_block = m_block;
  p.m_head = m_head;
  p.heads = heads;
  p.width = width;
  p.most = (int)most;
  p.lg_block = __builtin_ctz((unsigned)seqs->block);
  // a wave an item, as far as the chip holds waves: with `start` the items are as many
  // as the new keys touch, which only the device knows
  int64_t items = seqs->n_seqs * most;
  if (seqs->pages == nullptr) items = std::min(items, seqs->n_rows / seqs->block + seqs->n_seqs);
  if (start != nullptr && seqs->q_offsets == nullptr) items = std::min(items, seqs->n_seqs);  // (a decode step's)
  const int64_t blocks = std::min<int64_t>(ceil_div(items * heads, 4), 256 * 8);
  auto run = [&](auto v) -> int {
    using T = decltype(v);
    hipLaunchKernelGGL((block_means_kernel<T>), dim3((uint32_t)blocks), dim3(256), 0, stream, p);
    FS_CHECK_MAIN_LAUNCH("block_means_kernel");
    return FS_OK;
  };
  return val_t == FS_F16 ? run((_Float16)0) : val_t == FS_BF16 ? run((__bf16)0) : run(0.0f);
}
