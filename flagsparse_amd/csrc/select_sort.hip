// select_sort.hip — positions sorted by a small key: the transpose of a
// selection matrix (one entry a row, in column ids[i]).
//
// order lists the positions 0..n-1 by key, equal keys in position order;
// inverse is its inverse.  The key of an id outside [0, n_keys) is n_keys, so
// such positions come last.  A token's experts and a batch's tokens are sorted
// by this one routine (expert order; the embedding gradient's segments).
//
// Counting sort, least significant digit first: up to 10 key bits a pass, one
// pass for experts, two for a vocabulary.  A pass counts the digits of each tile
// of 512 to 4096 positions, scans the counts, and scatters: a tile is ranked
// stably, a wave taking 64 positions at a time, the lanes with its digit found
// by ballots, and waves owning consecutive sub-tiles, so ranks need no order of
// atomics.  Up to 4096 positions are sorted by one workgroup in one launch, all
// passes through LDS.
//
// Bound by launches and the latency of their steps, not by bytes: us, 64 x 8 slots
// of 64 experts 5 (one launch), 131072 x 8 of 128 18 (16.8 MB; three launches),
// 4095 tokens of 20011 13 (one launch), 65536 of 131072 22 (four).
#include <type_traits>

#include "radix_tile.hpp"
#include "select_rows.hpp"

namespace fs {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMaxBits = 10;
constexpr int kMaxDigits = 1 << kMaxBits;
// Up to this many counts, 64 a thread, a scatter adds up those of the tiles
// before it itself; more are scanned by a launch of their own.  us with a scan and
// without: 32768 x 2 slots of 64 experts 14.0 and 11.6, 8192 x 8 of 256 (512
// digits, 64 tiles) 13.5 and 11.5; an embedding gradient of 65536 tokens, 1000 rows
// of 512 (1024 digits, 64 tiles), 40.3 and 43.9 in all.
constexpr int64_t kSelfScan = 64 * kThreads;

template <class Id>
__device__ inline uint32_t key_of(Id id, uint32_t n_keys) {
  // (a negative id is a large unsigned one)
  return sizeof(Id) == 8 ? ((uint64_t)id < n_keys ? (uint32_t)id : n_keys)
                         : ((uint32_t)id < n_keys ? (uint32_t)id : n_keys);
}

// Keys from the ids themselves (KEYS = false) or from an earlier pass.
template <class Id, bool KEYS>
__device__ inline uint32_t load_key(const void* __restrict__ src, int64_t i, uint32_t n_keys) {
  if constexpr (KEYS) return static_cast<const uint32_t*>(src)[i];
  else return key_of(static_cast<const Id*>(src)[i], n_keys);
}

template <class Id, bool KEYS, int CH>
__global__ __launch_bounds__(kThreads) void select_count_kernel(const void* __restrict__ src, int64_t n,
                                                                uint32_t n_keys, int shift, int nd,
                                                                uint32_t* __restrict__ cnt) {
  __shared__ uint32_t s_cnt[kMaxDigits];
  for (int d = threadIdx.x; d < nd; d += kThreads) s_cnt[d] = 0u;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * (kThreads * CH);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t i = base + c * kThreads + threadIdx.x;
    if (i < n) atomicAdd(&s_cnt[(load_key<Id, KEYS>(src, i, n_keys) >> shift) & (uint32_t)(nd - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < nd; d += kThreads) cnt[(int64_t)blockIdx.x * nd + d] = s_cnt[d];
}

// scanned: cnt holds, per digit, the sum over the tiles before, and totals that
// over all; otherwise the tiles' counts are added up here.
// Writes sorted keys, order, inverse and offsets where asked for.
template <class Id, bool KEYS, int CH>
__global__ __launch_bounds__(kThreads) void select_scatter_kernel(
    const void* __restrict__ src, const int32_t* __restrict__ pos_in, int64_t n, uint32_t n_keys, int shift, int nd,
    const uint32_t* __restrict__ cnt, const uint32_t* __restrict__ totals, int64_t n_tiles, bool scanned,
    uint32_t* __restrict__ keys_out, int32_t* __restrict__ pos_out, int32_t* __restrict__ inverse,
    int32_t* __restrict__ offsets) {
  constexpr int kTile = kThreads * CH;
  __shared__ uint32_t s_cnt[kWaves][kMaxDigits];  // then the tile's keys, in order of their digits
  __shared__ uint32_t s_base[kMaxDigits];
  __shared__ uint32_t s_part[2 * kThreads];
  __shared__ uint32_t s_wave[kWaves], s_wave_own[kWaves];
  __shared__ int32_t s_pos[kTile];
  static_assert(sizeof(uint32_t) * kTile <= sizeof(s_cnt), "a tile's keys fit its counters");
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t tile = blockIdx.x;
  const int64_t first = (tile * kWaves + w) * (64 * CH) + lane;
  const int64_t wave_left = n - (first - lane);  // (the same for the whole wave)
  for (int d = tid; d < nd; d += kThreads)
    for (int k = 0; k < kWaves; ++k) s_cnt[k][d] = 0u;

  uint32_t key[CH];
  int32_t pos[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t i = first + c * 64;
    key[c] = i < n ? load_key<Id, KEYS>(src, i, n_keys) : 0u;
    pos[c] = pos_in != nullptr && i < n ? pos_in[i] : (int32_t)i;
  }
  // per digit: the count of all tiles (tot) and of those before this one (pre),
  // loaded before anything waits; a thread's digits are tid * per + j, or tid % nd
  // with the tiles shared by groups of threads
  uint32_t tot[kMaxDigits / kThreads] = {}, pre[kMaxDigits / kThreads] = {};
  const int per = nd > kThreads ? nd / kThreads : 1, groups = nd < kThreads ? kThreads / nd : 1;
  if (!scanned) {
    for (int j = 0; j < per; ++j) {
      const int d = groups > 1 ? tid % nd : tid * per + j;
      uint32_t a = 0u, b = 0u;
#pragma unroll 8
      for (int64_t t = groups > 1 ? tid / nd : 0; t < n_tiles; t += groups) {
        const uint32_t v = cnt[t * nd + d];
        a += v;
        b += t < tile ? v : 0u;
      }
      tot[j] = a;
      pre[j] = b;
    }
  } else {
    for (int j = 0; j < per; ++j)
      if (tid * per + j < nd) {
        tot[j] = totals[tid * per + j];
        pre[j] = cnt[tile * nd + tid * per + j];
      }
  }

  __syncthreads();
  uint32_t rank[CH];
  const uint32_t mask = (uint32_t)(nd - 1);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    rank[c] = 0u;
    if (c * 64 >= wave_left) continue;
    const bool active = first + c * 64 < n;
    const uint32_t digit = (key[c] >> shift) & mask;
    const uint64_t peers = match_lanes<kMaxBits>(digit, __ballot(active), mask);
    const int below = count_below_t(peers);
    uint32_t before = 0u;
    if (active) before = s_cnt[w][digit];
    wave_sync_t();
    if (active && below == 0) s_cnt[w][digit] = before + (uint32_t)__popcll(peers);
    wave_sync_t();
    rank[c] = before + (uint32_t)below;
  }
  __syncthreads();
  // counts of the waves -> places within the tile's run of each digit
  uint32_t own[kMaxDigits / kThreads] = {};  // the tile's own counts, digits tid * per + j
  for (int j = 0; j < per; ++j) {
    const int d = tid * per + j;
    if (d >= nd) break;
    uint32_t v[kWaves], run = 0u;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) v[k] = s_cnt[k][d];
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
      s_cnt[k][d] = run;
      run += v[k];
    }
    own[j] = run;
  }
  if (!scanned && groups > 1) {
    s_part[tid] = tot[0];
    s_part[kThreads + tid] = pre[0];
    __syncthreads();
    if (tid < nd)
      for (int g = 1; g < groups; ++g) {
        tot[0] += s_part[g * nd + tid];
        pre[0] += s_part[kThreads + g * nd + tid];
      }
  }
  // first places of the digits, in the whole and within the tile
  uint32_t mine = 0u, mine_own = 0u;
  if (tid * per < nd)
    for (int j = 0; j < per; ++j) {
      mine += tot[j];
      mine_own += own[j];
    }
  const uint32_t upto = wave_sum_scan(mine), upto_own = wave_sum_scan(mine_own);
  if (lane == 63) {
    s_wave[w] = upto;
    s_wave_own[w] = upto_own;
  }
  __syncthreads();
  uint32_t run = upto - mine, run_own = upto_own - mine_own;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    run += k < w ? s_wave[k] : 0u;
    run_own += k < w ? s_wave_own[k] : 0u;
  }
  if (tid * per < nd)
    for (int j = 0; j < per; ++j) {
      const int d = tid * per + j;
      // places within the tile for ranking; what to add to one for the place in the whole
      for (int k = 0; k < kWaves; ++k) s_cnt[k][d] += run_own;
      s_base[d] = run + pre[j] - run_own;
      // one pass: the digit is the key
      if (offsets != nullptr && tile == 0 && (uint32_t)d <= n_keys) offsets[d] = (int32_t)run;
      run += tot[j];
      run_own += own[j];
    }
  __syncthreads();
  uint32_t at[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) at[c] = s_cnt[w][(key[c] >> shift) & mask] + rank[c];
  __syncthreads();
  // through LDS, so that a digit's run leaves as whole lines (order[at] straight
  // from the lanes that ranked it: 13.0 us for 131072 x 8 slots of 128 experts, 11.2 so)
  uint32_t* s_key = &s_cnt[0][0];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int64_t i = first + c * 64;
    if (i >= n) continue;
    s_key[at[c]] = key[c];
    s_pos[at[c]] = pos[c];
    if (inverse != nullptr) inverse[pos[c]] = (int32_t)(s_base[(key[c] >> shift) & mask] + at[c]);
  }
  __syncthreads();
  const int64_t tile_left = n - tile * kTile;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = c * kThreads + tid;
    if (i >= tile_left) continue;
    const uint32_t k = s_key[i], to = s_base[(k >> shift) & mask] + (uint32_t)i;
    if (keys_out != nullptr) keys_out[to] = k;
    if (pos_out != nullptr) pos_out[to] = s_pos[i];
  }
}

// All of the sort by one workgroup of W waves, 64 CH positions each, W = 1..16.
// The others write zeros meanwhile, for the embedding gradient: as many bytes as
// the sort hides (table gradients, us without and with: 4096 tokens of 32000 x 4096
// bf16 78 and 61, 4095 of 20011 x 1001 f32 39 and 34, with twice the bytes 75 and 34;
// 1 of 32000 x 1024 bf16 23 and 18, 512 of 50000 x 1024 f32 39 and 40).
constexpr int kSmallWaves = 16, kSmallChunks = 4;
constexpr int64_t kSmall = 64 * kSmallWaves * kSmallChunks;
constexpr uint32_t kFillGroups = 512;
template <bool PAST>
__device__ inline void fill_zeros(uint8_t* __restrict__ p, int64_t bytes) {
  const int64_t i = (int64_t)(blockIdx.x - 1) * blockDim.x + threadIdx.x, step = (int64_t)kFillGroups * blockDim.x;
  const Slice<uint16_t> zero{};
  for (int64_t q = i; q < bytes / 16; q += step) store_slice<PAST>(reinterpret_cast<uint16_t*>(p + q * 16), zero);
  if (i < bytes % 16) p[bytes / 16 * 16 + i] = 0;
}
template <class Id, int CH>
__global__ __launch_bounds__(64 * kSmallWaves) void select_small_kernel(
    const Id* __restrict__ ids, int n, uint32_t n_keys, int bits, int passes, uint32_t* __restrict__ keys_out,
    int32_t* __restrict__ order, int32_t* __restrict__ inverse, int32_t* __restrict__ offsets,
    uint8_t* __restrict__ zeros, int64_t zero_bytes) {
  if (blockIdx.x > 0) return fill_zeros<(CH > 1)>(zeros, zero_bytes);
  __shared__ uint16_t s_cnt[kSmallWaves][kMaxDigits];
  __shared__ uint32_t s_base[kMaxDigits];
  __shared__ uint32_t s_wave[kSmallWaves];
  __shared__ uint32_t s_key[64 * kSmallWaves * CH];
  __shared__ uint16_t s_pos[64 * kSmallWaves * CH];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), threads = blockDim.x,
            waves = threads >> 6;
  const int nd = 1 << bits, per = (nd + threads - 1) / threads;
  const uint32_t mask = (uint32_t)(nd - 1);
  uint32_t key[CH], rank[CH];
  int pos[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int i = (w * CH + c) * 64 + lane;
    key[c] = i < n ? key_of(ids[i], n_keys) : 0u;
    pos[c] = i;
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    for (int k = 0; k < waves; ++k)
      for (int d = tid; d < nd; d += threads) s_cnt[k][d] = 0;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      rank[c] = 0u;
      if ((w * CH + c) * 64 >= n) continue;
      const bool active = (w * CH + c) * 64 + lane < n;
      const uint32_t digit = (key[c] >> shift) & mask;
      const uint64_t peers = match_lanes<kMaxBits>(digit, __ballot(active), mask);
      const int below = count_below_t(peers);
      uint32_t before = 0u;
      if (active) before = s_cnt[w][digit];
      wave_sync_t();
      if (active && below == 0) s_cnt[w][digit] = (uint16_t)(before + (uint32_t)__popcll(peers));
      wave_sync_t();
      rank[c] = before + (uint32_t)below;
    }
    __syncthreads();
    uint32_t mine = 0u;
    for (int j = 0; j < per; ++j) {
      const int d = tid * per + j;
      if (d >= nd) break;
      uint32_t v[kSmallWaves], run = 0u;
#pragma unroll
      for (int k = 0; k < kSmallWaves; ++k) v[k] = k < waves ? s_cnt[k][d] : 0u;
#pragma unroll
      for (int k = 0; k < kSmallWaves; ++k) {
        if (k < waves) s_cnt[k][d] = (uint16_t)run;  // (at most 4096)
        run += v[k];
      }
      s_base[d] = mine;  // within the thread's digits
      mine += run;
    }
    const uint32_t upto = wave_sum_scan(mine);
    if (lane == 63) s_wave[w] = upto;
    __syncthreads();
    const uint32_t waves_upto = wave_sum_scan(lane < waves ? s_wave[lane] : 0u);
    const uint32_t run = upto - mine + (w > 0 ? (uint32_t)__builtin_amdgcn_readlane((int)waves_upto, w - 1) : 0u);
    for (int j = 0; j < per; ++j) {
      const int d = tid * per + j;
      if (d >= nd) break;
      s_base[d] += run;
      // (one pass: the digit is the key)
      if (offsets != nullptr && (uint32_t)d <= n_keys) offsets[d] = (int32_t)s_base[d];
    }
    __syncthreads();
    const bool last = pass + 1 == passes;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if ((w * CH + c) * 64 + lane >= n) continue;
      const uint32_t digit = (key[c] >> shift) & mask, at = s_base[digit] + s_cnt[w][digit] + rank[c];
      if (!last) {
        s_key[at] = key[c];
        s_pos[at] = (uint16_t)pos[c];
      } else {
        if (keys_out != nullptr) keys_out[at] = key[c];
        if (order != nullptr) order[at] = pos[c];
        if (inverse != nullptr) inverse[pos[c]] = (int32_t)at;
      }
    }
    if (last) break;
    __syncthreads();
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int i = (w * CH + c) * 64 + lane;
      key[c] = i < n ? s_key[i] : 0u;
      pos[c] = i < n ? (int)s_pos[i] : 0;
    }
  }
}

// Passes over keys 0..n_keys: equal shares of their bits.
struct Passes {
  int count, bits;
};
Passes passes_of(int64_t n_keys) {
  int bits = 1;
  while (bits < 32 && (n_keys >> bits) != 0) ++bits;
  const int count = (bits + kMaxBits - 1) / kMaxBits;
  return {count, (bits + count - 1) / count};
}

// Positions a tile: 512, 1024 or 2048, the fewest that make at most 64 tiles, or
// 4096 from 256 tiles on (more tiles are more counts to scan, fewer leave compute
// units idle).  us for slots of 64 experts, tiles of 2048 and 4096: 262144 10.5 and
// 13.0, 524288 12.3 and 14.1; of 128, 2097152 25.5 and 22.0.
int chunks_of(int64_t n) {
  int ch = 1;
  while (ch < 4 && n > (int64_t)kThreads * ch * 64) ch *= 2;
  return n > (int64_t)kThreads * ch * 256 ? 2 * ch : ch;
}

struct SortLayout {
  size_t cnt, totals, keys[2], pos[2], bytes;
  int ch;
  int64_t tiles;
};
SortLayout sort_layout(int64_t n, int64_t n_keys) {
  const Passes p = passes_of(n_keys);
  SortLayout l{};
  if (n <= kSmall) return l;
  l.ch = chunks_of(n);
  l.tiles = ceil_div(n, (int64_t)kThreads * l.ch);
  const int64_t nd = (int64_t)1 << p.bits;
  size_t at = 0;
  auto take = [&](size_t b) {
    const size_t a = at;
    at += (b + 255) / 256 * 256;
    return a;
  };
  l.cnt = take((size_t)(l.tiles * nd) * 4);
  if (l.tiles * nd > kSelfScan) l.totals = take((size_t)nd * 4);
  // passes before the last write keys and positions, in turn
  for (int k = 0; k < 2 && k + 1 < p.count; ++k) {
    l.keys[k] = take((size_t)n * 4);
    l.pos[k] = take((size_t)n * 4);
  }
  l.bytes = at;
  return l;
}

struct PassArgs {
  const void* src;
  const int32_t* pos_in;
  int64_t n;
  uint32_t n_keys;
  int shift, nd;
  uint32_t* keys_out;
  int32_t *pos_out, *inverse, *offsets;
};

template <class Id, bool KEYS, int CH>
int sort_pass(const PassArgs& a, uint8_t* ws, const SortLayout& l, hipStream_t s) {
  uint32_t* cnt = reinterpret_cast<uint32_t*>(ws + l.cnt);
  uint32_t* totals = reinterpret_cast<uint32_t*>(ws + l.totals);
  hipLaunchKernelGGL((select_count_kernel<Id, KEYS, CH>), dim3((uint32_t)l.tiles), dim3(kThreads), 0, s, a.src, a.n,
                     a.n_keys, a.shift, a.nd, cnt);
  FS_CHECK_LAUNCH("select_count_kernel");
  const bool scanned = l.tiles * a.nd > kSelfScan;
  if (scanned) {
    hipLaunchKernelGGL(wg_scan_column_kernel, dim3((uint32_t)a.nd), dim3(256), 0, s, cnt, l.tiles, a.nd, totals);
    FS_CHECK_LAUNCH("wg_scan_column_kernel");
  }
  hipLaunchKernelGGL((select_scatter_kernel<Id, KEYS, CH>), dim3((uint32_t)l.tiles), dim3(kThreads), 0, s, a.src,
                     a.pos_in, a.n, a.n_keys, a.shift, a.nd, cnt, totals, l.tiles, scanned, a.keys_out, a.pos_out,
                     a.inverse, a.offsets);
  FS_CHECK_MAIN_LAUNCH("select_scatter_kernel");
  return FS_OK;
}
template <class Id, bool KEYS>
int sort_pass(const PassArgs& a, uint8_t* ws, const SortLayout& l, hipStream_t s) {
  switch (l.ch) {
    case 1: return sort_pass<Id, KEYS, 1>(a, ws, l, s);
    case 2: return sort_pass<Id, KEYS, 2>(a, ws, l, s);
    case 4: return sort_pass<Id, KEYS, 4>(a, ws, l, s);
  }
  return sort_pass<Id, KEYS, 8>(a, ws, l, s);
}

__global__ __launch_bounds__(256) void zero_offsets_kernel(int32_t* __restrict__ p, int64_t n) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n) p[i] = 0;
}

}  // namespace

size_t select_sort_bytes(int64_t n, int64_t n_keys) { return n > 0 ? sort_layout(n, n_keys).bytes : 0; }

// The zeros that a sort can write beside its own work.  (Beside the launches of a
// sort of many positions they cost more than they save: each launch's end waits for
// them: 64 MB of them made the gradient of 65536 tokens, 131072 x 2048, 1.27 times as
// long.)
int64_t select_sort_fill_bytes(int64_t n) {
  return n == 0 || n > kSmall ? 0 : (int64_t)(n > 64 * kSmallWaves ? 96 : 64) << 20;
}

// keys_out, inverse and offsets may be null; offsets needs one pass.  Also writes
// zero_bytes zeros, at most select_sort_fill_bytes(n).
int select_sort(const void* ids, int id_t, int64_t n, int64_t n_keys, uint32_t* keys_out, int32_t* order,
                int32_t* inverse, int32_t* offsets, uint8_t* ws, hipStream_t s, void* zeros, int64_t zero_bytes) {
  if (n == 0) {
    if (offsets != nullptr) {
      hipLaunchKernelGGL(zero_offsets_kernel, dim3((uint32_t)ceil_div(n_keys + 1, 256)), dim3(256), 0, s, offsets,
                         n_keys + 1);
      FS_CHECK_LAUNCH("zero_offsets_kernel");
    }
    return FS_OK;
  }
  const Passes p = passes_of(n_keys);
  if (n <= kSmall) {
    auto launch = [&](auto id, auto chunks) {
      using Id = decltype(id);
      constexpr int CH = decltype(chunks)::value;
      hipLaunchKernelGGL((select_small_kernel<Id, CH>), dim3(zero_bytes > 0 ? 1 + kFillGroups : 1),
                         dim3((uint32_t)(ceil_div(n, 64 * CH) * 64)), 0, s, (const Id*)ids, (int)n, (uint32_t)n_keys,
                         p.bits, p.count, keys_out, order, inverse, offsets, static_cast<uint8_t*>(zeros), zero_bytes);
    };
    using One = std::integral_constant<int, 1>;
    using Four = std::integral_constant<int, kSmallChunks>;
    const bool one = n <= 64 * kSmallWaves;
    if (id_t == FS_I64) one ? launch(int64_t(0), One{}) : launch(int64_t(0), Four{});
    else one ? launch(int32_t(0), One{}) : launch(int32_t(0), Four{});
    FS_CHECK_MAIN_LAUNCH("select_small_kernel");
    return FS_OK;
  }
  const SortLayout l = sort_layout(n, n_keys);
  const int nd = 1 << p.bits;
  const void* src = ids;
  const int32_t* pos = nullptr;
  for (int k = 0; k < p.count; ++k) {
    const bool last = k + 1 == p.count;
    uint32_t* ko = last ? keys_out : reinterpret_cast<uint32_t*>(ws + l.keys[k & 1]);
    int32_t* po = last ? order : reinterpret_cast<int32_t*>(ws + l.pos[k & 1]);
    int32_t* inv = last ? inverse : nullptr;
    const PassArgs a{src, pos, n, (uint32_t)n_keys, k * p.bits, nd, ko, po, inv, offsets};
    const int rc = k > 0            ? sort_pass<int32_t, true>(a, ws, l, s)
                   : id_t == FS_I64 ? sort_pass<int64_t, false>(a, ws, l, s)
                                    : sort_pass<int32_t, false>(a, ws, l, s);
    if (rc != FS_OK) return rc;
    src = ko;
    pos = po;
  }
  return FS_OK;
}

int select_max_one_pass_keys() { return kMaxDigits - 1; }

}  // namespace fs

extern "C" size_t fs_expert_route_workspace_bytes(int64_t n, int64_t n_experts) {
  if (n <= 0 || n > INT32_MAX || n_experts < 1 || n_experts > fs::select_max_one_pass_keys()) return 0;
  return fs::select_sort_bytes(n, n_experts);
}

extern "C" int fs_expert_route(int id_t, int64_t n, int64_t n_experts, const void* experts, int32_t* order,
                               int32_t* inverse, int32_t* offsets, void* ws, size_t ws_bytes, hipStream_t stream) {
  if (id_t != FS_I32 && id_t != FS_I64) return fs::fail(FS_E_INVALID, "fs_expert_route: bad type code");
  if (n < 0 || n > INT32_MAX) return fs::fail(FS_E_INVALID, "fs_expert_route: slots out of range");
  if (n_experts < 1 || n_experts > fs::select_max_one_pass_keys())
    return fs::fail(FS_E_INVALID, "fs_expert_route: n_experts out of range");
  if (offsets == nullptr || (n > 0 && (experts == nullptr || order == nullptr || inverse == nullptr)))
    return fs::fail(FS_E_INVALID, "fs_expert_route: null pointer");
  const size_t need = fs_expert_route_workspace_bytes(n, n_experts);
  if (need > 0 && (ws == nullptr || ws_bytes < need))
    return fs::fail(FS_E_WORKSPACE, "fs_expert_route: workspace too small");
  return fs::select_sort(experts, id_t, n, n_experts, nullptr, order, inverse, offsets, static_cast<uint8_t*>(ws),
                         stream, nullptr, 0);
}
