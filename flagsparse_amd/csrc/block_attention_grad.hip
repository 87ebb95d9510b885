// block_attention_grad.hip — gradients of the attention over selected blocks.
//
// With S = scale Q K^T on the selection, P = exp(S - lse) its rows' softmax, which
// the forward pass's lse gives again without their sums, and G the gradient of the
// result O:
//   dV = P^T G          dP = G V^T          dS = P (dP - <G, O>)
//   dQ = scale dS K     dK = scale dS^T Q
// The queries' gradient walks a workgroup's blocks as the forward pass does.  The
// keys' and values' need the selection's transpose, the tokens of each block: the
// entries sorted by block (select_sort.hip), in pieces of about the same length,
// since the first block has every token and most have few.  A workgroup takes one
// piece and 32 or 64 of a block's keys; pieces of one block leave their sums in the
// workspace, which are added in order, so no atomics' order shows.
//
// P and dS of 16-bit values go through the matrix cores in two parts (Rows::halves), as
// the forward pass's weights do: in one, errors are 1.4 times as large and the case below
// takes 1437 us.
//
// 8192 tokens of 4 x 8 heads of 128, 16 blocks of 64 keys, bf16: 1556 us, 201 TFLOP/s; kernels
// under the profiler: the queries' part 770, bound as the forward pass is, by what its waves wait for each other
// (matrix instructions busy for 21% of the cycles, LDS for 31%), the keys' 724: eight
// waves of 16 keys, so that two are on a SIMD (four of 32 keys, one on each, took 14%
// longer), which wait for 47% of their cycles, for a step's rows and at its barrier
// (matrix instructions 22%, LDS 26%), joining the pieces' sums 70, sorting and cutting the
// lists 40.  The queries' gradient alone 732, the keys' and values' 865.
#include "block_walk.hpp"

namespace fs {
namespace {

// Waves that read, of the queries' gradient, by the bytes of a row: with the loaders as
// many as have the registers that they need, 128, 168 or 256.
constexpr int query_readers(int row) { return row <= 128 ? 12 : row <= 256 ? 8 : 6; }

// dS of float16, whose small values have few bits, times a power of two: of a query's
// own in its gradient, of a key's own in the key's.  It follows the largest value so far,
// as the softmax's maximum does, and keeps it between 2^8 and 2^15; what is summed up is
// scaled again where it changes, and the gradients are divided by it in 32 bits.  So
// neither rows whose gradient is small beside others' nor small weights lose bits.
// (bfloat16 and float32 have the exponents.)
template <class T>
constexpr bool kFactored = std::is_same_v<T, _Float16>;
constexpr float kFirstFactor = 0x1p100f;

// `most`: the largest value of a step, of the lane's query or key.  Not finite: the sum
// will not be either, whatever the factor.
template <int N>
__device__ inline void follow(float most, float& factor, f32x4 (&sum)[N]) {
  const bool grown = most * factor > 0x1p15f && most < INFINITY;
  if (__ballot(grown) == 0) return;
  const int at = (int)((__float_as_uint(factor) >> 23) & 255u);
  const int to = grown ? 262 - (int)((__float_as_uint(most) >> 23) & 255u) : at;  // most: [2^8, 2^9)
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) sum[n][r] = __builtin_amdgcn_ldexpf(sum[n][r], to - at);
  factor = __uint_as_float((uint32_t)to << 23);
}

// P of float16 in the values' gradient: times 2^15, at most.
template <class T>
constexpr float kWeightLift = std::is_same_v<T, _Float16> ? 15.0f : 0.0f;

// ---- gradient of the queries ------------------------------------------------------

template <class T, int DP>
struct QueryGrad {
  typename Mma<T>::frag q[Rows<T, DP>::kFrags], g[Rows<T, DP>::kFrags];
  f32x4 d[DP / 16];
  float lse, delta;  // in powers of two; <G, O>
  float factor;
};

template <class T, int DP, int AHEAD, class Wait, class Done>
__device__ inline void take(QueryGrad<T, DP>& st, uint32_t kb, uint32_t vb, bool sel, int now, bool some,
                            bool edge, const RowOf& row, float c, int used, int lane, Wait values, Done done) {
  using R = Rows<T, DP>;
  constexpr int G = R::kGroups, P = R::kUnit / 16;
  f32x4 s[G], dp[G];
#pragma unroll
  for (int gr = 0; gr < G; ++gr) s[gr] = dp[gr] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  products<T, DP, AHEAD>(kb, st.q, s, used, lane);
  values();  // are there
  products<T, DP, AHEAD>(vb, st.g, dp, used, lane);
  Columns<T, DP, AHEAD> k;
  k.read(kb, 0, used, lane);
#pragma unroll
  for (int gr = 0; gr < G; ++gr)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[gr][r], c, -st.lse));
      s[gr][r] = x * (dp[gr][r] - st.delta);
    }
  if (edge) {
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      const int last = row.pos - now - 16 * gr - 4 * (lane >> 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[gr][r] = r <= last ? s[gr][r] : 0.0f;
    }
  }
  if (some) {
#pragma unroll
    for (int gr = 0; gr < G; ++gr)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[gr][r] = sel ? s[gr][r] : 0.0f;
  }
  if constexpr (kFactored<T>) {
    float most = 0.0f;
#pragma unroll
    for (int gr = 0; gr < G; ++gr)
#pragma unroll
      for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(s[gr][r]));
    follow(across_max(most), st.factor, st.d);
#pragma unroll
    for (int gr = 0; gr < G; ++gr) s[gr] *= st.factor;
  }
  // dS in two parts of the values' type, as the forward pass's weights
  typename R::Halves w[G / P];
#pragma unroll
  for (int u = 0; u < G / P; ++u) w[u] = R::halves(&s[u * P]);
  k.add(kb, w, st.d, used, lane, done);
}

struct GradArgs {
  BlockArgs b;  // q, k, v, blocks; out: the queries' gradient
  const void* grad;
  const void* o;
  const float* lse;
  float* delta;        // <G, O> of each row
  const int32_t* order;
  const int4* pieces;  // key, first entry, one behind the last, place of its sums or -1
  const int32_t* n_pieces;
  const int2* sums;    // of each key: place of its first sums, and their number
  float* parts;
  void* dk;
  void* dv;
  int lists;           // selections a token: heads, or 1 where the heads share one
  int key_blocks;      // blocks that keys may name, of all sequences
  uint32_t per_group;  // 2^32 / group, rounded up
};

// A row without what is left out, see careful_row.
template <class T, int DP>
__device__ __forceinline__ void careful_query(const GradArgs& a, const Sequence& sq, int seq, int64_t token, int head,
                                           int in_group, int pos, float lse, float delta, int lane) {
  const BlockArgs& p = a.b;
  const int hq = head * p.group + in_group, block = p.seqs.block, lg = p.lg_groups + 4;
  const int64_t at = token * p.heads * p.group + hq;
  const T* q = static_cast<const T*>(p.q) + token * p.q_token + (int64_t)hq * p.q_head;
  const T* g = static_cast<const T*>(a.grad) + at * p.width;
  const int32_t* ids = p.blocks + token * p.b_token + (int64_t)head * p.b_head;
  const float c = p.scale * kLog2e;
  float d[(DP + 63) / 64];
#pragma unroll
  for (int i = 0; i < (DP + 63) / 64; ++i) d[i] = 0.0f;
  for (int e = 0; e < p.top; ++e) {
    const int id = ids[e];
    bool use = id >= 0 && id <= (pos >> lg);
    for (int b = 0; b < e; ++b) use = use && ids[b] != id;
    if (!use) continue;
    for (int j0 = 0; j0 < block; j0 += 64) {
      const int j = id * block + j0 + lane;
      const bool seen = j0 + lane < block && j <= pos && j < sq.keys;
      float w = 0.0f;
      if (seen) {
        const T* k = key_rows<T>(p.seqs, sq, seq, p.k, head, j & ~15) + (int64_t)(j & 15) * p.k.row;
        const T* v = key_rows<T>(p.seqs, sq, seq, p.v, head, j & ~15) + (int64_t)(j & 15) * p.v.row;
        float s = 0.0f, y = 0.0f;
        for (int x = 0; x < p.width; ++x) {
          s = __builtin_fmaf((float)q[x], (float)k[x], s);
          y = __builtin_fmaf((float)g[x], (float)v[x], y);
        }
        w = __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -lse)) * (y - delta);
      }
      for (uint64_t left = __ballot(seen); left != 0; left &= left - 1) {
        const int l = __builtin_ctzll(left), jj = id * block + j0 + l;
        const float weight = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(w), l));
        const T* k = key_rows<T>(p.seqs, sq, seq, p.k, head, jj & ~15) + (int64_t)(jj & 15) * p.k.row;
#pragma unroll
        for (int i = 0; i < (DP + 63) / 64; ++i)
          if (i * 64 + lane < p.width) d[i] = __builtin_fmaf(weight, (float)k[i * 64 + lane], d[i]);
      }
    }
  }
  T* out = static_cast<T*>(p.out) + at * p.width;
#pragma unroll
  for (int i = 0; i < (DP + 63) / 64; ++i)
    if (i * 64 + lane < p.width) out[i * 64 + lane] = (T)(d[i] * p.scale);
}

template <class T, int DP>
struct QueryGradShape : WalkShape<T, DP, query_readers(DP * (int)sizeof(T)), (DP * sizeof(T) > 256 ? 2 : 4)> {
  static constexpr int kAhead = 8;
};

template <class T, int DP>
__global__ __launch_bounds__((QueryGradShape<T, DP>::kThreads)) void block_query_grad_kernel(const GradArgs a) {
  using R = Rows<T, DP>;
  using Shape = QueryGradShape<T, DP>;
  __shared__ typename Shape::Memory mem;
  const BlockArgs& p = a.b;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  WalkTile t;
  if (!walk_tile(p, blockIdx.x, lane, t)) {
    if (tid < Shape::kReaders) p.again[(int64_t)blockIdx.x * Shape::kReaders + tid] = 0u;
    return;
  }
  const bool all = p.out != nullptr;  // or <G, O> alone, for the keys
  walk_start<Shape>(mem, tid);
  if (w >= Shape::kReaders) {
    if (all) walk_loads<T, DP, Shape>(p, t, mem, lds_address(&mem), tid, w, lane);
    return;
  }
  const RowOf row = row_of(p, t, w, lane);
  QueryGrad<T, DP> st;
  st.factor = kFactored<T> ? kFirstFactor : 1.0f;
  const int hq = t.head * p.group + row.head;
  const int64_t at = (int64_t)(t.token0 + row.token) * p.heads * p.group + hq;
  load_row<T, DP>(static_cast<const T*>(p.q) + (int64_t)(t.token0 + row.token) * p.q_token + (int64_t)hq * p.q_head,
                  row.in, p.width, lane, st.q);
  load_row<T, DP>(static_cast<const T*>(a.grad) + at * p.width, row.in, p.width, lane, st.g);
  {
    typename R::frag o[R::kFrags];
    load_row<T, DP>(static_cast<const T*>(a.o) + at * p.width, row.in, p.width, lane, o);
    float sum = 0.0f;
#pragma unroll
    for (int ks = 0; ks < R::kFrags; ++ks)
#pragma unroll
      for (int e = 0; e < 16 / (int)sizeof(T); ++e) sum = __builtin_fmaf((float)st.g[ks][e], (float)o[ks][e], sum);
    sum = across_sum(sum);
    if (row.in && lane < 16) a.delta[at] = sum;
    if (!all) return;
    st.delta = sum;
    st.lse = row.in ? a.lse[at] * kLog2e : 0.0f;
  }
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt) st.d[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const float c = p.scale * kLog2e;
  const int used = (p.width + 15) / 16;
  walk_blocks<T, DP, Shape, false>(p, t, row, mem, lds_address(&mem), tid, w, lane,
                            [&](int now, bool sel, bool some, bool edge, uint32_t, uint32_t kb, uint32_t vb, auto values,
                                auto done) {
                              take<T, DP, Shape::kAhead>(st, kb, vb, sel, now, some, edge, row, c, used, lane, values,
                                                         done);
                            });
  bool bad = false;
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) bad |= !__builtin_isfinite(st.d[dt][r]);
  const uint64_t rows = __ballot(bad && row.in);
  if (row.in) store_row<T, DP>(static_cast<T*>(p.out) + at * p.width, st.d, p.scale / st.factor, p.width, lane);
  if (lane == 0)
    p.again[(int64_t)blockIdx.x * Shape::kReaders + w] = (uint32_t)(rows | rows >> 16 | rows >> 32 | rows >> 48) & 0xffffu;
}

// Rows whose gradient is not finite, key after key: those of one workgroup of the kernel
// above, by `waves` waves.
template <class T, int DP>
__device__ inline void queries_again(const GradArgs& a, uint32_t block, int w, int waves, int lane) {
  const BlockArgs& p = a.b;
  constexpr int READERS = QueryGradShape<T, DP>::kReaders;
  for (; w < READERS; w += waves) {
    uint32_t rows = (uint32_t)alike((int)p.again[(int64_t)block * READERS + w]);
    WalkTile t;
    if (rows == 0 || !walk_tile(p, block, lane, t)) continue;
    for (; rows != 0; rows &= rows - 1) {
      const int r = w * 16 + __builtin_ctz(rows), tok = r / p.group, in_group = r - tok * p.group;
      const int64_t at = (int64_t)(t.token0 + tok) * p.heads * p.group + t.head * p.group + in_group;
      careful_query<T, DP>(a, t.sq, t.seq, t.token0 + tok, t.head, in_group, t.pos0 + tok, a.lse[at] * kLog2e, a.delta[at],
                           lane);
    }
  }
}

// ---- the selection's transpose ----------------------------------------------------

// Number of a sequence's first block among all blocks: those of one sequence are
// consecutive, and no two sequences share one, without their lengths' sum.
__device__ inline int first_block(const fs_block_seqs& s, int b, int lg_block) {
  return (clamp_to(s.k_offsets[b], 0, s.n_rows) >> lg_block) + b;
}

// The key that each entry of the selection is sorted by, head by head and block by
// block; one too large for entries that name nothing or the same block again.  A
// wave takes a token.  Also zeros the gradients of rows of no sequence.
__global__ __launch_bounds__(256) void block_keys_kernel(const BlockArgs p, int lists, int key_blocks, int32_t* keys,
                                                         uint32_t* dk, uint32_t* dv, int64_t row_words) {
  const int lane = threadIdx.x & 63, lg = p.lg_groups + 4;
  const int64_t waves = (int64_t)gridDim.x * 4, first = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int n_keys = lists * key_blocks;
  for (int64_t token = first; token < p.seqs.n_tokens; token += waves) {
    int seq, pos, base = 0;
    Sequence sq;
    const bool some = [&] {
      seq = (int)p.seqs.n_seqs;
      if (p.seqs.q_offsets == nullptr) {
        seq = (int)token;
      } else {
        for (int64_t b0 = 0; b0 < p.seqs.n_seqs; b0 += 64) {
          bool mine = false;
          if (b0 + lane < p.seqs.n_seqs) {
            const Sequence q = sequence_at(p.seqs, (int)b0 + lane);
            mine = token >= q.first && token < q.first + q.count;
          }
          const uint64_t m = __ballot(mine);
          if (m != 0) {
            seq = (int)b0 + __builtin_ctzll(m);
            break;
          }
        }
      }
      return seq < p.seqs.n_seqs;
    }();
    pos = -1;
    if (some) {
      sq = sequence_at(p.seqs, seq);
      pos = sq.keys - sq.count + (int)(token - sq.first);
      base = first_block(p.seqs, seq, lg);
    }
    for (int e = lane; e < lists * p.top; e += 64) {
      const int list = e / p.top, at = e - list * p.top;
      const int32_t* ids = p.blocks + token * p.b_token + (int64_t)list * p.b_head;
      const int id = ids[at];
      bool use = id >= 0 && id <= (pos >> lg);
      for (int b = 0; b < at; ++b) use = use && ids[b] != id;
      const int64_t key = (int64_t)list * key_blocks + base + id;
      keys[token * lists * p.top + e] = use && base + id < key_blocks ? (int32_t)key : n_keys;
    }
  }
  const int64_t head = p.seqs.n_seqs > 0 ? clamp_to(p.seqs.k_offsets[0], 0, p.seqs.n_rows) : 0;
  const int64_t tail = p.seqs.n_seqs > 0 ? clamp_to(p.seqs.k_offsets[p.seqs.n_seqs], 0, p.seqs.n_rows) : 0;
  const int64_t threads = (int64_t)gridDim.x * 256, me = (int64_t)blockIdx.x * 256 + threadIdx.x;
  for (int64_t i = me; i < head * row_words; i += threads) dk[i] = dv[i] = 0u;
  for (int64_t i = tail * row_words + me; i < p.seqs.n_rows * row_words; i += threads) dk[i] = dv[i] = 0u;
}

// First sorted entry of each key.
__device__ inline int32_t first_of(const uint32_t* keys, int64_t n, uint32_t k) {
  int64_t lo = 0, hi = n;
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < k) lo = mid + 1;
    else hi = mid;
  }
  return (int32_t)lo;
}
__global__ __launch_bounds__(256) void block_lists_kernel(const uint32_t* keys, int64_t n, int n_keys, int32_t* starts) {
  const int k = (int)(blockIdx.x * 256 + threadIdx.x);
  if (k <= n_keys) starts[k] = first_of(keys, n, (uint32_t)k);
}

// Lists cut into pieces of `most` entries at most, one at least, and places for the
// sums of those with more than one.  One workgroup; of few keys and entries it finds the
// lists itself (FIND), which saves a launch: 9 us for 1024 keys of 65536 entries, 20 for
// 2000 of 630000, 12 with the kernel above.
constexpr int kFewKeys = 1024;
constexpr int64_t kFewEntries = 65536;
template <bool FIND>
__global__ __launch_bounds__(1024) void block_pieces_kernel(const uint32_t* keys, int64_t entries, const int32_t* starts,
                                                            int n_keys, int most, int4* pieces, int2* sums,
                                                            int32_t* n_pieces) {
  __shared__ uint32_t s_total[2][16];
  __shared__ int32_t s_first[FIND ? kFewKeys + 1 : 1];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  if constexpr (FIND) {
    for (int k = tid; k <= n_keys; k += 1024) s_first[k] = first_of(keys, entries, (uint32_t)k);
    __syncthreads();
  }
  auto first = [&](int k) { return FIND ? s_first[FIND ? k : 0] : starts[k]; };
  uint32_t at = 0, place = 0;
  for (int k0 = 0; k0 < n_keys; k0 += 1024) {
    const int k = k0 + tid;
    const int from = k < n_keys ? first(k) : 0, to = k < n_keys ? first(k + 1) : 0;
    const uint32_t length = to > from ? (uint32_t)(to - from) : 0u;
    const uint32_t n = k < n_keys ? (length > 0u ? (length + (uint32_t)most - 1u) / (uint32_t)most : 1u) : 0u;
    const uint32_t shared = n > 1 ? n : 0u;
    const uint32_t upto = wave_sum_scan(n), upto2 = wave_sum_scan(shared);
    if (lane == 63) {
      s_total[0][w] = upto;
      s_total[1][w] = upto2;
    }
    __syncthreads();
    uint32_t mine = at + upto - n, mine2 = place + upto2 - shared;
    for (int i = 0; i < 16; ++i) {
      if (i < w) {
        mine += s_total[0][i];
        mine2 += s_total[1][i];
      }
      at += s_total[0][i];
      place += s_total[1][i];
    }
    if (k < n_keys) {
      sums[k] = int2{(int)mine2, (int)shared};
      // (of like length)
      const uint32_t each = (length + n - 1u) / n;
      for (uint32_t i = 0; i < n; ++i) {
        const uint32_t a = i * each < length ? i * each : length, b = length - a < each ? length : a + each;
        pieces[mine + i] = int4{k, from + (int)a, from + (int)b, n > 1 ? (int)(mine2 + i) : -1};
      }
    }
    __syncthreads();
  }
  if (tid == 0) *n_pieces = (int32_t)at;
}

// ---- gradients of keys and values -------------------------------------------------

// 16 keys a wave, KW waves over the keys, RW over the rows.
template <class T, int DP, int BK>
struct KeyShape {
  static constexpr int kWaves = DP * (int)sizeof(T) > 256 ? 4 : 8, kThreads = 64 * kWaves;
  static constexpr int KT = 1, KW = BK / (16 * KT), RW = kWaves / KW;
  static constexpr int kStep = 32 * RW;  // rows a step
  // waves a SIMD: of rows of 128 bytes two workgroups share a compute unit
  static constexpr int kOccupancy = DP * (int)sizeof(T) <= 128 ? 4 : 1;
};

struct KeyPlace {
  int seq, head, first;  // position of the first key
  Sequence sq;
};

// 4 rows' numbers, by a lane's group.
struct RowStats {
  float lse[128], delta[128];
  int pos[128];
};

template <class T, int DP>
__device__ __forceinline__ void careful_key(const GradArgs& a, const KeyPlace& at, const int32_t* order, int64_t rows, int j,
                                         float (&k_sum)[(DP + 63) / 64], float (&v_sum)[(DP + 63) / 64], int lane) {
  const BlockArgs& p = a.b;
  const float c = p.scale * kLog2e;
  constexpr int N = (DP + 63) / 64;
#pragma unroll
  for (int i = 0; i < N; ++i) k_sum[i] = v_sum[i] = 0.0f;
  if (j >= at.sq.keys) return;
  const T* k = static_cast<const T*>(p.k.base) + (at.sq.row0 + j) * p.k.row + at.head * p.k.head;
  const T* v = static_cast<const T*>(p.v.base) + (at.sq.row0 + j) * p.v.row + at.head * p.v.head;
  for (int64_t r0 = 0; r0 < rows; r0 += 64) {
    const int64_t r = r0 + lane;
    float x = 0.0f, y = 0.0f;
    bool seen = false;
    int64_t row = 0, q_row = 0;
    if (r < rows) {
      const int token = order[r / p.group] / (a.lists * p.top), hq = at.head * p.group + (int)(r % p.group);
      seen = at.sq.keys - at.sq.count + token - at.sq.first >= j;
      row = (int64_t)token * p.heads * p.group + hq;
      q_row = token * p.q_token + hq * p.q_head;
      if (seen) {
        const T* q = static_cast<const T*>(p.q) + q_row;
        const T* g = static_cast<const T*>(a.grad) + row * p.width;
        float s = 0.0f, d = 0.0f;
        for (int i = 0; i < p.width; ++i) {
          s = __builtin_fmaf((float)q[i], (float)k[i], s);
          d = __builtin_fmaf((float)g[i], (float)v[i], d);
        }
        x = __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -a.lse[row] * kLog2e));
        y = x * (d - a.delta[row]);
      }
    }
    for (uint64_t left = __ballot(seen); left != 0; left &= left - 1) {
      const int l = __builtin_ctzll(left);
      const float wx = __shfl(x, l), wy = __shfl(y, l);
      const T* g = static_cast<const T*>(a.grad) + __shfl(row, l) * p.width;
      const T* q = static_cast<const T*>(p.q) + __shfl(q_row, l);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i * 64 + lane < p.width) {
          v_sum[i] = __builtin_fmaf(wx, (float)g[i * 64 + lane], v_sum[i]);
          k_sum[i] = __builtin_fmaf(wy, (float)q[i * 64 + lane], k_sum[i]);
        }
    }
  }
}

constexpr int kWindow = 1024;  // entries of a piece whose tokens LDS holds at a time

template <class T, int DP, int BK>
__global__ __launch_bounds__((KeyShape<T, DP, BK>::kThreads), (KeyShape<T, DP, BK>::kOccupancy)) void block_key_grad_kernel(const GradArgs a) {
  using R = Rows<T, DP>;
  using S = KeyShape<T, DP, BK>;
  constexpr int KT = S::KT, KW = S::KW, RW = S::RW, STEP = S::kStep, F = R::kFrags;
  constexpr int WAVES = S::kWaves, THREADS = S::kThreads;
  constexpr int kSlot = STEP * R::kRow, P = R::kUnit / 16;
  constexpr int kJoin = (RW - 1) * KW * KT * 16 * DP * 4 * 2;
  constexpr int kMemory = 4 * kSlot > kJoin ? 4 * kSlot : kJoin;
  __shared__ alignas(1024) uint8_t s_mem[kMemory];
  __shared__ RowStats s_stats[2];
  __shared__ int32_t s_token[kWindow];
  __shared__ int s_bad;
  const BlockArgs& p = a.b;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = w % KW, rw = w / KW;
  const int lg_block = p.lg_groups + 4, parts = p.seqs.block / BK, shared = p.heads / a.lists;
  int64_t at = xcd_range_block(blockIdx.x, gridDim.x);
  const int part = (int)(at % parts);
  at /= parts;
  const int copy = (int)(at % shared);
  at /= shared;
  if (at >= *a.n_pieces) return;
  const int4 piece = a.pieces[at];
  KeyPlace o;
  const int list = piece.x / a.key_blocks, number = piece.x - list * a.key_blocks;
  o.head = a.lists == 1 ? copy : list;
  o.seq = -1;
  for (int64_t b0 = 0; b0 < p.seqs.n_seqs; b0 += 64) {
    bool mine = false;
    if (b0 + lane < p.seqs.n_seqs) {
      const Sequence q = sequence_at(p.seqs, (int)b0 + lane);
      const int f = first_block(p.seqs, (int)b0 + lane, lg_block);
      mine = number >= f && number - f < ((q.keys + p.seqs.block - 1) >> lg_block);
    }
    const uint64_t m = __ballot(mine);
    if (m != 0) {
      o.seq = (int)b0 + __builtin_ctzll(m);
      break;
    }
  }
  if (o.seq < 0) return;  // a number that no sequence's block has
  o.sq = sequence_of(p.seqs, o.seq);
  o.first = ((number - first_block(p.seqs, o.seq, lg_block)) << lg_block) + part * BK;
  const int entries = piece.z - piece.y;
  if (tid == 0) s_bad = 0;

  // the wave's keys and values, as second operands
  typename R::frag kf[KT][F], vf[KT][F];
#pragma unroll
  for (int n = 0; n < KT; ++n) {
    const int j = o.first + (kw * KT + n) * 16 + (lane & 15);
    const bool in = j < o.sq.keys;
    load_row<T, DP>(static_cast<const T*>(p.k.base) + (o.sq.row0 + j) * p.k.row + o.head * p.k.head, in, p.width, lane,
                    kf[n]);
    load_row<T, DP>(static_cast<const T*>(p.v.base) + (o.sq.row0 + j) * p.v.row + o.head * p.v.head, in, p.width, lane,
                    vf[n]);
  }
  f32x4 dk[KT][DP / 16], dv[KT][DP / 16];
#pragma unroll
  for (int n = 0; n < KT; ++n)
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) dk[n][dt] = dv[n][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  float factor[KT];  // of the lane's keys
#pragma unroll
  for (int n = 0; n < KT; ++n) factor[n] = kFactored<T> ? kFirstFactor : 1.0f;
  const float c = p.scale * kLog2e;
  const int offset = o.sq.keys - o.sq.count - o.sq.first;  // of positions from tokens
  const int used = (p.width + 15) / 16;
  int rows = 0;  // of a window
  auto place = [&](int r, int& token, int& hq) {
    const int e = (int)__umulhi((uint32_t)r, a.per_group);
    const int entry = p.group == 1 ? r : e;
    token = s_token[entry];
    hq = o.head * p.group + r - entry * p.group;
  };
  float n_lse = 0.0f, n_delta = 0.0f;
  int n_pos = 0;
  auto issue = [&](int s) {
    constexpr int kLoads = kSlot / 1024 / WAVES;
    static_assert(kSlot % (1024 * WAVES) == 0, "whole loads a wave");
    const uint32_t qb = lds_address(s_mem) + (uint32_t)((s & 1) * 2 * kSlot), gb = qb + kSlot;
    const int lr = R::lane_row(lane), pos = lane % R::kPieces;
#pragma unroll
    for (int n = 0; n < kLoads; ++n) {
      const int r0 = (w * kLoads + n) * R::kAtOnce;
      const int at_step = s * STEP + r0 + lr;
      int token, hq;
      place(at_step < rows ? at_step : rows - 1, token, hq);  // (past the end: some row of the list, left out below)
      const int piece16 = pos ^ R::swizzle((r0 + lr) & 15);
      const bool in = piece16 * 16 < p.width * (int)sizeof(T);
      const int64_t d = in ? piece16 * (16 / (int)sizeof(T)) : 0;
      const T* q = static_cast<const T*>(p.q) + token * p.q_token + hq * p.q_head + d;
      const T* g = static_cast<const T*>(a.grad) + ((int64_t)token * p.heads * p.group + hq) * p.width + d;
      lds_dma_at((uint32_t)__builtin_amdgcn_readfirstlane((int)(qb + (uint32_t)r0 * R::kRow)), q);
      lds_dma_at((uint32_t)__builtin_amdgcn_readfirstlane((int)(gb + (uint32_t)r0 * R::kRow)), g);
    }
    if (tid < STEP) {
      const int r = s * STEP + tid;
      int token, hq;
      place(r < rows ? r : rows - 1, token, hq);
      const int64_t row = (int64_t)token * p.heads * p.group + hq;
      n_lse = a.lse[row];
      n_delta = a.delta[row];
      n_pos = r < rows ? token + offset : INT32_MIN;
    }
  };
  for (int e0 = 0; e0 < entries; e0 += kWindow) {
    const int here = entries - e0 < kWindow ? entries - e0 : kWindow;
    wait_reads();  // (the window before has been read)
    __syncthreads();
    for (int e = tid; e < here; e += THREADS) s_token[e] = a.order[piece.y + e0 + e] / (a.lists * p.top);
    __syncthreads();
    rows = here * p.group;
    const int steps = (rows + STEP - 1) / STEP;
    issue(0);
    for (int s = 0; s < steps; ++s) {
      RowStats& stats = s_stats[s & 1];
      if (tid < STEP) {
        stats.lse[tid] = n_lse * kLog2e - kWeightLift<T>;
        stats.delta[tid] = n_delta;
        stats.pos[tid] = n_pos;
      }
      wait_loads<0>();
      wait_reads();
      barrier();
      if (s + 1 < steps) issue(s + 1);
      const uint32_t qb = lds_address(s_mem) + (uint32_t)((s & 1) * 2 * kSlot) + (uint32_t)(rw * 32 * R::kRow);
      const uint32_t gb = qb + kSlot;
      f32x4 x[2][KT], y[2][KT];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < KT; ++n) x[m][n] = y[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < F; ++ks) {
        if (leave_out<T>(ks, used)) break;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          const auto q = R::across(qb, m * 16, ks, lane);
          const auto g = R::across(gb, m * 16, ks, lane);
#pragma unroll
          for (int n = 0; n < KT; ++n) {
            x[m][n] = Mma<T>::run(q, kf[n][ks], x[m][n]);
            y[m][n] = Mma<T>::run(g, vf[n][ks], y[m][n]);
          }
        }
      }
      typename R::Halves pf[KT][2 / P], sf[KT][2 / P];
      f32x4 wx[KT][2], wy[KT][2];
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int r0 = rw * 32 + m * 16 + (lane >> 4) * 4;
        const f32x4 lse = *reinterpret_cast<const f32x4*>(&stats.lse[r0]);
        const f32x4 delta = *reinterpret_cast<const f32x4*>(&stats.delta[r0]);
        const int4 pos = *reinterpret_cast<const int4*>(&stats.pos[r0]);
        const int row_pos[4] = {pos.x, pos.y, pos.z, pos.w};
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          const int j = o.first + (kw * KT + n) * 16 + (lane & 15);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            // (keys behind the last one are behind every position, rows past the list's
            // end before every key)
            const bool in = j <= row_pos[r];
            const float u = __builtin_amdgcn_exp2f(__builtin_fmaf(x[m][n][r], c, -lse[r]));
            const float v = u * (y[m][n][r] - delta[r]);
            wx[n][m][r] = in ? u : 0.0f;
            wy[n][m][r] = in ? v : 0.0f;
          }
        }
      }
      if constexpr (kFactored<T>) {
#pragma unroll
        for (int n = 0; n < KT; ++n) {
          float most = 0.0f;
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) most = fmaxf(most, fabsf(wy[n][m][r]));
          follow(across_max(most), factor[n], dk[n]);
#pragma unroll
          for (int m = 0; m < 2; ++m) wy[n][m] *= factor[n];
        }
      }
      // P and dS in two parts of the values' type
#pragma unroll
      for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int u = 0; u < 2 / P; ++u) {
          pf[n][u] = R::halves(&wx[n][u * P]);
          sf[n][u] = R::halves(&wy[n][u * P]);
        }
#pragma unroll
      for (int u = 0; u < 2 / P; ++u)
#pragma unroll
        for (int dt = 0; dt < DP / 16; ++dt) {
          if (leave_out<T>(dt, used)) break;
          const auto g = R::down(gb, u * R::kUnit, dt, lane);
          const auto q = R::down(qb, u * R::kUnit, dt, lane);
#pragma unroll
          for (int i = 0; i < R::kParts; ++i)
#pragma unroll
            for (int n = 0; n < KT; ++n) {
              dv[n][dt] = Mma<T>::run(g, pf[n][u].part[i], dv[n][dt]);
              dk[n][dt] = Mma<T>::run(q, sf[n][u].part[i], dk[n][dt]);
            }
        }
    }
  }
  if constexpr (kFactored<T>) {
    constexpr float kDown = 0x1p-15f;
    static_assert(kWeightLift<T> == 15.0f);
#pragma unroll
    for (int n = 0; n < KT; ++n)
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt) {
        dk[n][dt] *= kDown / factor[n];
        dv[n][dt] *= kDown;
      }
  }
  // sums of the waves over the rows
  wait_reads();
  __syncthreads();
  float* s_join = reinterpret_cast<float*>(s_mem);
  constexpr int kWaveSums = KT * 16 * DP * 2;
  if (rw > 0) {
    float* mine = s_join + ((rw - 1) * KW + kw) * kWaveSums;
#pragma unroll
    for (int n = 0; n < KT; ++n)
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt) {
        float* e = mine + ((n * (DP / 16) + dt) * 2) * 256 + lane * 4;
        *reinterpret_cast<f32x4*>(e) = dk[n][dt];
        *reinterpret_cast<f32x4*>(e + 256) = dv[n][dt];
      }
  }
  __syncthreads();
  bool bad = false;
  if (rw == 0) {
#pragma unroll
    for (int i = 1; i < RW; ++i) {
      const float* other = s_join + ((i - 1) * KW + kw) * kWaveSums;
#pragma unroll
      for (int n = 0; n < KT; ++n)
#pragma unroll
        for (int dt = 0; dt < DP / 16; ++dt) {
          const float* e = other + ((n * (DP / 16) + dt) * 2) * 256 + lane * 4;
          dk[n][dt] += *reinterpret_cast<const f32x4*>(e);
          dv[n][dt] += *reinterpret_cast<const f32x4*>(e + 256);
        }
    }
#pragma unroll
    for (int n = 0; n < KT; ++n)
#pragma unroll
      for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r) bad |= !__builtin_isfinite(dk[n][dt][r]) || !__builtin_isfinite(dv[n][dt][r]);
    if (__ballot(bad) != 0 && lane == 0) s_bad = 1;
  }
  __syncthreads();
  const bool again = s_bad != 0;
  const int64_t place_of = piece.w >= 0 ? ((int64_t)piece.w * shared + copy) * p.seqs.block + part * BK : 0;
  if (!again) {
    if (rw == 0) {
#pragma unroll
      for (int n = 0; n < KT; ++n) {
        const int jj = (kw * KT + n) * 16 + (lane & 15), j = o.first + jj;
        if (piece.w >= 0) {
          float* sums = a.parts + (place_of + jj) * 2 * DP;
#pragma unroll
          for (int dt = 0; dt < DP / 16; ++dt) {
            *reinterpret_cast<f32x4*>(sums + dt * 16 + (lane >> 4) * 4) = dk[n][dt] * p.scale;
            *reinterpret_cast<f32x4*>(sums + DP + dt * 16 + (lane >> 4) * 4) = dv[n][dt];
          }
        } else if (j < o.sq.keys) {
          const int64_t row = ((o.sq.row0 + j) * p.heads + o.head) * p.width;
          store_row<T, DP>(static_cast<T*>(a.dk) + row, dk[n], p.scale, p.width, lane);
          store_row<T, DP>(static_cast<T*>(a.dv) + row, dv[n], 1.0f, p.width, lane);
        }
      }
    }
    return;
  }
  // a sum that is not finite: each key by itself, without products of what it is not seen by
  for (int jj = w; jj < BK; jj += WAVES) {
    const int j = o.first + jj;
    constexpr int N = (DP + 63) / 64;
    float k_sum[N], v_sum[N];
    careful_key<T, DP>(a, o, a.order + piece.y, (int64_t)entries * p.group, j, k_sum, v_sum, lane);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = i * 64 + lane;
      if (piece.w >= 0) {
        float* sums = a.parts + (place_of + jj) * 2 * DP;
        sums[d] = k_sum[i] * p.scale;
        sums[DP + d] = v_sum[i];
      } else if (j < o.sq.keys && d < p.width) {
        const int64_t row = ((o.sq.row0 + j) * p.heads + o.head) * p.width;
        static_cast<T*>(a.dk)[row + d] = (T)(k_sum[i] * p.scale);
        static_cast<T*>(a.dv)[row + d] = (T)v_sum[i];
      }
    }
  }
}

// Sums of a block's pieces, in order: a workgroup 16 keys of one.  The first `again`
// workgroups take the queries' rows that are not finite.
template <class T, int DP>
__global__ __launch_bounds__(256) void block_key_join_kernel(const GradArgs a, int64_t again) {
  const BlockArgs& p = a.b;
  const int lane = threadIdx.x & 63, lg_block = p.lg_groups + 4, shared = p.heads / a.lists;
  int64_t at = row_block() - again;
  if (at < 0) {
    queries_again<T, DP>(a, (uint32_t)(at + again), __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), 4, lane);
    return;
  }
  if (a.dk == nullptr) return;
  const int group = (int)(at & ((1 << p.lg_groups) - 1));
  at >>= p.lg_groups;
  const int copy = (int)(at % shared), key = (int)(at / shared);
  if (key >= a.lists * a.key_blocks) return;
  const int2 sums = a.sums[key];
  if (sums.y == 0) return;
  const int list = key / a.key_blocks, number = key - list * a.key_blocks;
  const int head = a.lists == 1 ? copy : list;
  for (int64_t b0 = 0; b0 < p.seqs.n_seqs; b0 += 64) {
    bool mine = false;
    if (b0 + lane < p.seqs.n_seqs) {
      const Sequence q = sequence_at(p.seqs, (int)b0 + lane);
      const int f = first_block(p.seqs, (int)b0 + lane, lg_block);
      mine = number >= f && number - f < ((q.keys + p.seqs.block - 1) >> lg_block);
    }
    const uint64_t m = __ballot(mine);
    if (m == 0) continue;
    const int seq = (int)b0 + __builtin_ctzll(m);
    const Sequence sq = sequence_at(p.seqs, seq);
    const int first = ((number - first_block(p.seqs, seq, lg_block)) << lg_block) + group * 16;
    for (int e = threadIdx.x; e < 16 * (DP / 4) * 2; e += 256) {
      const int d = e % (DP / 4) * 4, which = e / (DP / 4) % 2, jj = e / (DP / 4) / 2, j = first + jj;
      if (d >= p.width || j >= sq.keys) continue;
      f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int i = 0; i < sums.y; ++i)
        sum += *reinterpret_cast<const f32x4*>(
            a.parts + ((((int64_t)(sums.x + i) * shared + copy) * p.seqs.block + group * 16 + jj) * 2 + which) * DP + d);
      T out[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) out[r] = (T)sum[r];
      const int64_t row = ((sq.row0 + j) * p.heads + head) * p.width + d;
      __builtin_memcpy(static_cast<T*>(which ? a.dv : a.dk) + row, out, sizeof out);
    }
    return;
  }
}

// ---- host -------------------------------------------------------------------------

// Keys of a workgroup of the keys' gradient.
constexpr int keys_at_once(int block) { return block == 32 ? 32 : 64; }

struct GradPlan {
  int64_t entries;  // of the selection
  int64_t key_blocks, n_keys;
  int64_t pieces, places;  // at most
  int most;                // entries a piece
  int per;                 // tokens a workgroup of the queries' gradient
  int64_t tiles;
  size_t again, sort, keys, sorted, order, starts, list, sums, count, delta, parts, bytes;
};
GradPlan grad_plan(int val_t, const fs_block_seqs& s, int heads, int group, int lists, int width, int top) {
  GradPlan l{};
  const int64_t tokens = s.n_tokens, rows = s.n_rows, n_seqs = s.n_seqs;
  const int block = s.block;
  l.entries = tokens * lists * top;
  l.key_blocks = rows / block + n_seqs + 1;
  l.n_keys = l.key_blocks * lists;
  // Pieces enough for a few rounds of the chip, and long enough that their sums cost little;
  // so many at most, whatever the sizes: their sums are the workspace's largest part.  us
  // with 2048 pieces, with 1024 and with 4096: 8192 tokens of 4 x 8 heads 1563, 1587, 1643;
  // 2048 of 4 x 16 594, 557, 727; 4 x 2048 of 8 x 1 370, 348, 366; f32, 8192 of 4 x 8 10787,
  // 11587, 10417.  With 512 rows a piece at least, 256 and 1024: 1024 tokens of 4 x 4 heads
  // 148, 162, 143, f32 621, 601, 699.
  const int64_t shared = heads / lists, parts = std::max(1, block / 64);
  const int64_t most = std::max<int64_t>(ceil_div(l.entries * shared * parts, 2048), ceil_div(512, group));
  l.most = (int)std::min<int64_t>(most, INT32_MAX);
  l.pieces = l.entries / l.most + l.n_keys;
  l.places = 2 * (l.entries / l.most) + 2;
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  size_t at = 0;
  auto take = [&](size_t n) {
    const size_t a = at;
    at += up(n);
    return a;
  };
  const int dp = width <= 64 ? 64 : width <= 128 ? 128 : 256;
  const int readers = query_readers(dp * (val_t == FS_F32 ? 4 : 2));
  l.per = readers * 16 / group;
  l.tiles = block_tiles(s, l.per);
  l.again = take((size_t)(l.tiles * heads) * readers * 4);
  l.sort = take(select_sort_bytes(l.entries, l.n_keys));
  l.keys = take((size_t)l.entries * 4);
  l.sorted = take((size_t)l.entries * 4);
  l.order = take((size_t)l.entries * 4);
  l.starts = take((size_t)(l.n_keys + 1) * 4);
  l.list = take((size_t)l.pieces * 16);
  l.sums = take((size_t)l.n_keys * 8);
  l.count = take(4);
  l.delta = take((size_t)tokens * heads * group * 4);
  l.parts = take((size_t)(l.places * shared) * block * 2 * dp * 4);
  l.bytes = at;
  return l;
}

int grad_fault(const char* who, int val_t, const fs_block_seqs* seqs, int heads, int group, int width, int lists,
               int top) {
  if (const int rc = block_sizes_fault(who, val_t, seqs, heads, group, width)) return rc;
  if (seqs->pages != nullptr) return fail(FS_E_INVALID, std::string(who) + ": keys of a cache have no gradient");
  if (top < 1 || top > kMostTop) return fail(FS_E_INVALID, std::string(who) + ": top out of range");
  const int row = (width <= 64 ? 64 : width <= 128 ? 128 : 256) * (val_t == FS_F32 ? 4 : 2);
  if (group > query_readers(row) * 16) return fail(FS_E_INVALID, std::string(who) + ": heads out of range for this width");
  if (lists != 1 && lists != heads) return fail(FS_E_INVALID, std::string(who) + ": lists is 1 or the heads");
  const int64_t blocks = (seqs->n_rows / seqs->block + seqs->n_seqs + 1) * lists;
  if (seqs->n_tokens * lists * top > INT32_MAX || blocks >= INT32_MAX)
    return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
  // (here, before anything is launched)
  const GradPlan l = grad_plan(val_t, *seqs, heads, group, lists, width, top);
  if (l.tiles * heads > kMostWorkgroups ||
      l.pieces * (heads / lists) * (seqs->block / keys_at_once(seqs->block)) > kMostWorkgroups)
    return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
  return FS_OK;
}

}  // namespace
}  // namespace fs

extern "C" size_t fs_block_attention_grad_workspace_bytes(int val_t, const fs_block_seqs* seqs, int heads, int group,
                                                          int width, int lists, int top) {
  using namespace fs;
  if (grad_fault("", val_t, seqs, heads, group, width, lists, top) != FS_OK) return 0;
  return grad_plan(val_t, *seqs, heads, group, lists, width, top).bytes;
}

extern "C" int fs_block_attention_grad(int val_t, const fs_block_seqs* seqs, int heads, int group, int width, int lists,
                                       int top, const void* grad, const void* q, int64_t q_token, int64_t q_head,
                                       const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                                       int64_t v_head, const int32_t* blocks, int64_t b_token, int64_t b_head,
                                       double scale, const void* out, const float* lse, void* dq, void* dk, void* dv,
                                       void* ws, size_t ws_bytes, hipStream_t stream) {
  using namespace fs;
  const char* who = "fs_block_attention_grad";
  if (const int rc = grad_fault(who, val_t, seqs, heads, group, width, lists, top)) return rc;
  const int64_t size = val_t == FS_F32 ? 4 : 2, tokens = seqs->n_tokens;
  if (tokens == 0 && seqs->n_rows == 0) return FS_OK;
  const bool queries = tokens > 0 && dq != nullptr, of_keys = seqs->n_rows > 0 && dk != nullptr;
  if ((tokens > 0 && (!grad || !q || !blocks || !out || !lse)) || !k || !v || (seqs->n_rows > 0 && !dk != !dv) ||
      (!queries && !of_keys) || q_token < 0 || q_head < 0 || b_token < 0 || b_head < 0)
    return fail(FS_E_INVALID, std::string(who) + ": bad pointer or stride");
  if (!block_rows_fit(k, 0, k_row, k_head, size) || !block_rows_fit(v, 0, v_row, v_head, size) ||
      (((int64_t)(uintptr_t)q | (int64_t)(uintptr_t)grad | q_token * size | q_head * size) & 15) != 0)
    return fail(FS_E_INVALID, std::string(who) + ": queries, keys, values and grad need rows at multiples of 16 bytes");
  if (!(scale > 0.0) || !(scale < 1e30)) return fail(FS_E_INVALID, std::string(who) + ": scale must be positive");
  const GradPlan l = grad_plan(val_t, *seqs, heads, group, lists, width, top);
  if (ws == nullptr || ws_bytes < l.bytes) return fail(FS_E_WORKSPACE, std::string(who) + ": workspace too small");
  uint8_t* m = static_cast<uint8_t*>(ws);
  GradArgs a{};
  BlockArgs& p = a.b;
  p.again = reinterpret_cast<uint32_t*>(m + l.again);
  p.seqs = *seqs;
  p.k = RowLayout{k, 0, k_row, k_head};
  p.v = RowLayout{v, 0, v_row, v_head};
  p.q = q;
  p.q_token = q_token;
  p.q_head = q_head;
  p.out = dq;
  p.blocks = blocks;
  p.b_token = b_token;
  p.b_head = b_head;
  p.top = top;
  p.heads = heads;
  p.group = group;
  p.width = width;
  p.lg_groups = __builtin_ctz((unsigned)seqs->block) - 4;
  p.scale = (float)scale;
  a.grad = grad;
  a.o = out;
  a.lse = lse;
  a.delta = reinterpret_cast<float*>(m + l.delta);
  a.order = reinterpret_cast<int32_t*>(m + l.order);
  a.pieces = reinterpret_cast<int4*>(m + l.list);
  a.n_pieces = reinterpret_cast<int32_t*>(m + l.count);
  a.sums = reinterpret_cast<int2*>(m + l.sums);
  a.parts = reinterpret_cast<float*>(m + l.parts);
  a.dk = dk;
  a.dv = dv;
  a.lists = lists;
  a.key_blocks = (int)l.key_blocks;
  a.per_group = group == 1 ? 0u : (uint32_t)((((uint64_t)1 << 32) + group - 1) / group);
  int32_t* keys = reinterpret_cast<int32_t*>(m + l.keys);
  uint32_t* sorted = reinterpret_cast<uint32_t*>(m + l.sorted);
  int32_t* starts = reinterpret_cast<int32_t*>(m + l.starts);

  if (of_keys) {
    const int64_t key_groups = std::min<int64_t>(ceil_div(std::max<int64_t>(tokens, 4), 4), 4096);
    hipLaunchKernelGGL(block_keys_kernel, dim3((uint32_t)key_groups), dim3(256), 0, stream, p, lists, (int)l.key_blocks, keys,
                       static_cast<uint32_t*>(dk), static_cast<uint32_t*>(dv), (int64_t)heads * width * size / 4);
    FS_CHECK_LAUNCH("block_keys_kernel");
    if (l.entries > 0) {
      if (const int rc = select_sort(keys, FS_I32, l.entries, l.n_keys, sorted, reinterpret_cast<int32_t*>(m + l.order),
                                     nullptr, nullptr, m + l.sort, stream, nullptr, 0))
        return rc;
    }
    int4* pieces = const_cast<int4*>(a.pieces);
    int2* sums = const_cast<int2*>(a.sums);
    int32_t* n_pieces = const_cast<int32_t*>(a.n_pieces);
    if (l.n_keys <= kFewKeys && l.entries <= kFewEntries) {
      hipLaunchKernelGGL((block_pieces_kernel<true>), dim3(1), dim3(1024), 0, stream, sorted, l.entries, starts,
                         (int)l.n_keys, l.most, pieces, sums, n_pieces);
    } else {
      hipLaunchKernelGGL(block_lists_kernel, dim3((uint32_t)ceil_div(l.n_keys + 1, 256)), dim3(256), 0, stream, sorted,
                         l.entries, (int)l.n_keys, starts);
      FS_CHECK_LAUNCH("block_lists_kernel");
      hipLaunchKernelGGL((block_pieces_kernel<false>), dim3(1), dim3(1024), 0, stream, sorted, l.entries, starts,
                         (int)l.n_keys, l.most, pieces, sums, n_pieces);
    }
    FS_CHECK_LAUNCH("block_pieces_kernel");
  }
  return with_block_width(val_t, width, who, [&](auto val, auto dp) -> int {
    using T = decltype(val);
    constexpr int DP = decltype(dp)::value;
    if (tokens > 0) {
      p.tiles = l.tiles;
      p.per = l.per;
      const dim3 grid((uint32_t)(p.tiles * heads));
      hipLaunchKernelGGL((block_query_grad_kernel<T, DP>), grid, dim3(QueryGradShape<T, DP>::kThreads), 0, stream, a);
      FS_CHECK_MAIN_LAUNCH("block_query_grad_kernel");
    }
    const int64_t shared = of_keys ? heads / lists : 0;
    auto keys_of = [&](auto bk) -> int {
      constexpr int BK = decltype(bk)::value;
      const int64_t groups = l.pieces * shared * (seqs->block / BK);
      hipLaunchKernelGGL((block_key_grad_kernel<T, DP, BK>), dim3((uint32_t)groups), dim3(KeyShape<T, DP, BK>::kThreads), 0,
                         stream, a);
      FS_CHECK_LAUNCH("block_key_grad_kernel");
      return FS_OK;
    };
    if (of_keys) {
      const int rc = keys_at_once(seqs->block) == 32 ? keys_of(std::integral_constant<int, 32>{})
                                                     : keys_of(std::integral_constant<int, 64>{});
      if (rc != FS_OK) return rc;
    }
    const int64_t again = queries ? p.tiles * heads : 0;
    hipLaunchKernelGGL((block_key_join_kernel<T, DP>), row_grid(again + ((l.n_keys * shared) << p.lg_groups)), dim3(256), 0,
                       stream, a, again);
    FS_CHECK_LAUNCH("block_key_join_kernel");
    return FS_OK;
  });
}
