// block_attention.hip — attention over the blocks of keys that each query selects.
//
//   out[t, h] = sum over j of softmax_j(scale <q[t, h], k[j]>) v[j]
// over the keys j of the blocks that blocks[t, h / group] names, up to the query's
// own position: a product of dense matrices sampled where the selection is, a softmax
// along its rows, and the sparse matrix so made times the values, in one pass with the
// running maximum and sum of each row.  A block named twice counts once.
//
// Weights of 16-bit values go through the matrix cores in two parts (Rows::halves), so that
// results are off by their own rounding alone.  In one part, 8 bits of bfloat16, errors are
// 1.4 times as large, and 16384 tokens take 1631 us instead of 1729.
//
// Many queries (block_walk.hpp): 16384 tokens of 4 x 16 heads of 128, 16 blocks of 64
// keys, bf16 1729 us, 299 TFLOP/s; 4 x 512 tokens of 4 x 8 heads over 16384 keys in pages
// of 16, 32 blocks, f16 443 us.  The 12 tokens (24 of groups of 8) of a workgroup select 79
// (172) different blocks of 256, so a step has 2.4 (3.6) of its twelve readers, and what
// bounds it is a step's way through a slot (load, announcement, reading): 1240 (1570)
// cycles, where a reader's matrix instructions take 384.  Those are busy for 18% (16%) of
// the cycles, LDS for 26% (21%); waves wait for half of theirs.  Of rows of 128 16-bit
// values the kernel fills its 128 registers (float16 spills two, outside the steps, and
// both 47 scalars).  Few queries: 64 tokens of 8 x 8 heads over as many caches 61 us, 262
// MB at 4.3 TB/s.
#include "block_walk.hpp"

namespace fs {
namespace {

// A wave's 16 rows: a lane has a part of row lane % 16.
template <class T, int DP>
struct Online {
  typename Mma<T>::frag q[Rows<T, DP>::kFrags];
  f32x4 o[DP / 16];  // columns 16 dt + 4 g ..
  float m, l;        // maximum in powers of two, and the lane's own part of the sum
};

template <class T, int DP>
__device__ inline void start(Online<T, DP>& st) {
  st.m = -INFINITY;
  st.l = 0.0f;
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt) st.o[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
}

// The maximum follows the scores only where it grows by more than this, in powers of
// two: weights are 2^8 at most, and rescaling is left out of most steps.
constexpr float kSlack = 8.0f;
// float16's weights times 2^7, so up to 2^15: its last step is then 2^-32 of the weight
// of the largest score instead of 2^-25, and the small weights of 131072 keys, the most
// that a query selects, are not lost together.  Their sum has the factor too.
template <class T>
constexpr float kLift = std::is_same_v<T, _Float16> ? 7.0f : 0.0f;

// One step's keys and values.
template <class T, int DP, int AHEAD, class Wait, class Done>
__device__ inline void attend(Online<T, DP>& st, uint32_t kb, uint32_t vb, bool sel, int now, bool some,
                              bool edge, uint32_t missing, const RowOf& row, float c, int used, int lane, Wait values,
                              Done done) {
  using R = Rows<T, DP>;
  constexpr int G = R::kGroups, P = R::kUnit / 16;
  f32x4 s[G];
#pragma unroll
  for (int gr = 0; gr < G; ++gr) s[gr] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  products<T, DP, AHEAD>(kb, st.q, s, used, lane);
  values();  // are there: they are read while the weights are computed
  Columns<T, DP, AHEAD> v;
  v.read(vb, 0, used, lane);
  if (edge) {
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      const int last = (missing >> gr) & 1u ? -1 : row.pos - now - 16 * gr - 4 * (lane >> 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) s[gr][r] = r <= last ? s[gr][r] : -INFINITY;
    }
  }
  if (some) {
#pragma unroll
    for (int gr = 0; gr < G; ++gr)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[gr][r] = sel ? s[gr][r] : -INFINITY;
  }
  float most = -INFINITY;
#pragma unroll
  for (int gr = 0; gr < G; ++gr)
#pragma unroll
    for (int r = 0; r < 4; ++r) most = fmaxf(most, s[gr][r]);
  most = across_max(most) * c;
  if (__ballot(most > st.m + kSlack) != 0) {
    // (a row without keys yet: its maximum stays at minus infinity, its sums are zero)
    const float m = fmaxf(st.m, most);
    const float by = __builtin_amdgcn_exp2f(st.m - (m == -INFINITY ? 0.0f : m));
    st.l *= by;
#pragma unroll
    for (int dt = 0; dt < DP / 16; ++dt) st.o[dt] *= by;
    st.m = m;
  }
  const float base = (st.m == -INFINITY ? 0.0f : st.m) - kLift<T>;
  float sum = 0.0f;
#pragma unroll
  for (int gr = 0; gr < G; ++gr)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[gr][r], c, -base));
      sum += x;
      s[gr][r] = x;
    }
  st.l += sum;
  // weights in two parts of the values' type: together off by 2^-16 (float16: 2^-22) of each
  typename R::Halves w[G / P];
#pragma unroll
  for (int u = 0; u < G / P; ++u) w[u] = R::halves(&s[u * P]);
  v.add(vb, w, st.o, used, lane, done);
}

// One row by a wave, key after key, without products of what is left out: a weight
// of zero times a value that is not finite would be NaN.  Taken where a result is
// not finite, whoever's it is, and where a sum of weights is zero: of a row without keys,
// which is zero, or of one whose scores are all minus infinity, which is not a number.
template <class T, int DP>
__device__ __forceinline__ void careful_row(const BlockArgs& p, const Sequence& sq, int seq, int64_t token, int head,
                                         int in_group, int pos, int lane) {
  const int hq = head * p.group + in_group, block = p.seqs.block, lg = p.lg_groups + 4;
  const T* q = static_cast<const T*>(p.q) + token * p.q_token + (int64_t)hq * p.q_head;
  const int32_t* ids = p.blocks + token * p.b_token + (int64_t)head * p.b_head;
  const float c = p.scale * kLog2e;
  bool any = false;  // key is seen
  float m = -INFINITY, l = 0.0f, o[(DP + 63) / 64];
#pragma unroll
  for (int i = 0; i < (DP + 63) / 64; ++i) o[i] = 0.0f;
  for (int pass = 0; pass < 2; ++pass) {
    for (int e = 0; e < p.top; ++e) {
      const int id = ids[e];
      bool use = id >= 0 && id <= (pos >> lg);
      for (int b = 0; use && b < e; ++b) use = ids[b] != id;
      if (!use) continue;
      for (int j0 = 0; j0 < block; j0 += 64) {
        const int j = id * block + j0 + lane;
        bool seen = j0 + lane < block && j <= pos && j < sq.keys;
        float s = -INFINITY;
        if (seen) {
          const T* k = key_rows<T>(p.seqs, sq, seq, p.k, head, j & ~15);
          seen = k != nullptr;
          if (seen) {
            k += (int64_t)(j & 15) * p.k.row;
            s = 0.0f;
            for (int d = 0; d < p.width; ++d) s = __builtin_fmaf((float)q[d], (float)k[d], s);
          }
        }
        if (pass == 0) {
          any |= __ballot(seen) != 0;
          m = fmaxf(m, s);
          continue;
        }
        const float w = seen ? __builtin_amdgcn_exp2f(__builtin_fmaf(s, c, -m)) : 0.0f;
        l += w;
        for (uint64_t left = __ballot(seen); left != 0; left &= left - 1) {
          const int at = __builtin_ctzll(left), jj = id * block + j0 + at;
          const float weight = __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(w), at));
          const T* v = key_rows<T>(p.seqs, sq, seq, p.v, head, jj & ~15) + (int64_t)(jj & 15) * p.v.row;
#pragma unroll
          for (int i = 0; i < (DP + 63) / 64; ++i)
            if (i * 64 + lane < p.width) o[i] = __builtin_fmaf(weight, (float)v[i * 64 + lane], o[i]);
        }
      }
    }
    if (pass == 0) {
#pragma unroll
      for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
      m = m == -INFINITY ? 0.0f : m * c;
    }
  }
  l = wave_sum(l);
  const int64_t at = token * p.heads * p.group + hq;
  T* out = static_cast<T*>(p.out) + at * p.width;
#pragma unroll
  for (int i = 0; i < (DP + 63) / 64; ++i)
    if (i * 64 + lane < p.width) out[i * 64 + lane] = (T)(any ? o[i] / l : 0.0f);
  if (p.lse != nullptr && lane == 0) p.lse[at] = l == 0.0f ? -INFINITY : (m + __builtin_log2f(l)) * kLn2;
}

// Many queries.  A row whose result is not finite is left to the next kernel.
// Waves that read, by the bytes of a row: with the loaders the 16 waves that have 128
// registers each, or, of rows of 512 bytes, which need 208, the 8 that have 256.
constexpr int many_readers(int row) { return row <= 256 ? 12 : 6; }
template <class T, int DP>
struct ManyShape : WalkShape<T, DP, many_readers(DP * (int)sizeof(T)), (DP * sizeof(T) > 256 ? 2 : 4)> {
  static constexpr int kAhead = 8;
};

template <class T, int DP>
__global__ __launch_bounds__((ManyShape<T, DP>::kThreads)) void block_attention_kernel(const BlockArgs p) {
  using Shape = ManyShape<T, DP>;
  __shared__ typename Shape::Memory mem;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  WalkTile t;
  if (!walk_tile(p, blockIdx.x, lane, t)) return;
  walk_start<Shape>(mem, tid);
  if (w >= Shape::kReaders) {
    walk_loads<T, DP, Shape>(p, t, mem, lds_address(&mem), tid, w, lane);
    return;
  }
  const RowOf row = row_of(p, t, w, lane);
  Online<T, DP> st;
  start(st);
  const int64_t at = (int64_t)(t.token0 + row.token) * p.heads * p.group + t.head * p.group + row.head;
  load_row<T, DP>(static_cast<const T*>(p.q) + (int64_t)(t.token0 + row.token) * p.q_token +
                      (int64_t)(t.head * p.group + row.head) * p.q_head,
                  row.in, p.width, lane, st.q);
  const float c = p.scale * kLog2e;
  const int used = (p.width + 15) / 16;
  walk_blocks<T, DP, Shape, false>(p, t, row, mem, lds_address(&mem), tid, w, lane,
                            [&](int now, bool sel, bool some, bool edge, uint32_t missing, uint32_t kb,
                                uint32_t vb, auto values, auto done) {
                              attend<T, DP, Shape::kAhead>(st, kb, vb, sel, now, some, edge, missing, row, c, used, lane, values,
                                                           done);
                            });
  const float l = across_sum(st.l), by = l > 0.0f ? 1.0f / l : 0.0f;
  bool bad = !__builtin_isfinite(l);
  if (__ballot(l == 0.0f && row.pos >= 0) != 0) {  // (looked up here: a bit kept in the walk costs it 1.5%)
    const int32_t* ids = p.blocks + (int64_t)(t.token0 + row.token) * p.b_token + (int64_t)t.head * p.b_head;
    for (int e = 0; e < p.top; ++e) {
      const int id = ids[e];
      bad |= l == 0.0f && id >= 0 && id <= (row.pos >> (p.lg_groups + 4));
    }
  }
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt)
#pragma unroll
    for (int r = 0; r < 4; ++r) bad |= !__builtin_isfinite(st.o[dt][r]);
  const uint64_t rows = __ballot(bad && row.in);
  if (row.in) {
    store_row<T, DP>(static_cast<T*>(p.out) + at * p.width, st.o, by, p.width, lane);
    if (p.lse != nullptr && lane < 16) p.lse[at] = l > 0.0f ? (st.m - kLift<T> + __builtin_log2f(l)) * kLn2 : -INFINITY;
  }
  if (lane == 0)
    p.again[(int64_t)blockIdx.x * Shape::kReaders + w] = (uint32_t)(rows | rows >> 16 | rows >> 32 | rows >> 48) & 0xffffu;
}

// Those rows, key after key.
template <class T, int DP>
__global__ __launch_bounds__((64 * ManyShape<T, DP>::kReaders)) void block_attention_again_kernel(const BlockArgs p) {
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  WalkTile t;
  uint32_t rows = alike((int)p.again[(int64_t)blockIdx.x * ManyShape<T, DP>::kReaders + w]);
  if (rows == 0 || !walk_tile(p, blockIdx.x, lane, t)) return;
  for (; rows != 0; rows &= rows - 1) {
    const int r = w * 16 + __builtin_ctz(rows), tok = r / p.group;
    careful_row<T, DP>(p, t.sq, t.seq, t.token0 + tok, t.head, r - tok * p.group, t.pos0 + tok, lane);
  }
}

// Few queries: a workgroup takes one token's rows of a group, up to 16 of them, and
// its waves the steps of the token's own blocks in turn, each with keys and values of
// its own in LDS; their states are joined at the end, with `splits` workgroups a
// token those by the next kernel.
constexpr int kFewWaves = 8;

template <class T, int DP>
struct FewShape {
  static constexpr int kWaves = DP * (int)sizeof(T) > 256 ? kFewWaves / 2 : kFewWaves;
};
// (floats of a split's part: maximum and sum of 16 rows, then the rows)
template <int DP>
__host__ __device__ constexpr int part_floats() { return 32 + 16 * DP; }

struct FewPlace {
  int64_t token;
  int head, chunk, split;
};
__device__ inline FewPlace few_place(const BlockArgs& p, int64_t at) {
  FewPlace f;
  f.split = (int)(at % p.splits);
  at /= p.splits;
  const int chunks = (p.group + 15) / 16;
  f.chunk = (int)(at % chunks);
  at /= chunks;
  f.head = (int)(at % p.heads);
  f.token = at / p.heads;
  return f;
}
// Sequence and position of a token; false: of none.
__device__ inline bool token_at(const fs_block_seqs& s, int64_t token, int lane, int& seq, Sequence& sq, int& pos) {
  if (s.q_offsets == nullptr) {
    seq = (int)token;
  } else {
    seq = (int)s.n_seqs;
    for (int64_t b0 = 0; b0 < s.n_seqs; b0 += 64) {
      const int64_t b = b0 + lane;
      bool mine = false;
      if (b < s.n_seqs) {
        const Sequence q = sequence_at(s, (int)b);
        mine = token >= q.first && token < q.first + q.count;
      }
      const uint64_t m = __ballot(mine);
      if (m != 0) {
        seq = (int)b0 + __builtin_ctzll(m);
        break;
      }
    }
  }
  if (seq >= s.n_seqs) return false;
  sq = sequence_of(s, seq);
  pos = sq.keys - sq.count + (int)(token - sq.first);
  return true;
}

// Rows of one token and chunk from the states of `n` waves or splits: part(i) gives
// the i-th one's 16 maxima, 16 sums and 16 rows.
template <class T, int DP, int THREADS, class Part>
__device__ inline void join_rows(const BlockArgs& p, const FewPlace& f, int seq, const Sequence& sq, int pos, int n,
                                 int tid, int* s_bad, Part part) {
  const int rows = p.group - f.chunk * 16 < 16 ? p.group - f.chunk * 16 : 16;
  const int fours = p.width / 4;
  int any = 0;
  if (tid < 16) s_bad[tid] = 0;
  __syncthreads();
  for (int e = tid; e < rows * fours; e += THREADS) {
    const int r = e / fours, d = (e - r * fours) * 4;
    float m = -INFINITY, l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = 0; i < n; ++i) m = fmaxf(m, part(i)[r]);
    const float base = m == -INFINITY ? 0.0f : m;
    for (int i = 0; i < n; ++i) {
      const float* x = part(i);
      const float by = __builtin_amdgcn_exp2f(x[r] - base);
      l = __builtin_fmaf(by, x[16 + r], l);
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = __builtin_fmaf(by, x[32 + r * DP + d + j], o[j]);
    }
    const float by = l > 0.0f ? 1.0f / l : 0.0f;
    bool bad = !__builtin_isfinite(l) || (l == 0.0f && pos >= 0);
    T out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bad |= !__builtin_isfinite(o[j]);
      out[j] = (T)(o[j] * by);
    }
    const int64_t at = (f.token * p.heads + f.head) * p.group + f.chunk * 16 + r;
    __builtin_memcpy(static_cast<T*>(p.out) + at * p.width + d, out, sizeof out);
    if (p.lse != nullptr && d == 0) p.lse[at] = l > 0.0f ? (m - kLift<T> + __builtin_log2f(l)) * kLn2 : -INFINITY;
    if (bad) any = s_bad[r] = 1;
  }
  if (!__syncthreads_or(any)) return;
  __threadfence();  // the rows above are written before they are written again
  __syncthreads();
  for (int r = tid >> 6; r < rows; r += THREADS / 64)
    if (s_bad[r]) careful_row<T, DP>(p, sq, seq, f.token, f.head, f.chunk * 16 + r, pos, tid & 63);
}

template <class T, int DP>
__device__ inline void zero_rows(const BlockArgs& p, const FewPlace& f, int tid, int threads) {
  const int rows = p.group - f.chunk * 16 < 16 ? p.group - f.chunk * 16 : 16;
  const int64_t at = (f.token * p.heads + f.head) * p.group + f.chunk * 16;
  for (int e = tid; e < rows * p.width; e += threads) static_cast<T*>(p.out)[at * p.width + e] = (T)0.0f;
  if (p.lse != nullptr && tid < rows) p.lse[at + tid] = -INFINITY;
}

template <class T, int DP>
__global__ __launch_bounds__((64 * FewShape<T, DP>::kWaves)) void block_attention_few_kernel(const BlockArgs p) {
  using R = Rows<T, DP>;
  constexpr int WAVES = FewShape<T, DP>::kWaves, THREADS = 64 * WAVES;
  static_assert(part_floats<DP>() * 4 <= 2 * R::kBytes, "a wave's state fits where its keys were");
  __shared__ alignas(1024) uint8_t s_kv[WAVES][2][R::kBytes];
  __shared__ int s_ids[kMostTop];
  __shared__ int s_count, s_bad[16];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const FewPlace f = few_place(p, row_block());
  if (f.token >= p.seqs.n_tokens) return;
  int seq, pos;
  Sequence sq;
  if (!token_at(p.seqs, f.token, lane, seq, sq, pos)) {
    if (f.split == 0) zero_rows<T, DP>(p, f, tid, THREADS);
    return;
  }
  const int lg = p.lg_groups + 4;
  const int32_t* ids = p.blocks + f.token * p.b_token + (int64_t)f.head * p.b_head;
  for (int e = tid; e < p.top; e += THREADS) {
    const int id = ids[e];
    s_ids[e] = id >= 0 && id <= (pos >> lg) ? id : -1;
  }
  __syncthreads();
  if (w == 0) {  // those that are blocks, each once
    int count = 0;
    for (int e0 = 0; e0 < p.top; e0 += 64) {
      const int e = e0 + lane, id = e < p.top ? s_ids[e] : -1;
      bool use = id >= 0;
      for (int b = 0; b < count; ++b) use = use && s_ids[b] != id;
      for (int b = 0; b < 63; ++b) {
        const int other = __builtin_amdgcn_readlane(id, b);
        use = use && !(b < lane && other == id);
      }
      const uint64_t m = __ballot(use);
      if (use) s_ids[count + __builtin_popcountll(m & (((uint64_t)1 << lane) - 1))] = id;
      count += __builtin_popcountll(m);
    }
    if (lane == 0) s_count = count;
  }
  RowOf row;
  row.in = f.chunk * 16 + (lane & 15) < p.group;
  row.head = row.in ? f.chunk * 16 + (lane & 15) : 0;
  row.token = 0;
  row.pos = row.in ? pos : -1;
  Online<T, DP> st;
  start(st);
  load_row<T, DP>(static_cast<const T*>(p.q) + f.token * p.q_token + (int64_t)(f.head * p.group + row.head) * p.q_head,
                  row.in, p.width, lane, st.q);
  __syncthreads();
  const int lg_steps = lg - 5, steps = alike(s_count) << lg_steps;
  const float c = p.scale * kLog2e;
  const int used = (p.width + 15) / 16;
  const uint32_t kb = lds_address(s_kv[w][0]), vb = lds_address(s_kv[w][1]);
  KeySource<T, DP> keys, values;
  keys.init(p, p.k, sq, seq, f.head, lane);
  values.init(p, p.v, sq, seq, f.head, lane);
  for (int s = f.split * WAVES + w; s < steps; s += WAVES * p.splits) {
    const int now = (alike(s_ids[s >> lg_steps]) << lg) + (s & ((1 << lg_steps) - 1)) * R::kKeys;
    const bool edge = now + R::kKeys - 1 > pos;
    typename KeySource<T, DP>::Place k_place, v_place;
    keys.find(now, k_place);
    values.find(now, v_place);
    wait_reads();  // the step before has read its rows
    keys.load(kb, k_place, lane);
    values.load(vb, v_place, lane);
    wait_loads<KeySource<T, DP>::kLoads>();
    attend<T, DP, 8>(st, kb, vb, row.in, now, true, edge || k_place.missing != 0, k_place.missing, row, c, used, lane,
                  [] { wait_loads<0>(); }, [] {});
  }
  wait_reads();
  float* mine = reinterpret_cast<float*>(s_kv[w][0]);
  const int r16 = lane & 15;
  const float sum = across_sum(st.l);
  if (lane < 16) {
    mine[r16] = st.m;
    mine[16 + r16] = sum;
  }
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt)
    *reinterpret_cast<f32x4*>(&mine[32 + r16 * DP + dt * 16 + (lane >> 4) * 4]) = st.o[dt];
  __syncthreads();
  if (p.splits == 1) {
    join_rows<T, DP, THREADS>(p, f, seq, sq, pos, WAVES, tid, s_bad,
                              [&](int i) { return reinterpret_cast<const float*>(s_kv[i][0]); });
    return;
  }
  // joined over the waves, into the split's part
  float* part = p.parts + row_block() * part_floats<DP>();
  for (int e = tid; e < 16 * (DP / 4); e += THREADS) {
    const int r = e / (DP / 4), d = e % (DP / 4) * 4;
    float m = -INFINITY, l = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < WAVES; ++i) m = fmaxf(m, reinterpret_cast<const float*>(s_kv[i][0])[r]);
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) {
      const float* x = reinterpret_cast<const float*>(s_kv[i][0]);
      const float by = __builtin_amdgcn_exp2f(x[r] - base);
      l = __builtin_fmaf(by, x[16 + r], l);
      o += by * *reinterpret_cast<const f32x4*>(&x[32 + r * DP + d]);
    }
    if (d == 0) {
      part[r] = m;
      part[16 + r] = l;
    }
    *reinterpret_cast<f32x4*>(&part[32 + r * DP + d]) = o;
  }
}

template <class T, int DP>
__global__ __launch_bounds__(128) void block_attention_join_kernel(const BlockArgs p) {
  __shared__ int s_bad[16];
  const int64_t at = row_block();
  const FewPlace f = few_place(p, at * p.splits);
  if (f.token >= p.seqs.n_tokens) return;
  int seq, pos;
  Sequence sq;
  if (!token_at(p.seqs, f.token, threadIdx.x & 63, seq, sq, pos)) return;  // (zeros are there already)
  join_rows<T, DP, 128>(p, f, seq, sq, pos, p.splits, threadIdx.x, s_bad, [&](int i) {
    return p.parts + (at * p.splits + i) * part_floats<DP>();
  });
}

// The few rows' kernel takes each (token, key-value head, 16 of the group) by itself: its
// time goes with their number and their width.  The other one's hardly changes until the
// chip has a workgroup for each compute unit, and falls with the group, as fewer tokens
// share a walk.  us of both (few, many), bf16, widths of 128, 16 blocks of 64 of 8192 to
// 16384 keys, by token and head:
//   group 1   2048 124, 371; 4096 239, 375   (of 64 sequences 326, 308)
//   group 4   2048 124, 205; 4096 240, 206   (of 64 sequences 330, 256)
//   group 16  1024 66, 99; 2048 126, 99; 4096 241, 177   (of 64 sequences 2048 175, 175)
//   group 64  64 29, 39; 192 70, 60; 400 104, 60
//   group 8, 64 blocks  2048 281, 345; 4096 552, 357
//   group 4, width 256  1600 199, 205; 2048 230, 203;  width 64 (f16) 4096 106, 136
//   group 4, f32  2048 344, 632; 4096 681, 637
// Even at about 6500 of widths of 128 by the root of the group; never above 4096.  Of
// single tokens nothing is shared, unless 16 of the group at a time share a token's blocks,
// and of two a sequence little (8 heads, group 8):
//   of one a sequence  4096 290, 388; 16384 1713, 2275;  group 64 128 55, 41
//   of two             2048 189, 214; 4096 376, 422; 16384 1203, 990;  width 256 2048 345, 304
constexpr int64_t kFewMost = 4096, kEven = 6500;
inline bool few_rows(const fs_block_seqs& s, int heads, int group, int width) {
  const int64_t all = s.n_tokens * heads * ((group + 15) / 16);
  if (group <= 16 && s.n_tokens <= s.n_seqs) return true;
  if (all > kFewMost) return false;
  if (group <= 16 && width <= 128 && s.n_tokens <= 2 * s.n_seqs) return true;
  const int64_t wide = all * (width <= 64 ? 64 : width <= 128 ? 128 : 256);
  return wide * wide * group <= (kEven * 128) * (kEven * 128);
}

struct Plan {
  bool few;
  int splits;
  int64_t groups;  // (token, head, chunk) triples of the few rows' kernel
  int readers, per;
  int64_t tiles;
  size_t bytes;
};
Plan plan_of(int val_t, const fs_block_seqs& s, int heads, int group, int width, int top) {
  Plan o{};
  const int64_t tokens = s.n_tokens;
  const int block = s.block;
  o.readers = many_readers((width <= 64 ? 64 : width <= 128 ? 128 : 256) * (val_t == FS_F32 ? 4 : 2));
  // (a group whose rows do not fit a workgroup of the other kernel, too)
  o.few = few_rows(s, heads, group, width) || o.readers * 16 < group;
  o.groups = tokens * heads * ((group + 15) / 16);
  o.splits = 1;
  if (o.few) {
    const int bytes = (width <= 64 ? 64 : width <= 128 ? 128 : 256) * (val_t == FS_F32 ? 4 : 2);
    const int waves = bytes > 256 ? kFewWaves / 2 : kFewWaves;
    const int64_t steps = (int64_t)top * block / 32;
    // until a wave has four steps, or there are two workgroups a compute unit: the join is a
    // launch of its own (us with four, with one and with 16, one token of 8 x 4 heads of 128,
    // blocks of 64 keys: 16 blocks 20, 24, 20; 64 blocks 25, 25, 36; 128 blocks 29, 36, 50)
    while ((int64_t)o.splits * waves * 4 < steps && o.groups * o.splits < 512 && o.splits < 64) o.splits *= 2;
    if (o.splits > 1)
      o.bytes = (size_t)(o.groups * o.splits) * (32 + 16 * (width <= 64 ? 64 : width <= 128 ? 128 : 256)) * 4;
  } else {
    o.per = o.readers * 16 / group;
    o.tiles = block_tiles(s, o.per);
    o.bytes = (size_t)(o.tiles * heads) * o.readers * 4;
  }
  return o;
}

}  // namespace
}  // namespace fs

extern "C" size_t fs_block_attention_workspace_bytes(int val_t, const fs_block_seqs* seqs, int heads, int group,
                                                     int width, int top) {
  using namespace fs;
  if (block_sizes_fault("", val_t, seqs, heads, group, width) != FS_OK || top < 1 || top > kMostTop) return 0;
  return plan_of(val_t, *seqs, heads, group, width, top).bytes;
}

extern "C" int fs_block_attention(int val_t, const fs_block_seqs* seqs, int heads, int group, int width, int top,
                                  const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_page,
                                  int64_t k_row, int64_t k_head, const void* v, int64_t v_page, int64_t v_row,
                                  int64_t v_head, const int32_t* blocks, int64_t b_token, int64_t b_head, double scale,
                                  void* out, float* lse, void* ws, size_t ws_bytes, hipStream_t stream) {
  using namespace fs;
  const char* who = "fs_block_attention";
  if (const int rc = block_sizes_fault(who, val_t, seqs, heads, group, width)) return rc;
  if (top < 1 || top > kMostTop) return fail(FS_E_INVALID, std::string(who) + ": top out of range");
  if (seqs->n_tokens == 0) return FS_OK;
  const int64_t size = val_t == FS_F32 ? 4 : 2;
  if (!q || !k || !v || !blocks || !out || q_token < 0 || q_head < 0 || b_token < 0 || b_head < 0)
    return fail(FS_E_INVALID, std::string(who) + ": bad pointer or stride");
  if (!block_rows_fit(k, k_page, k_row, k_head, size) || !block_rows_fit(v, v_page, v_row, v_head, size))
    return fail(FS_E_INVALID, std::string(who) + ": keys and values need rows at multiples of 16 bytes");
  if (!(scale > 0.0) || !(scale < 1e30)) return fail(FS_E_INVALID, std::string(who) + ": scale must be positive");
  const Plan plan = plan_of(val_t, *seqs, heads, group, width, top);
  if (plan.bytes > 0 && (ws == nullptr || ws_bytes < plan.bytes))
    return fail(FS_E_WORKSPACE, std::string(who) + ": workspace too small");
  BlockArgs p{};
  p.seqs = *seqs;
  p.k = RowLayout{k, k_page, k_row, k_head};
  p.v = RowLayout{v, v_page, v_row, v_head};
  p.q = q;
  p.q_token = q_token;
  p.q_head = q_head;
  p.out = out;
  p.lse = lse;
  p.blocks = blocks;
  p.b_token = b_token;
  p.b_head = b_head;
  p.top = top;
  p.heads = heads;
  p.group = group;
  p.width = width;
  p.lg_groups = __builtin_ctz((unsigned)seqs->block) - 4;
  p.scale = (float)scale;
  p.splits = plan.splits;
  p.parts = static_cast<float*>(ws);
  p.again = static_cast<uint32_t*>(ws);
  return with_block_width(val_t, width, who, [&](auto val, auto dp) -> int {
    using T = decltype(val);
    constexpr int DP = decltype(dp)::value;
    if (plan.few) {
      const dim3 grid = row_grid(plan.groups * plan.splits), threads(64 * FewShape<T, DP>::kWaves);
      hipLaunchKernelGGL((block_attention_few_kernel<T, DP>), grid, threads, 0, stream, p);
      FS_CHECK_MAIN_LAUNCH("block_attention_few_kernel");
      if (plan.splits > 1) {
        hipLaunchKernelGGL((block_attention_join_kernel<T, DP>), row_grid(plan.groups), dim3(128), 0, stream, p);
        FS_CHECK_LAUNCH("block_attention_join_kernel");
      }
      return FS_OK;
    }
    p.tiles = plan.tiles;
    p.per = plan.per;
    if (p.tiles * heads > kMostWorkgroups) return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
    const dim3 grid((uint32_t)(p.tiles * heads));
    hipLaunchKernelGGL((block_attention_kernel<T, DP>), grid, dim3(ManyShape<T, DP>::kThreads), 0, stream, p);
    FS_CHECK_MAIN_LAUNCH("block_attention_kernel");
    hipLaunchKernelGGL((block_attention_again_kernel<T, DP>), grid, dim3(64 * ManyShape<T, DP>::kReaders), 0, stream, p);
    FS_CHECK_LAUNCH("block_attention_again_kernel");
    return FS_OK;
  });
}
