// block_tile.hpp — what the kernels over selected blocks share (block_*.hip): where
// sequences, pages and blocks lie, a tile of keys or values in LDS, fragments of it,
// and the softmax of a tile of queries.
//
// A matrix instruction takes 16 keys by 16 query rows.  Scores come transposed,
// keys down and queries across (K Q^T): a lane then holds scores of one query, so
// its maximum and sum need two exchanges between lanes and no more, and the scores
// of 4 keys in a row that it holds are, as they lie, the second operand of the
// product with the values (V^T P^T), whose first operand the LDS read transposes.
#pragma once

#include <type_traits>

#include "matrix_core.hpp"
#include "select_rows.hpp"

namespace fs {
namespace {

constexpr int kMostTop = 128;  // blocks that a query may select
// Keys of a sequence, so that the position behind its last block fits 32 bits too.
constexpr int64_t kMostKeys = INT32_MAX - 2047;

// ---- sequences, pages -----------------------------------------------------------

__device__ inline int clamp_to(int64_t v, int64_t lo, int64_t hi) { return (int)(v < lo ? lo : v > hi ? hi : v); }

// Query tokens and keys of sequence b; of n_seqs the tokens behind the last
// sequence, without keys.  Offsets are on the device and unchecked: whatever they
// hold, tokens and rows are within their arrays.
struct Sequence {
  int first, count;  // tokens
  int keys;
  int64_t row0;  // of the keys, packed
};
__device__ inline int alike(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline Sequence sequence_at(const fs_block_seqs& s, int b) {
  Sequence o;
  o.keys = 0;
  o.row0 = 0;
  if (s.q_offsets == nullptr) {
    o.first = b;
    o.count = b < s.n_seqs ? 1 : 0;
  } else {
    o.first = b == 0 ? 0 : clamp_to(s.q_offsets[b], 0, s.n_tokens);
    o.count = (b < s.n_seqs ? clamp_to(s.q_offsets[b + 1], o.first, s.n_tokens) : (int)s.n_tokens) - o.first;
  }
  if (b < s.n_seqs) {
    if (s.pages != nullptr) {
      const int64_t most = s.pages_per_seq * s.page_size;
      o.keys = clamp_to(s.k_lengths[b], 0, most < kMostKeys ? most : kMostKeys);
    } else {
      o.row0 = clamp_to(s.k_offsets[b], 0, s.n_rows);
      o.keys = clamp_to(s.k_offsets[b + 1], o.row0, s.n_rows) - (int)o.row0;
    }
  }
  return o;
}

// The same of a b that all lanes have, in scalar registers.
__device__ inline Sequence sequence_of(const fs_block_seqs& s, int b) {
  Sequence o = sequence_at(s, alike(b));
  o.first = alike(o.first);
  o.count = alike(o.count);
  o.keys = alike(o.keys);
  o.row0 = alike((int)o.row0);
  return o;
}

// The sequence and tile of tile i, `per` tokens a tile: sequences in order, the
// tokens behind the last one as one more.  false: there is no such tile.
// (All lanes alike.)
__device__ inline bool find_tile(const fs_block_seqs& s, int per, int64_t i, int lane, int& seq, int& tile) {
  if (s.q_offsets == nullptr) {
    seq = (int)i;
    tile = 0;
    return i < s.n_seqs;
  }
  int64_t before = 0;
  for (int64_t b0 = 0; b0 <= s.n_seqs; b0 += 64) {
    const int64_t b = b0 + lane;
    const int own = b <= s.n_seqs ? (sequence_at(s, (int)b).count + per - 1) / per : 0;
    const int64_t upto = (int64_t)wave_sum_scan((uint32_t)own) + before;
    const uint64_t m = __ballot(upto > i);
    if (m != 0) {
      const int l = __builtin_ctzll(m);
      seq = (int)b0 + l;
      tile = (int)(i - before) - (__builtin_amdgcn_readlane((int)(upto - before), l) - __builtin_amdgcn_readlane(own, l));
      return true;
    }
    before += __builtin_amdgcn_readlane((int)(upto - before), 63);
  }
  return false;
}

// A cache's or packed rows' layout: distances in elements.
struct RowLayout {
  const void* base;
  int64_t page, row, head;
};

// First element of 16 keys that begin at position j (a multiple of 16) of a
// sequence, or null where their page is outside the cache.
template <class T>
__device__ inline const T* key_rows(const fs_block_seqs& s, const Sequence& q, int seq, const RowLayout& l, int head,
                                    int j) {
  const T* base = static_cast<const T*>(l.base) + (int64_t)head * l.head;
  if (s.pages == nullptr) return base + (q.row0 + j) * l.row;
  const int64_t at = j >> s.page_shift;
  if (at >= s.pages_per_seq) return nullptr;
  const int64_t page = s.pages[(int64_t)seq * s.ld_pages + at];
  if (page < 0 || page >= s.n_pages) return nullptr;
  return base + page * l.page + (int64_t)(j & (s.page_size - 1)) * l.row;
}

// ---- tiles in LDS ---------------------------------------------------------------

typedef __attribute__((address_space(3))) uint32_t lds_word;
typedef __attribute__((address_space(3))) const uint8_t clds_byte;

__device__ inline uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// Rows of DP elements (a head's width, filled up), 16-byte pieces exchanged within
// a row so that neither a fragment of 16 rows by one piece nor a transposing read
// of 4 rows by 32 bytes meets a bank twice.
template <class T, int DP>
struct Rows {
  static constexpr int kRow = DP * (int)sizeof(T);  // bytes: 128, 256 or 512
  static constexpr int kPieces = kRow / 16;
  static constexpr int kUnit = sizeof(T) == 2 ? 32 : 16;  // rows that one product over rows takes
  static constexpr int kKeys = 32;                         // keys a step
  static constexpr int kGroups = kKeys / 16;
  static constexpr int kBytes = kKeys * kRow;
  static constexpr int kFrags = kRow / 64;     // fragments of 16 rows
  static constexpr int kTiles = DP / 16;       // tiles of 16 columns
  using frag = typename Mma<T>::frag;

  __device__ static int swizzle(int row) {
    if constexpr (sizeof(T) == 4) return ((row >> 2) & 3) * 4 + (row & 3);
    else if constexpr (kRow == 128) return ((row >> 1) & 3) * 2 + ((row >> 3) & 1);
    else return (row & 7) * 2 + ((row >> 3) & 1);
  }

  // One load instruction: 64 lanes' pieces of kAtOnce rows.
  static constexpr int kAtOnce = 64 / kPieces;
  __device__ static int lane_row(int lane) { return lane / kPieces; }

  // Fragment of rows r0 .. r0 + 15 (a multiple of 16), column piece 4 ks + lane / 16.
  __device__ static frag across(uint32_t lds, int r0, int ks, int lane) {
    const int i = lane & 15, g = lane >> 4;
    const uint32_t at = lds + (uint32_t)(r0 * kRow) + (uint32_t)(i * kRow) +
                        (uint32_t)(((ks << 2) ^ (g ^ swizzle(i))) << 4);
    const u32x4 v = *(const lds_u32x4*)(lds_byte*)(uintptr_t)at;
    frag f;
    __builtin_memcpy(&f, &v, 16);
    return f;
  }
  // Fragment of columns 16 dt .. 16 dt + 15 over kUnit rows from r0: lane i of its
  // 16 has column i of rows 4 g .. 4 g + 3 (16-bit values: and of those 16 further).
  __device__ static frag down(uint32_t lds, int r0, int dt, int lane) {
    const int i = lane & 15, g = lane >> 4;
    frag f;
    if constexpr (sizeof(T) == 2) {
      const int r = 4 * g + (i >> 2);
      const uint32_t at = lds + (uint32_t)(r0 * kRow) + (uint32_t)(r * kRow) +
                          (uint32_t)((((dt << 1) ^ ((i & 3) >> 1) ^ swizzle(r)) << 4) + (i & 1) * 8);
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_byte*)(uintptr_t)at);
      const s16x4 hi =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(lds_byte*)(uintptr_t)(at + 16 * kRow));
      __builtin_memcpy(&f, &lo, 8);
      __builtin_memcpy((char*)&f + 8, &hi, 8);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * g + j;
        const uint32_t at = lds + (uint32_t)(r0 * kRow) + (uint32_t)(r * kRow) +
                            (uint32_t)((((dt << 2) + (i >> 2)) ^ swizzle(r)) << 4) + (uint32_t)(i & 3) * 4;
        f[j] = *(const lds_float*)(lds_byte*)(uintptr_t)at;
      }
    }
    return f;
  }
  // The other operand: values of kUnit rows that products of 16 rows left, rounded
  // to the value type.
  __device__ static frag rounded(const f32x4* s) {
    frag f;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        f[j] = (T)s[0][j];
        f[4 + j] = (T)s[1][j];
      }
    } else {
      f = s[0];
    }
    return f;
  }
  // The same in two parts of 16 bits, the second what rounding to the first leaves out:
  // 16 bits of a bfloat16 value and 22 of a float16 one, for 32-bit sums, instead of 8 and
  // 11.  A product takes two instructions; the fragment of rows beside it is read once.
  static constexpr int kParts = sizeof(T) == 2 ? 2 : 1;
  struct Halves {
    frag part[kParts];
  };
  __device__ static Halves halves(const f32x4* s) {
    Halves o;
    o.part[0] = rounded(s);
    if constexpr (kParts == 2) {
      uint32_t pair[4];
      __builtin_memcpy(pair, &o.part[0], 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // (from the pairs as they are: by elements the compiler rounds a second time)
        float first, second;
        if constexpr (std::is_same_v<T, __bf16>) {
          first = __uint_as_float(pair[j] << 16);
          second = __uint_as_float(pair[j] & 0xffff0000u);
        } else {
          first = (float)o.part[0][2 * j];
          second = (float)o.part[0][2 * j + 1];
        }
        o.part[1][2 * j] = (T)(s[j >> 1][2 * (j & 1)] - first);
        o.part[1][2 * j + 1] = (T)(s[j >> 1][2 * (j & 1) + 1] - second);
      }
    }
    return o;
  }
};

// Reads of LDS run ahead of the products that use them, AHEAD fragments at a time:
// left to itself the compiler waits for each by itself.
__device__ inline void fence() { __builtin_amdgcn_sched_barrier(0); }

// Of 32-bit values, whose products are eight times as slow, columns past the width are
// left out: `used` counts the 16 columns at a time that are not (float32, 3 sequences of
// 2501 tokens and fewer, 12 heads of 80 columns: 314 us, without this 385).
template <class T>
__device__ inline bool leave_out(int at, int used) { return sizeof(T) == 4 && at >= used; }

// s[gr] += rows 16 gr .. of the tile at lds times the lane's row, in f: scores, or
// products of values with a gradient.
template <class T, int DP, int AHEAD>
__device__ inline void products(uint32_t lds, const typename Mma<T>::frag (&f)[Rows<T, DP>::kFrags],
                                f32x4 (&s)[Rows<T, DP>::kGroups], int used, int lane) {
  using R = Rows<T, DP>;
  constexpr int G = R::kGroups, F = R::kFrags, kStep = AHEAD / G < F ? AHEAD / G : F;  // fragments' columns at a time
#pragma unroll
  for (int k0 = 0; k0 < F; k0 += kStep) {
    typename R::frag x[kStep][G];
#pragma unroll
    for (int ks = 0; ks < kStep; ++ks)
#pragma unroll
      for (int gr = 0; gr < G; ++gr)
        if (!leave_out<T>(k0 + ks, used)) x[ks][gr] = R::across(lds, gr * 16, k0 + ks, lane);
    fence();
#pragma unroll
    for (int ks = 0; ks < kStep; ++ks)
      if (!leave_out<T>(k0 + ks, used))
#pragma unroll
        for (int gr = 0; gr < G; ++gr) s[gr] = Mma<T>::run(x[ks][gr], f[k0 + ks], s[gr]);
  }
}
// Columns of the tile: the first operands of the products over its rows.
template <class T, int DP, int AHEAD>
struct Columns {
  using R = Rows<T, DP>;
  static constexpr int kUnits = R::kKeys / R::kUnit, kAll = kUnits * (DP / 16), kStep = kAll < AHEAD ? kAll : AHEAD;
  typename R::frag x[kStep];
  __device__ void read(uint32_t lds, int first, int used, int lane) {
#pragma unroll
    for (int i = 0; i < kStep; ++i) {
      const int at = first + i;
      if (!leave_out<T>(at % (DP / 16), used)) x[i] = R::down(lds, at / (DP / 16) * R::kUnit, at % (DP / 16), lane);
    }
    fence();
  }
  // o[dt] += columns times w, after read(lds, 0): what is left is read here.  done() once
  // all is read, before the last products: nobody waits for those.
  template <class Done>
  __device__ void add(uint32_t lds, const typename R::Halves (&w)[kUnits], f32x4 (&o)[DP / 16], int used, int lane,
                      Done done) {
#pragma unroll
    for (int first = 0; first < kAll; first += kStep) {
      if (first > 0) read(lds, first, used, lane);
      if (first + kStep == kAll) done();
#pragma unroll
      for (int n = 0; n < R::kParts; ++n) {
#pragma unroll
        for (int i = 0; i < kStep; ++i) {
          const int at = first + i;
          if (!leave_out<T>(at % (DP / 16), used))
            o[at % (DP / 16)] = Mma<T>::run(x[i], w[at / (DP / 16)].part[n], o[at % (DP / 16)]);
        }
      }
    }
  }
};

// The largest, and the sum, of a value over the four lanes of a query.
__device__ inline float across_max(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ inline float across_sum(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// What the kernels of queries take.
struct BlockArgs {
  fs_block_seqs seqs;
  RowLayout k, v;
  const void* q;
  int64_t q_token, q_head;  // distances in elements
  void* out;                // tokens x heads * group x width, dense
  float* lse;               // tokens x heads * group; may be null
  const int32_t* blocks;
  int64_t b_token, b_head;
  int top, heads, group, width;
  int lg_groups;  // log2 of a block's groups of 16 keys
  float scale;
  int64_t tiles;    // workgroups a head
  int per;          // tokens a workgroup
  uint32_t* again;  // many rows: a word a wave, its rows whose result is not finite
  int splits;
  float* parts;
};

// Keys, or values, of one sequence and head, and a wave's loads of a step of them.
template <class T, int DP>
struct KeySource {
  using R = Rows<T, DP>;
  static constexpr int kLoads = R::kBytes / 1024, kGroups = R::kGroups;
  static constexpr int kAGroup = 16 / R::kAtOnce;  // loads of 16 rows
  const char* base;
  uint32_t row;           // bytes
  uint32_t off[kAGroup];  // a lane's, within 16 rows
  // the sequence's pages, or null (constant for the call: scalar loads, which leave the
  // count of loads under way alone)
  typedef const __attribute__((address_space(4))) int32_t Constant;
  Constant* table;
  int64_t page, n_pages;
  int per_seq, shift, keys;

  __device__ void init(const BlockArgs& p, const RowLayout& l, const Sequence& sq, int seq, int head, int lane) {
    base = static_cast<const char*>(l.base) + (head * l.head + sq.row0 * l.row) * (int64_t)sizeof(T);
    row = (uint32_t)(l.row * (int64_t)sizeof(T));
    keys = sq.keys;
    table = p.seqs.pages == nullptr ? nullptr : (Constant*)(p.seqs.pages + (int64_t)seq * p.seqs.ld_pages);
    page = l.page * (int64_t)sizeof(T);
    n_pages = p.seqs.n_pages;
    per_seq = (int)p.seqs.pages_per_seq;
    shift = p.seqs.page_shift;
#pragma unroll
    for (int n = 0; n < kAGroup; ++n) {
      const int r = R::lane_row(lane) + n * R::kAtOnce, piece = (lane % R::kPieces) ^ R::swizzle(r);
      const bool in = piece * 16 < p.width * (int)sizeof(T);
      off[n] = in ? (uint32_t)r * row + (uint32_t)piece * 16 : 2u * kInBuffer;
    }
  }
  // Where a step lies.  `whole`: all its rows are keys and one behind the other, from
  // at[0] on; otherwise the first byte of each group of 16 keys, and how many of its rows
  // are keys.  Bits of the groups whose page is outside the cache.
  struct Place {
    const char* at[kGroups];
    int left[kGroups];
    uint32_t missing;
    bool whole;
  };
  // Key j on, of the page `id` (without pages: any).
  __device__ const char* rows_at(int64_t id, int j) const {
    return table == nullptr ? base + (int64_t)j * row : base + id * page + (int64_t)(j & ((1 << shift) - 1)) * row;
  }
  __device__ void find(int first, Place& o) const {
    o.missing = 0;
    o.whole = false;
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr) {
      const int j = first + gr * 16;
      o.at[gr] = base;
      o.left[gr] = 0;
      if (j < keys) {
        int64_t id = 0;
        if (table != nullptr) {
          const int t = j >> shift;
          id = t < per_seq ? table[t] : -1;
          if (id >= n_pages) id = -1;
        }
        if (id >= 0) {
          o.at[gr] = rows_at(id, j);
          o.left[gr] = keys - j;
        } else {
          o.missing |= 1u << gr;
        }
      }
    }
  }
  // One step to LDS, zeros past the sequence's end, past the width and for pages outside
  // the cache.
  __device__ void load(uint32_t lds, const Place& o, int lane) const {
    if (o.whole) {
      const u32x4 rsrc = buffer_at(o.at[0]);
#pragma unroll
      for (int gr = 0; gr < kGroups; ++gr)
#pragma unroll
        for (int n = 0; n < kAGroup; ++n)
          lds_dma_shifted(lds + (uint32_t)(gr * 16 * R::kRow + n * 1024), off[n], rsrc, (uint32_t)(gr * 16) * row);
      return;
    }
#pragma unroll
    for (int gr = 0; gr < kGroups; ++gr) {
      const u32x4 rsrc = buffer_at(o.at[gr]);
      const uint32_t to = lds + (uint32_t)(gr * 16 * R::kRow);
#pragma unroll
      for (int n = 0; n < kAGroup; ++n) {
        const bool in = R::lane_row(lane) + n * R::kAtOnce < o.left[gr];
        lds_dma<16>(to + (uint32_t)n * 1024, in ? off[n] : 2u * kInBuffer, rsrc);
      }
    }
  }
};

// 16 query rows of a wave: lanes with the same lane % 16 hold one row's state.
struct RowOf {
  int token;  // within the workgroup's tile
  int head;   // within the group
  int pos;    // its position; -1 and less: before the first key
  bool in;
};

// Fragments of a lane's row of a dense or strided array, zeros outside.
template <class T, int DP>
__device__ inline void load_row(const T* row, bool in, int width, int lane,
                                typename Mma<T>::frag (&f)[Rows<T, DP>::kFrags]) {
#pragma unroll
  for (int ks = 0; ks < Rows<T, DP>::kFrags; ++ks) {
    const int piece = ks * 4 + (lane >> 4);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (in && piece * 16 < width * (int)sizeof(T)) __builtin_memcpy(&v, (const char*)row + piece * 16, 16);
    __builtin_memcpy(&f[ks], &v, 16);
  }
}

// Columns 16 dt + 4 g .. + 3 of a lane's row.
template <class T, int DP>
__device__ inline void store_row(T* row, const f32x4 (&o)[DP / 16], float by, int width, int lane) {
#pragma unroll
  for (int dt = 0; dt < DP / 16; ++dt) {
    const int d = dt * 16 + (lane >> 4) * 4;
    if (d < width) {  // (a multiple of 4)
      T e[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = (T)(o[dt][j] * by);
      __builtin_memcpy(row + d, e, sizeof e);
    }
  }
}

// ---- host side ------------------------------------------------------------------

constexpr int64_t kMostWorkgroups = ((int64_t)1 << 32) / 1024 - 1;  // of up to 1024 threads, in one dimension

inline int64_t block_tiles(const fs_block_seqs& s, int per) {
  return s.q_offsets == nullptr ? s.n_seqs : s.n_tokens / per + s.n_seqs + 1;
}

inline int block_seqs_fault(const char* who, const fs_block_seqs* s) {
  auto refuse = [&](const char* text) { return fail(FS_E_INVALID, std::string(who) + ": " + text); };
  if (s == nullptr) return refuse("null pointer");
  if (s->n_seqs < 0 || s->n_seqs > INT32_MAX / 2 || s->n_tokens < 0 || s->n_tokens > INT32_MAX || s->n_rows < 0 ||
      s->n_rows > kMostKeys)
    return refuse("sizes out of range");
  if (s->block < 32 || s->block > 1024 || (s->block & (s->block - 1)) != 0)
    return refuse("blocks are of 32, 64, 128, 256, 512 or 1024 keys");
  if (s->q_offsets == nullptr && s->n_tokens != s->n_seqs) return refuse("without offsets a sequence has one token");
  if (s->pages != nullptr) {
    if (s->k_lengths == nullptr && s->n_seqs > 0) return refuse("null pointer");
    if (s->page_size < 16 || s->page_size > (1 << 20) || (s->page_size & (s->page_size - 1)) != 0 ||
        s->page_shift != __builtin_ctz((unsigned)s->page_size))
      return refuse("pages are of a power of two of rows, 16 at least");
    if (s->n_pages < 0 || s->pages_per_seq < 0 || s->ld_pages < 0) return refuse("sizes out of range");
  } else if (s->k_offsets == nullptr && s->n_seqs > 0) {
    return refuse("null pointer");
  }
  return FS_OK;
}

inline int block_sizes_fault(const char* who, int val_t, const fs_block_seqs* s, int heads, int group, int width) {
  if (const int rc = block_seqs_fault(who, s)) return rc;
  auto refuse = [&](const char* text) { return fail(FS_E_INVALID, std::string(who) + ": " + text); };
  if (val_t != FS_F16 && val_t != FS_BF16 && val_t != FS_F32) return refuse("value types are FS_F16, FS_BF16 and FS_F32");
  if (heads < 1 || heads > 65535 || group < 1 || group > 128) return refuse("heads out of range");
  if (width < 8 || width % 8 != 0 || width > (val_t == FS_F32 ? 128 : 256)) return refuse("width out of range");
  return FS_OK;
}

// Whether loads of 16 bytes can take the rows, and the distances of 64 of them fit.
inline bool block_rows_fit(const void* base, int64_t page, int64_t row, int64_t head, int64_t size) {
  if (page < 0 || row < 0 || head < 0 || row > ((int64_t)1 << 22)) return false;
  return (((int64_t)(uintptr_t)base | page * size | row * size | head * size) & 15) == 0;
}

// Runs f with a value of the value type and the width filled up.
template <class F>
int with_block_width(int val_t, int width, const char* who, F&& f) {
  auto by_width = [&](auto v) -> int {
    using T = decltype(v);
    if (width <= 64) return f(v, std::integral_constant<int, 64>{});
    if (width <= 128) return f(v, std::integral_constant<int, 128>{});
    if constexpr (sizeof(T) == 2) return f(v, std::integral_constant<int, 256>{});
    return fail(FS_E_INVALID, std::string(who) + ": width out of range");
  };
  if (val_t == FS_F16) return by_width((_Float16)0);
  if (val_t == FS_BF16) return by_width((__bf16)0);
  return by_width(0.0f);
}

}  // namespace
}  // namespace fs
