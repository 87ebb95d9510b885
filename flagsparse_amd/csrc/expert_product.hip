// expert_product.hip — the experts' products on matrix cores.
//
// Rows of expert order, a block of consecutive rows an expert (offsets, from
// fs_expert_route), times the expert's matrix: a block-diagonal product.
//   rows    C[r, n] = sum_k A[r, k] B_e(k, n), e the expert of row r, with
//           B_e stored (N, K) ("trans", k contiguous) or (K, N) ("non")
//   matrix  C_e[m, n] = sum over the rows r of e of A[r, m] B[r, n], the
//           gradient of the matrices
// Rows of no expert (from offsets[n_experts] on) are written as zeros.
//
// A workgroup computes one BM x BN tile of one expert, 64 bytes of k (one
// fragment) a step: both operands' slices go to LDS, 16-byte pieces exchanged
// within a row so that fragment reads meet no bank twice, and feed 16x16 matrix
// instructions that accumulate in 32 bits.  Results are rounded once.
// Where an operand is contiguous in k a fragment is one 16-byte LDS read; where
// it is contiguous along the tile, 16-bit fragments are transposed by the LDS
// read itself and 32-bit ones are read element by element.
// How many rows an expert has is known on the device only: the grid is an upper
// bound, each workgroup finds its tile from the offsets, and those beyond the
// last tile leave.
//
// Many rows: bound by the matrix instructions at the clock the card's power allows
// (1.4 to 1.6 GHz): bf16, 8192 x 8192 x 8192 1340 to 1440 TFLOP/s, 32768 rows of 16
// experts 4096 x 4096 of unlike popularity 957 us, 1150 TFLOP/s; both gradients of
// 16044 rows of 8 experts 2048 x 5120 f16 647 us, 1060 TFLOP/s.  Few rows: by the
// matrices' bytes, 64 rows of 25 of 32 experts 2048 x 4096 bf16 82 us, 420 MB at
// 5.1 TB/s, the rate of a copy.
#include <initializer_list>
#include <type_traits>

#include "matrix_core.hpp"
#include "select_rows.hpp"

namespace fs {
namespace {

constexpr int kRowBytes = 64;  // k of one step, of an operand contiguous in k

// One operand's slice in LDS, and the way there.  KC: contiguous in k, R rows
// of the tile by 64 bytes of k; otherwise BK rows of k by R elements.
template <class T, bool KC, int R, int THREADS>
struct Operand {
  static constexpr int E = 16 / (int)sizeof(T);        // elements a piece
  static constexpr int BK = kRowBytes / (int)sizeof(T);
  static constexpr int kBytes = R * kRowBytes;
  static constexpr int kPieces = kBytes / 16 / THREADS;  // a thread's, each step
  static constexpr int kPerRow = KC ? 4 : R * (int)sizeof(T) / 16;
  static_assert(kBytes % (16 * THREADS) == 0, "whole pieces a thread");

  // Exchange of the pieces of LDS row `row`.
  __device__ static int swizzle(int row) {
    if constexpr (KC) return (row >> 1) & 3;
    else if constexpr (sizeof(T) == 4) return ((row >> 2) & 1) * 4;
    else return ((row & 3) + (kPerRow >= 16 ? ((row >> 3) & 1) * 4 : 0)) * 2;
  }
  // The q-th piece of the slice in LDS: its row, and which piece of it it is.
  __device__ static int row_at(int q) { return q / kPerRow; }
  __device__ static int piece_at(int q) { return (q % kPerRow) ^ swizzle(row_at(q)); }
  __device__ static int row_of(int i, int tid) { return row_at(i * THREADS + tid); }
  __device__ static int piece_of(int i, int tid) { return piece_at(i * THREADS + tid); }

  // Fragment of 16 tile rows from r0: lane l has tile row l % 16, k piece l / 16.
  __device__ static uint32_t frag_offset(int r0, int lane) {
    const int g = lane >> 4, i = lane & 15;
    if constexpr (KC) {
      return (uint32_t)((r0 + i) * kRowBytes + ((g ^ ((i >> 1) & 3)) * 16));
    } else if constexpr (sizeof(T) == 4) {
      const int row = 4 * g;
      return (uint32_t)(row * R * 4 + ((r0 / 4 + i / 4) ^ swizzle(row)) * 16 + (i & 3) * 4);
    } else {
      const int row = 8 * g + i / 4;
      return (uint32_t)(row * R * 2 + ((r0 / 8 + (i & 3) / 2) ^ swizzle(row)) * 16 + (i & 1) * 8);
    }
  }
  __device__ static typename Mma<T>::frag frag(const lds_byte* p) {
    typename Mma<T>::frag f;
    if constexpr (KC) {
      const u32x4 v = *(const lds_u32x4*)p;
      __builtin_memcpy(&f, &v, 16);
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = *(const lds_float*)(p + i * R * 4);
    } else {
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 4 * R * 2));
      __builtin_memcpy(&f, &lo, 8);
      __builtin_memcpy((char*)&f + 8, &hi, 8);
    }
    return f;
  }
};

// A wave's fragments of one operand: F of them, from tile row r0 on.
template <class O, bool KC, int F>
struct Frags {
  uint32_t at[KC ? 1 : F];
  __device__ void init(int r0, int lane) {
#pragma unroll
    for (int j = 0; j < (KC ? 1 : F); ++j) at[j] = O::frag_offset(r0 + j * 16, lane);
  }
  // (the first `some` of them)
  template <class X>
  __device__ void read(uint32_t slice, X (&f)[F], int some = F) const {
#pragma unroll
    for (int j = 0; j < F; ++j)
      if (j < some) {
        const lds_byte* p = (const lds_byte*)(uintptr_t)(slice + at[KC ? 0 : j]);
        f[j] = O::frag(p + (KC ? j * 16 * kRowBytes : 0));
      }
  }
};

// What one operand's loads need: the tile's first element, the distance of its
// rows (of the tile if KC, of k otherwise), and how many there are of each.
template <class T>
struct Source {
  const T* base;
  int64_t ld;
  int tile_rows;  // tile rows within the operand
  int64_t k;      // k within it
};

// The i-th piece of thread tid in step kt of an operand.
template <class O, class T, bool KC>
struct Piece {
  const T* p;
  int64_t left;  // elements of its row from its first on
  __device__ Piece(const Source<T>& s, int64_t kt, int tid, int i) {
    const int row = O::row_of(i, tid), piece = O::piece_of(i, tid);
    const int64_t k0 = kt * O::BK;
    const int64_t line = KC ? row : k0 + row;                            // row of memory
    const int64_t first = KC ? k0 + (int64_t)piece * O::E : piece * O::E;  // element in it
    p = s.base + line * s.ld + first;
    left = line < (KC ? (int64_t)s.tile_rows : s.k) ? (KC ? s.k : (int64_t)s.tile_rows) - first : 0;
  }
};
// A thread's pieces of step kt in registers, zeros outside the operand.  A piece
// that its row ends in is taken element by element at the end of k, once; at the
// end of the tile's columns, which is met in every step, it is loaded so that it
// ends with the row, and shifted when it is stored (us, element by element and so:
// two of 8 experts 4095 x 4095 bf16, (K, N), 39 and 22, matrix gradient of 4096 x
// 2 rows, 8 of 1001 x 3001 122 and 97; for the end of k, (N, K), 56 and 70).
template <class O, class T, bool KC>
__device__ inline bool shifts(const Source<T>& s) {
  return !KC && s.tile_rows >= O::E;
}
template <class O, class T, bool KC>
__device__ inline void load_pieces(const Source<T>& s, int64_t kt, int tid, u32x4 (&r)[O::kPieces]) {
  constexpr int E = O::E;
  const bool shift = shifts<O, T, KC>(s);
#pragma unroll
  for (int i = 0; i < O::kPieces; ++i) {
    const Piece<O, T, KC> a(s, kt, tid, i);
    u32x4 v = {0u, 0u, 0u, 0u};
    if (a.left >= E || (shift && a.left > 0)) {
      __builtin_memcpy(&v, a.p - (!KC && a.left < E ? E - a.left : 0), 16);
    } else if (a.left > 0) {
      T e[E];
#pragma unroll
      for (int q = 0; q < E; ++q) e[q] = q < a.left ? a.p[q] : (T)0;
      __builtin_memcpy(&v, e, 16);
    }
    r[i] = v;
  }
}
template <class O, class T, bool KC>
__device__ inline void store_pieces(const Source<T>& s, int64_t kt, uint32_t lds, int tid, u32x4 (&r)[O::kPieces],
                                    int threads) {
  const bool shift = shifts<O, T, KC>(s);
#pragma unroll
  for (int i = 0; i < O::kPieces; ++i) {
    u32x4 v = r[i];
    const int64_t left = shift ? Piece<O, T, KC>(s, kt, tid, i).left : 0;
    if (left > 0 && left < O::E) {
      const unsigned bits = (unsigned)(O::E - left) * 8u * (unsigned)sizeof(T);  // 16 to 112
      const uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
      const uint64_t x = bits < 64 ? lo >> bits | hi << (64 - bits) : hi >> (bits - 64), y = bits < 64 ? hi >> bits : 0;
      v = u32x4{(uint32_t)x, (uint32_t)(x >> 32), (uint32_t)y, (uint32_t)(y >> 32)};
    }
    *(lds_u32x4*)(lds_byte*)(uintptr_t)(lds + (uint32_t)(i * threads + tid) * 16) = v;
  }
}

// The same straight to LDS (buffer loads that write LDS, 64 lanes x WIDTH bytes
// from the address in M0): nothing in registers but an offset a load.  WIDTH 16
// takes whole pieces, 4 operands whose rows only start on whole words (2046 x
// 4094 bf16, 32 experts, 8192 rows: 250 us, through registers 376, 2048 x 4096
// with WIDTH 16 190); 16-bit rows off whole words go through registers.
// Offsets below kInBuffer count from the step's base, which moves; a load
// outside the operand gets one beyond it, and writes zeros.
template <class O, class T, bool KC, int THREADS, int WIDTH>
struct Dma {
  static constexpr int kLoads = O::kBytes / THREADS / WIDTH;  // a thread's, each step
  uint32_t off[kLoads];
  const char* base;
  int64_t step;  // bytes from one step to the next
  // the i-th load of thread tid: LDS row, and element in it
  __device__ static int row(int i, int tid) { return O::row_at((i * THREADS + tid) * WIDTH / 16); }
  __device__ static int element(int i, int tid) {
    const int at = (i * THREADS + tid) * WIDTH;
    return O::piece_at(at / 16) * O::E + at % 16 / (int)sizeof(T);
  }
  __device__ void init(const Source<T>& s, int tid) {
    base = (const char*)s.base;
    step = KC ? (int64_t)kRowBytes : s.ld * (int64_t)sizeof(T) * O::BK;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const bool in = (KC ? row(i, tid) : element(i, tid)) < s.tile_rows;
      off[i] = in ? (uint32_t)((row(i, tid) * s.ld + element(i, tid)) * (int64_t)sizeof(T)) : 2u * kInBuffer;
    }
  }
  // Before the loads of a step that has only `left` of k (none or less: zeros).
  __device__ void cut(int64_t left, int tid) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if ((KC ? element(i, tid) : row(i, tid)) >= left) off[i] |= kInBuffer;
  }
  __device__ u32x4 at(int64_t kt) const { return buffer_at(base + kt * step); }
  __device__ void issue(uint32_t lds, u32x4 rsrc, int i, int w) const {
    lds_dma<WIDTH>(lds + (uint32_t)(i * THREADS + w * 64) * WIDTH, off[i], rsrc);
  }
};

struct ProductArgs {
  const void* a;
  const void* b;
  void* c;
  const int32_t* offsets;
  int64_t lda, ldb, ldc;   // distances of rows
  int64_t b_expert, c_expert;  // distances of experts' matrices
  int64_t n_rows;          // rows of A
  int64_t m, n, k;         // m: of a matrix gradient; k: of a product of rows
  int n_experts;
  int cus;                 // compute units
  bool turn;               // whether tiles may begin at different steps
  float* parts;            // room for the sums of split tiles, or null
};

struct TileAt {
  int expert;  // n_experts: rows of no expert
  int64_t row0;
  int rows;
  int m, n;  // tile within the expert
};

constexpr int kGroupN = 4;  // neighbouring tiles share 4 column panels

// Tile r of an expert with mt x nt tiles: groups of kGroupN columns, rows first.
__device__ inline void tile_in_group(uint32_t r, uint32_t mt, uint32_t nt, TileAt& t) {
  const uint32_t g = r / (mt * kGroupN), left = nt - g * kGroupN, gn = left < kGroupN ? left : kGroupN;
  const uint32_t q = r - g * mt * kGroupN;
  t.m = (int)(q / gn);
  t.n = (int)(g * kGroupN + q % gn);
}

enum Mode { kRowsTrans = 0, kRowsNon = 1, kMatrix = 2 };

// The tiles of a call: `real` ones, of which the last `rest` are each shared by
// `parts` workgroups, and those of rows of no expert, only written.
struct TilePlan {
  uint32_t real, zero, full, rest, parts;
};

// Tiles of a last round that leaves most of the chip idle are cut along k into
// the parts that take the least time: a large tile takes about 0.8 us a step,
// writing and adding a tile's sums 0.085 us a part and tile, so parts^2 = 9 steps
// / rest (smaller tiles: both in proportion).  `places`: tiles at a time.
constexpr int kLarge = 256;
constexpr uint32_t kMostParts = 32;
__host__ __device__ inline uint32_t places_of(int cus, int bm) { return (uint32_t)cus * (bm == kLarge ? 1 : 2); }
__host__ __device__ inline uint32_t parts_of(uint32_t rest, int64_t steps, uint32_t places) {
  uint32_t parts = 1;
  while (rest > 0 && parts < kMostParts && (parts + 1) * rest <= places &&
         (int64_t)(parts + 1) * (parts + 1) * rest <= 9 * steps)
    ++parts;
  return parts;
}

// (All waves alike; so are the places below.)
template <int MODE, int BM, int BN>
__device__ inline TilePlan plan_tiles(const ProductArgs& p, int lane) {
  const uint32_t nt = (uint32_t)((p.n + BN - 1) / BN);
  TilePlan l;
  int64_t steps;
  constexpr int kStep = kRowBytes / 2;  // k of a step of 16-bit values
  if constexpr (MODE == kMatrix) {
    l.real = (uint32_t)((p.m + BM - 1) / BM) * nt * (uint32_t)p.n_experts;
    l.zero = 0;
    steps = p.n_rows / p.n_experts / kStep;
  } else {
    int total = 0;
    for (int e0 = 0; e0 < p.n_experts; e0 += 64) {
      const int e = e0 + lane;
      const int own = e < p.n_experts ? (int)(((int64_t)p.offsets[e + 1] - p.offsets[e] + BM - 1) / BM) : 0;
      total += __builtin_amdgcn_readlane((int)wave_sum_scan((uint32_t)own), 63);
    }
    l.real = (uint32_t)total * nt;
    l.zero = (uint32_t)((p.n_rows - p.offsets[p.n_experts] + BM - 1) / BM) * nt;
    steps = p.k / kStep;
  }
  l.full = l.real;
  l.rest = 0;
  l.parts = 1;
  if (p.parts != nullptr) {
    const uint32_t places = places_of(p.cus, BM), rest = l.real % places, parts = parts_of(rest, steps, places);
    if (parts > 1) {
      l.rest = rest;
      l.parts = parts;
      l.full = l.real - rest;
    }
  }
  return l;
}

// A workgroup's tile, or one part of it.
struct Share {
  uint32_t tile, part, parts, slot;
};
template <int MODE, int BM, int BN>
__device__ inline bool find_share(const ProductArgs& p, const TilePlan& l, uint32_t block, Share& s) {
  s.part = 0;
  s.parts = 1;
  if (block < l.full) {
    if constexpr (MODE == kMatrix) {
      // an expert's tiles over all XCDs: with an expert or two to an XCD the one
      // with the most rows was waited for (1538 us with popularities log-normal,
      // sigma 0.5, over 16 experts of 4096 x 4096; 1022 so)
      const uint32_t per = (uint32_t)((p.m + BM - 1) / BM) * (uint32_t)((p.n + BN - 1) / BN);
      const uint32_t first = block / per * per, here = l.full - first < per ? l.full - first : per;
      s.tile = first + (uint32_t)xcd_range_block(block - first, here);
    } else {
      s.tile = (uint32_t)xcd_range_block(block, l.full);
    }
    return true;
  }
  block -= l.full;
  if (block < l.rest * l.parts) {
    s.tile = l.full + block % l.rest;
    s.part = block / l.rest;
    s.parts = l.parts;
    s.slot = block % l.rest * l.parts + s.part;
    return true;
  }
  block -= l.rest * l.parts;
  s.tile = l.real + block;
  return block < l.zero;
}

// Where tile `id` of a product of rows lies.
template <int BM>
__device__ inline void find_tile(const ProductArgs& p, uint32_t nt, int lane, uint32_t id, TileAt& t) {
  const int E = p.n_experts;
  const uint32_t q = id / nt;
  int before = 0;
  for (int e = 0;; e += 64) {
    int own = 0;
    if (e + lane <= E) {
      const int64_t a = p.offsets[e + lane], b = e + lane < E ? (int64_t)p.offsets[e + lane + 1] : p.n_rows;
      own = (int)((b - a + BM - 1) / BM);
    }
    const int upto = (int)wave_sum_scan((uint32_t)own) + before;
    const uint64_t m = __ballot((uint32_t)upto > q);
    if (m != 0 || e + 64 > E) {  // (found: id is below the number of tiles)
      const int l = m != 0 ? __builtin_ctzll(m) : 0;
      const int mt = __builtin_amdgcn_readlane(own, l), first = __builtin_amdgcn_readlane(upto, l) - mt;
      t.expert = e + l;
      tile_in_group(id - (uint32_t)first * nt, (uint32_t)mt, nt, t);
      const int64_t a = p.offsets[t.expert], b = t.expert < E ? (int64_t)p.offsets[t.expert + 1] : p.n_rows;
      t.row0 = a + (int64_t)t.m * BM;
      t.rows = (int)(b - t.row0 < BM ? b - t.row0 : BM);
      return;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
}

// A tile: both operands, the result, and how much of it there is.
template <class T>
struct TileWork {
  Source<T> a, b;
  T* c;
  int c_rows, c_cols;
};

template <class T, int MODE, int BM, int BN>
__device__ inline TileWork<T> tile_work(const ProductArgs& p, int lane, uint32_t id) {
  const uint32_t nt = (uint32_t)((p.n + BN - 1) / BN);
  TileWork<T> o;
  TileAt t;
  if constexpr (MODE == kMatrix) {
    const uint32_t mt = (uint32_t)((p.m + BM - 1) / BM);
    t.expert = (int)(id / (mt * nt));
    tile_in_group(id % (mt * nt), mt, nt, t);
    const int64_t r0 = p.offsets[t.expert], m0 = (int64_t)t.m * BM;
    o.a.k = o.b.k = p.offsets[t.expert + 1] - r0;
    o.a.base = (const T*)p.a + r0 * p.lda + m0;
    o.b.base = (const T*)p.b + r0 * p.ldb;
    o.a.tile_rows = (int)(p.m - m0 < BM ? p.m - m0 : BM);
    o.c = (T*)p.c + (int64_t)t.expert * p.c_expert + m0 * p.ldc;
  } else {
    find_tile<BM>(p, nt, lane, id, t);
    o.a.k = o.b.k = t.expert < p.n_experts ? p.k : 0;
    o.a.base = (const T*)p.a + t.row0 * p.lda;
    o.b.base = (const T*)p.b + (int64_t)t.expert * p.b_expert;
    o.a.tile_rows = t.rows;
    o.c = (T*)p.c + t.row0 * p.ldc;
  }
  const int64_t n0 = (int64_t)t.n * BN;
  o.b.base += MODE == kRowsTrans ? n0 * p.ldb : n0;
  o.b.tile_rows = (int)(p.n - n0 < BN ? p.n - n0 : BN);
  o.a.ld = p.lda;
  o.b.ld = p.ldb;
  o.c += n0;
  o.c_rows = o.a.tile_rows;
  o.c_cols = o.b.tile_rows;
  return o;
}

// Four neighbouring columns of a result row, from column n of the tile.
template <class T>
__device__ inline void store_four(T* row, int n, int cols, f32x4 v) {
  T out[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = (T)v[e];
  if (n + 4 <= cols) {
    __builtin_memcpy(row + n, out, sizeof out);
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (n + e < cols) row[n + e] = out[e];
  }
}

template <class T, int MODE, int WIDTH, int BM, int BN, int WM, int WN, int SLOTS, bool PAST>
__global__ __launch_bounds__(64 * WM * WN) void expert_product_kernel(const ProductArgs p) {
  constexpr int THREADS = 64 * WM * WN;
  constexpr bool AKC = MODE != kMatrix, BKC = MODE == kRowsTrans;
  using OA = Operand<T, AKC, BM, THREADS>;
  using OB = Operand<T, BKC, BN, THREADS>;
  constexpr int BK = OA::BK;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int kSlots = WIDTH == 0 ? 2 : SLOTS, kSlot = OA::kBytes + OB::kBytes;
  constexpr int kAhead = kSlots - 1;
  __shared__ alignas(1024) uint8_t s_mem[kSlots][kSlot];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const TilePlan plan = plan_tiles<MODE, BM, BN>(p, lane);
  Share share;
  if (!find_share<MODE, BM, BN>(p, plan, blockIdx.x, share)) return;
  TileWork<T> work = tile_work<T, MODE, BM, BN>(p, lane, share.tile);
  // the steps of this part of the tile
  const int64_t all_steps = (work.a.k + BK - 1) / BK;
  const int64_t first = all_steps * share.part / share.parts, steps = all_steps * (share.part + 1) / share.parts;
  if (steps < all_steps) work.a.k = work.b.k = steps * BK;
  const Source<T>&sa = work.a, &sb = work.b;

  const int wm = w / WN, wn = w % WN;
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_byte*)&s_mem[0][0];
  Frags<OA, AKC, FM> from_a;
  Frags<OB, BKC, FN> from_b;
  // 16-row blocks of a wave: half of what the tile has where two groups of waves
  // share it (an expert's last tile may have few rows)
  const int fm = BM == kLarge ? (work.c_rows + 31) / 32 : FM;
  from_a.init(wm * fm * 16, lane);
  from_b.init(wn * (BN / WN), lane);

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  typename Mma<T>::frag fa[FM], fb[FN];
  auto read_frags = [&](uint32_t slot, int some) {
    from_b.read(slot + OA::kBytes, fb);
    from_a.read(slot, fa, some);
  };
  auto multiply_row = [&](int i) {
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = Mma<T>::run(fb[j], fa[i], acc[i][j]);
  };
  if constexpr (WIDTH != 0) {
    // Loads are started kAhead steps ahead: three, or one with two slots.  Every
    // wave starts its share of every step's, also of the kAhead steps past the last
    // (zeros), so that counting those still under way tells which step has arrived.
    Dma<OA, T, AKC, THREADS, WIDTH> da;
    Dma<OB, T, BKC, THREADS, WIDTH> db;
    constexpr int kLoadsA = da.kLoads, kLoads = da.kLoads + db.kLoads;
    da.init(sa, tid);
    db.init(sb, tid);
    // With (N, K) matrices of few rows an expert, whose rows are read side by side
    // 64 bytes at a time, tiles begin at different steps: beginning together they
    // asked the same few memory channels where rows are 4 KB or 8 KB apart (64 and
    // 128 rows for each of 32 experts, 2048 x 4096 bf16: 120 and 149 us, 109 and
    // 124 so; from 512 rows on, where tiles share rows, 0.96 to 1.02 of the rate).
    int64_t turn = 0;
    if (MODE == kRowsTrans && p.turn && sa.k % BK == 0 && steps > first)
      turn = (int64_t)(share.tile * 5u) % (steps - first);
    u32x4 rsrc_a, rsrc_b;
    uint32_t next;
    auto begin_loads = [&](int64_t kt) {
      const int64_t left = sa.k - kt * BK;
      if (left < BK) {
        da.cut(left, tid);
        db.cut(left, tid);
      }
      const int64_t at = kt >= steps ? kt : kt + turn < steps ? kt + turn : kt + turn - (steps - first);
      rsrc_a = da.at(at);
      rsrc_b = db.at(at);
      next = lds + (uint32_t)(kt & kAhead) * kSlot;
    };
    auto load = [&](int i) {
      if (i < kLoadsA) da.issue(next, rsrc_a, i, w);
      else db.issue(next + OA::kBytes, rsrc_b, i - kLoadsA, w);
    };
    for (int64_t kt = first; kt < first + kAhead; ++kt) {
      begin_loads(kt);
#pragma unroll
      for (int i = 0; i < kLoads; ++i) load(i);
    }
    if constexpr (WM * WN == 8) {
      // Two groups of four waves, one wave a SIMD each, half a step apart: one
      // multiplies, and starts loads in between, while the other reads fragments.
      constexpr int kBetween = (kLoads + FM - 1) / FM;  // loads between the products of two rows
      const bool second = w >= 4;
      wait_loads<2 * kLoads>();
      barrier();
      if (second) barrier();
      auto run = [&](auto whole) {
        for (int64_t kt = first; kt < steps; ++kt) {
          read_frags(lds + (uint32_t)(kt & 3) * kSlot, whole ? FM : fm);
          begin_loads(kt + 3);
          wait_reads();
          if (second) wait_loads<kLoads>();  // step kt + 1, which the first group reads next
          barrier();
          __builtin_amdgcn_s_setprio(1);
#pragma unroll
          for (int i = 0; i < FM; ++i) {
            if (whole || i < fm) multiply_row(i);
#pragma unroll
            for (int q = 0; q < kBetween; ++q)
              if (i * kBetween + q < kLoads) load(i * kBetween + q);  // the slot was last read two phases ago
            __builtin_amdgcn_sched_barrier(0);
          }
          __builtin_amdgcn_s_setprio(0);
          if (!second) wait_loads<2 * kLoads>();
          barrier();
        }
      };
      if (fm == FM) run(std::true_type{});
      else run(std::false_type{});
      if (!second) barrier();
    } else {
      for (int64_t kt = first; kt < steps; ++kt) {
        wait_reads();
        wait_loads<(kAhead - 1) * kLoads>();
        barrier();  // step kt has arrived, step kt - 1 has been read
        begin_loads(kt + kAhead);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) load(i);
        read_frags(lds + (uint32_t)(kt & kAhead) * kSlot, FM);
#pragma unroll
        for (int i = 0; i < FM; ++i) multiply_row(i);
      }
    }
    wait_loads<0>();
  } else {
    u32x4 ra[OA::kPieces], rb[OB::kPieces];
    if (first < steps) {
      load_pieces<OA, T, AKC>(sa, first, tid, ra);
      load_pieces<OB, T, BKC>(sb, first, tid, rb);
    }
    for (int64_t kt = first; kt < steps; ++kt) {
      const uint32_t slot = lds + (uint32_t)(kt & 1) * kSlot;
      store_pieces<OA, T, AKC>(sa, kt, slot, tid, ra, THREADS);
      store_pieces<OB, T, BKC>(sb, kt, slot + OA::kBytes, tid, rb, THREADS);
      if (kt + 1 < steps) {
        load_pieces<OA, T, AKC>(sa, kt + 1, tid, ra);
        load_pieces<OB, T, BKC>(sb, kt + 1, tid, rb);
      }
      // one barrier a step: the slot written next was last read before it
      __syncthreads();
      read_frags(slot, FM);
#pragma unroll
      for (int i = 0; i < FM; ++i) multiply_row(i);
    }
  }

  if constexpr (BM == kLarge || MODE == kMatrix) {
    if (share.parts > 1) {  // sums for the join, as the lanes hold them
      f32x4* part = (f32x4*)p.parts + (int64_t)share.slot * (BM * BN / 4) + w * (FM * FN * 64) + lane;
#pragma unroll
      for (int i = 0; i < FM; ++i)
        if (i < fm)
#pragma unroll
          for (int j = 0; j < FN; ++j) part[(i * FN + j) * 64] = acc[i][j];
      return;
    }
  }
  // Lane l holds row l % 16 and 4 neighbouring columns of each 16x16 result: by way
  // of LDS a wave's 16 rows leave as lines of 128 or 256 bytes (us, 8 bytes a lane
  // and so: 16 experts of 2048 rows, 4096 x 4096 bf16 996 and 957, 8 of 4096 rows, 256 x
  // 1024 51 and 38, matrix gradient of 16 experts of 7 or 8 rows, 4368 x 4032 191 and
  // 125).  PAST: a matrix gradient's, where all lines are whole, go past the caches (32
  // experts of 8 rows, 2048 x 4096 116 and 84, of 256 rows 283 and 187, 8 of 256 rows,
  // 1024 x 1024 10.4 and 9.1; lines in two parts, 64 of 2 rows, 1800 x 1368, 66 and 148).
  constexpr int kRow = 16 * FN * (int)sizeof(T), kPitch = kRow + 16, kLanes = kRow / 16, kOut = 16 / (int)sizeof(T);
  static_assert(WM * WN * 16 * kPitch <= kSlots * kSlot, "the waves' rows fit the slots");
  __syncthreads();  // (no wave reads or fills the slots any more)
  lds_byte* own = (lds_byte*)(uintptr_t)lds + w * (16 * kPitch);
  const int col = wn * (BN / WN) + lane % kLanes * kOut;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    if (i >= fm) break;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      T out[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = (T)acc[i][j][e];
      lds_byte* to = own + (lane & 15) * kPitch + (j * 16 + (lane >> 4) * 4) * (int)sizeof(T);
      if constexpr (sizeof(T) == 2) {
        u32x2 v;
        __builtin_memcpy(&v, out, 8);
        *(lds_u32x2*)to = v;
      } else {
        *(lds_u32x4*)to = __builtin_bit_cast(u32x4, acc[i][j]);
      }
    }
    wait_reads();
#pragma unroll
    for (int q = 0; q < 16 * kLanes / 64; ++q) {
      const int r = q * (64 / kLanes) + lane / kLanes, m = (wm * fm + i) * 16 + r;
      const u32x4 v = *(const lds_u32x4*)(own + r * kPitch + lane % kLanes * 16);
      if (m >= work.c_rows) continue;
      T* row = work.c + (int64_t)m * p.ldc + col;
      if (col + kOut <= work.c_cols) {
        store_slice<PAST>(row, __builtin_bit_cast(Slice<T>, v));
      } else {
        T out[kOut];
        __builtin_memcpy(out, &v, 16);
#pragma unroll
        for (int e = 0; e < kOut - 1; ++e)
          if (col + e < work.c_cols) row[e] = out[e];
      }
    }
    wait_reads();
  }
}

// Tiles cut along k: their parts are added in order.  A workgroup adds the i-th
// 16-row block of each wave of one tile, then of others.
template <class T, int MODE, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void expert_product_join_kernel(const ProductArgs p) {
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const TilePlan plan = plan_tiles<MODE, BM, BN>(p, lane);
  for (uint32_t b = blockIdx.x; b < plan.rest * FM; b += gridDim.x) {
    const uint32_t r = b / FM;
    const int i = (int)(b % FM);
    const TileWork<T> work = tile_work<T, MODE, BM, BN>(p, lane, plan.full + r);
    const int fm = BM == kLarge ? (work.c_rows + 31) / 32 : FM, m = ((w / WN) * fm + i) * 16 + (lane & 15);
    if (i >= fm || m >= work.c_rows) continue;
    const f32x4* part = (const f32x4*)p.parts + (int64_t)r * plan.parts * (BM * BN / 4) + w * (FM * FN * 64) +
                        i * FN * 64 + lane;
    f32x4 sum[FN];
#pragma unroll
    for (int j = 0; j < FN; ++j) sum[j] = part[j * 64];
    for (uint32_t k = 1; k < plan.parts; ++k)
#pragma unroll
      for (int j = 0; j < FN; ++j) sum[j] += part[(int64_t)k * (BM * BN / 4) + j * 64];
#pragma unroll
    for (int j = 0; j < FN; ++j)
      store_four(work.c + (int64_t)m * p.ldc, (w % WN) * (BN / WN) + (lane >> 4) * 4 + j * 16, work.c_cols, sum[j]);
  }
}

// Few rows an expert: the matrices' bytes are what counts.  16 x 64 tiles, and
// the waves of a workgroup take every fourth (or eighth) step of k, each through
// slots of its own and without barriers, so that many loads are under way; their sums
// are added in wave order at the end.
constexpr int kFewRows = 16, kFewCols = 64;
template <class T, int MODE, int WIDTH, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void expert_product_few_kernel(const ProductArgs p) {
  constexpr bool BKC = MODE == kRowsTrans;
  using OA = Operand<T, true, kFewRows, 64>;
  using OB = Operand<T, BKC, kFewCols, 64>;
  constexpr int BK = OA::BK, FN = kFewCols / 16;
  constexpr int kSlots = WIDTH ? 4 : 1, kSlot = OA::kBytes + OB::kBytes;
  static_assert(kSlots * kSlot >= FN * 64 * 16, "a wave's sums fit its slots");
  __shared__ alignas(1024) uint8_t s_mem[kWaves][kSlots][kSlot];

  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const TilePlan plan = plan_tiles<MODE, kFewRows, kFewCols>(p, lane);
  Share share;
  if (!find_share<MODE, kFewRows, kFewCols>(p, plan, blockIdx.x, share)) return;
  const TileWork<T> work = tile_work<T, MODE, kFewRows, kFewCols>(p, lane, share.tile);
  const Source<T>&sa = work.a, &sb = work.b;
  const uint32_t lds = (uint32_t)(uintptr_t)(lds_byte*)&s_mem[w][0][0];
  Frags<OA, true, 1> from_a;
  Frags<OB, BKC, FN> from_b;
  from_a.init(0, lane);
  from_b.init(0, lane);
  f32x4 acc[FN];
#pragma unroll
  for (int j = 0; j < FN; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  typename Mma<T>::frag fa[1], fb[FN];
  auto read_frags = [&](uint32_t slot) {
    from_a.read(slot, fa);
    from_b.read(slot + OA::kBytes, fb);
  };
  const int64_t steps = (sa.k + BK - 1) / BK;

  if constexpr (WIDTH != 0) {
    Dma<OA, T, true, 64, WIDTH> da;
    Dma<OB, T, BKC, 64, WIDTH> db;
    constexpr int kLoads = da.kLoads + db.kLoads;
    da.init(sa, lane);
    db.init(sb, lane);
    auto load = [&](int64_t i) {  // the wave's i-th step
      const int64_t kt = w + i * kWaves, left = sa.k - kt * BK;
      if (left < BK) {
        da.cut(left, lane);
        db.cut(left, lane);
      }
      const u32x4 ra = da.at(kt), rb = db.at(kt);
      const uint32_t next = lds + (uint32_t)(i & 3) * kSlot;
#pragma unroll
      for (int q = 0; q < da.kLoads; ++q) da.issue(next, ra, q, 0);
#pragma unroll
      for (int q = 0; q < db.kLoads; ++q) db.issue(next + OA::kBytes, rb, q, 0);
    };
    for (int i = 0; i < 3; ++i) load(i);
    for (int64_t i = 0; w + i * kWaves < steps; ++i) {
      wait_loads<2 * kLoads>();
      read_frags(lds + (uint32_t)(i & 3) * kSlot);
      load(i + 3);  // (into the slot read last time round)
      wait_reads();
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[j] = Mma<T>::run(fb[j], fa[0], acc[j]);
    }
    wait_loads<0>();
  } else {
    u32x4 ra[2][OA::kPieces], rb[2][OB::kPieces];
    auto load = [&](int64_t i, int q) {
      if (w + i * kWaves >= steps) return;
      load_pieces<OA, T, true>(sa, w + i * kWaves, lane, ra[q]);
      load_pieces<OB, T, BKC>(sb, w + i * kWaves, lane, rb[q]);
    };
    auto step = [&](int64_t i, int q) {
      if (w + i * kWaves >= steps) return;
      store_pieces<OA, T, true>(sa, w + i * kWaves, lds, lane, ra[q], 64);
      store_pieces<OB, T, BKC>(sb, w + i * kWaves, lds + OA::kBytes, lane, rb[q], 64);
      load(i + 2, q);
      wait_reads();  // (one wave: its own stores)
      read_frags(lds);
      wait_reads();
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[j] = Mma<T>::run(fb[j], fa[0], acc[j]);
    };
    load(0, 0);
    load(1, 1);
    for (int64_t i = 0; w + i * kWaves < steps; i += 2) {
      step(i, 0);
      step(i + 1, 1);
    }
  }

#pragma unroll
  for (int j = 0; j < FN; ++j) *(f32x4*)&s_mem[w][0][(j * 64 + lane) * 16] = acc[j];
  __syncthreads();
  if (w >= FN) return;
  f32x4 sum = *(const f32x4*)&s_mem[0][0][tid * 16];
#pragma unroll
  for (int k = 1; k < kWaves; ++k) sum += *(const f32x4*)&s_mem[k][0][tid * 16];
  const int m = lane & 15;
  if (m < work.c_rows) store_four(work.c + (int64_t)m * p.ldc, w * 16 + (lane >> 4) * 4, work.c_cols, sum);
}

template <int MODE, int BM, int BN>
int64_t tiles_of(const ProductArgs& p) {
  const int64_t nt = ceil_div(p.n, BN);
  return MODE == kMatrix ? ceil_div(p.m, BM) * nt * p.n_experts : (p.n_rows / BM + p.n_experts + 1) * nt;
}

// Whether tiles of a last round may be split: of a matrix gradient it is known
// here; of a product of rows, whose tiles are counted on the device, large ones
// if they take long beside the join that is then launched in any case, and rounds
// are few.  us with and without: 4096 x 2 rows, 8 experts 4096 x 4096 bf16 272
// and 312, 8192 x 2 of 2048 x 2048 149 and 162, 4093 x 4 of 5120 x 2048 346 and
// 383; matrix gradients of 4 experts of 32768 rows, 256 x 320 89 and 226, of
// 1024 rows 14 and 12: from 2048 rows on.
template <int MODE, int BM, int BN>
bool may_split(const ProductArgs& p) {
  const int64_t nt = ceil_div(p.n, BN), rows = p.n_rows / p.n_experts;
  if (MODE == kMatrix) {
    const int64_t real = ceil_div(p.m, BM) * nt * p.n_experts;
    const uint32_t places = places_of(p.cus, BM);
    return real <= INT32_MAX && (BM == kLarge || rows >= 2048) &&
           parts_of((uint32_t)real % places, rows / 32, places) > 1;
  }
  return BM == kLarge && rows >= 112 && p.k >= 1536 && p.n_rows / kLarge * nt < 8 * p.cus;
}
// The sums that split tiles leave: at most one a place.
template <int MODE, int BM, int BN>
size_t parts_bytes(const ProductArgs& p) {
  return may_split<MODE, BM, BN>(p) ? (size_t)places_of(p.cus, BM) * BM * BN * sizeof(float) : 0;
}

// Whether a matrix gradient's smaller tiles have two slots instead of four, so that
// more workgroups share a compute unit: where there are more of them than places, with
// 32-bit values (us with two and four: 32 experts of 64 rows, 2048 x 4096, 317 and 362,
// of 4096 rows 15071 and 15853; 4 of 32768, 256 x 320, 295 and 307), and with 16-bit ones
// of few rows, whose time is the results' (32 of 8 rows, 2048 x 4096, 83 and 115, of 320
// 218 and 251; 16 of 384, 1024 x 2048 34 and 39, 64 of 384, 512 x 512 32 and 31, of 512 40
// and 36).  With fewer, two slots only start loads later (4 of 1024 rows, 512 x 512 17.5
// and 10.8, 1024 x 1024 19.3 and 14.9).
constexpr int64_t kShortRows = 384;
template <class T>
bool two_slots(const ProductArgs& p, int64_t workgroups, uint32_t places) {
  return workgroups > places && (sizeof(T) == 4 || p.n_rows / p.n_experts <= kShortRows);
}

template <class T, int MODE, int WIDTH, int BM, int BN, int WM, int WN>
int launch_tiles(ProductArgs p, void* ws, size_t ws_bytes, hipStream_t stream) {
  const size_t need = parts_bytes<MODE, BM, BN>(p);
  if (need > 0 && (ws == nullptr || ws_bytes < need))
    return fail(FS_E_WORKSPACE, "fs_expert_product: workspace too small");
  p.parts = need > 0 ? static_cast<float*>(ws) : nullptr;
  const int64_t tiles = tiles_of<MODE, BM, BN>(p) + (need > 0 ? places_of(p.cus, BM) : 0);
  if (tiles * 64 * WM * WN > INT32_MAX) return fail(FS_E_INVALID, "fs_expert_product: too many tiles");
  auto launch = [&](auto slots, auto past) {
    hipLaunchKernelGGL((expert_product_kernel<T, MODE, WIDTH, BM, BN, WM, WN, decltype(slots)::value,
                                              decltype(past)::value>),
                       dim3((uint32_t)tiles), dim3(64 * WM * WN), 0, stream, p);
  };
  using Four = std::integral_constant<int, 4>;
  using Two = std::integral_constant<int, MODE == kMatrix && WIDTH != 0 && BM != kLarge ? 2 : 4>;
  using Past = std::integral_constant<bool, MODE == kMatrix>;
  const bool past = MODE == kMatrix && ((uintptr_t)p.c | (size_t)p.ldc * sizeof(T)) % 128 == 0;
  if (two_slots<T>(p, tiles, places_of(p.cus, BM))) past ? launch(Two{}, Past{}) : launch(Two{}, std::false_type{});
  else past ? launch(Four{}, Past{}) : launch(Four{}, std::false_type{});
  FS_CHECK_MAIN_LAUNCH("expert_product_kernel");
  if constexpr (BM == kLarge || MODE == kMatrix) {
    if (need > 0) {
      hipLaunchKernelGGL((expert_product_join_kernel<T, MODE, BM, BN, WM, WN>), dim3((uint32_t)p.cus),
                         dim3(64 * WM * WN), 0, stream, p);
      FS_CHECK_LAUNCH("expert_product_join_kernel");
    }
  }
  return FS_OK;
}

template <class T, int MODE, int WIDTH>
int launch_few(ProductArgs p, hipStream_t stream) {
  p.parts = nullptr;
  const int64_t tiles = tiles_of<MODE, kFewRows, kFewCols>(p);
  if (tiles * 512 > INT32_MAX) return fail(FS_E_INVALID, "fs_expert_product: too many tiles");
  // Eight waves where half of the chip has no tile, so that as many loads are under
  // way (us with 4 and 8: one row, 4096 x 4096 f32 28 and 24; two of 8 experts
  // 4095 x 4095 bf16, (K, N) 68 and 39, (N, K) 21 and 20; of 4096 x 4096 bf16, whose
  // loads need no registers, 16.0 and 16.4).
  if constexpr (sizeof(T) == 4 || WIDTH == 0) {
    if (2 * ceil_div(p.n, kFewCols) * std::min<int64_t>(p.n_rows, p.n_experts) <= p.cus) {
      hipLaunchKernelGGL((expert_product_few_kernel<T, MODE, WIDTH, 8>), dim3((uint32_t)tiles), dim3(512), 0, stream,
                         p);
      FS_CHECK_MAIN_LAUNCH("expert_product_few_kernel");
      return FS_OK;
    }
  }
  hipLaunchKernelGGL((expert_product_few_kernel<T, MODE, WIDTH, 4>), dim3((uint32_t)tiles), dim3(256), 0, stream, p);
  FS_CHECK_MAIN_LAUNCH("expert_product_few_kernel");
  return FS_OK;
}

// Which tiles.  The larger, the fewer times operands are read and the nearer to
// the matrix cores' rate, if rows fill them and there are enough for the chip
// (kFill).  us, 32 experts 2048 x 4096, bf16 where not said otherwise, rows an
// expert, all alike; tiles few / 64 x 128 / 128 x 128 / 256 x 256:
//   matrices (K, N)      2: 102  93  89  88     4: 104  95  91  88    32: 143 101 101  92
//     unlike popularity  1:  60  64  64  74     2:  77  84  80  76     4:  82  89  85  78
//   (N, K), "trans"      2:  96  93  95  97    16: 103  97  99  99    32: 146 101 104 102
//                       48: 178 109 111 106   112:  -  178 127 122
//   2046 x 4094, (K, N)  6: 103  89            12: 109  92
//     (N, K)             6: 112 129            12: 121 134            16: 127 137
//   2047 x 4095, (K, N)  6: 109  96            12: 117  98
//     (N, K)             6: 129 155            12: 137 157            16: 142 157
//   float32, (K, N)     16: 195 285 500        32: 263 286 504
//     unlike popularity 32: 302 276 486       768:  - 1513 1498 (16 experts)
//   matrix gradient    256:  -   -  188 194   384:  -   -  308 268   640:  -   -  412 365
//     unlike popularity 320: -   -  226 221   384:  -   -  298 268   640:  -   -  451 363
//     16 of 1024 x 2048 384: -   -   34  39   448:  -   -   44  43
//     2046 x 4094       32:  -   -  176 186    48:  -   -  207 192    64:  -   -  208 194
// Of products of rows, 8 experts of 1024 rows, 1024 columns of k, 128 / 256: with
// 160 large tiles 39 / 32, 192 41 / 32, 128 26 / 29 (64 and 128 rows: 8 experts of 64
// rows, 256 tiles of 128 17 / 18, of 96 rows 25 / 20, 128 tiles of 96 rows 13 / 15).
// Fewer large tiles are split along k (8 experts of 1024 rows, popularities
// unlike, and alike): k 1536, 128 tiles 49 / 42 to 47, alike 41 / 46; k 2048, 128 tiles
// 62 / 51 to 55, 50 / 60, 96 tiles 44 to 48 / 56, 42 / 54; k 4096, 128 tiles 119 / 91 to 100,
// 93 / 93, 64 tiles 68 / 63, 54 / 64.  A matrix gradient's along the rows (4 experts):
// 96 tiles of 4096 rows 77 / 66, of 6144 115 / 87, of 1024 20 / 26; 64 tiles of 8192 rows
// 96 / 83; 160 tiles of 1024 rows 26 / 27, of 4096 110 / 87.
// 1.5 rounds of large tiles lose to smaller ones (64 experts of 1536 columns, 8
// rows: 87, 64 x 128 73).  One token (8 experts of 64, 4096 columns): few 23, 64
// x 128 23, 256 x 256 42; (1 of 8, 4096 x 4096): 12, 28, 72; 16 tokens, 2 of 8,
// 1024 x 1024: 9, 12.
constexpr int64_t kFill = 256;

enum Tiles { kFew, kTiles64, kTiles128, kTiles256 };
template <int MODE>
Tiles choose_tiles(const ProductArgs& p, bool half, int width) {
  const int64_t rows = p.n_rows / p.n_experts, active = std::min<int64_t>(p.n_rows, p.n_experts);
  // large tiles that do not fill the chip pay if their steps can be split
  if constexpr (MODE == kMatrix) {
    const int64_t tiles256 = tiles_of<MODE, kLarge, kLarge>(p);
    if (half && width != 0 && rows > (width == 16 ? kShortRows : 50) &&
        (tiles256 >= 160 || (tiles256 >= 96 && rows >= 6144)))
      return kTiles256;
    return tiles_of<MODE, 128, 128>(p) >= kFill ? kTiles128 : kTiles64;
  }
  const int64_t tiles256 = ceil_div(p.n, kLarge) * std::max(active, p.n_rows / kLarge);
  const int64_t tiles128 = ceil_div(p.n, 128) * std::max(active, p.n_rows / 128);
  const int64_t tiles64 = ceil_div(p.n, 128) * std::max(active, p.n_rows / 64);
  if (half && width != 0 &&
      (rows >= 112 ? tiles256 >= 160 || (p.k >= 1536 && tiles256 * p.k >= 192 * 1024)
                   : rows >= (MODE == kRowsNon ? 4 : 40) && tiles256 >= 2 * kFill))
    return kTiles256;
  if (rows < (!half ? 20 : width == 16 && tiles64 >= kFill ? 4 : 12)) return kFew;
  return rows >= (half ? 40 : 768) && tiles128 >= kFill ? kTiles128 : kTiles64;
}

template <class T, int MODE, int WIDTH>
int launch_product(const ProductArgs& p, void* ws, size_t ws_bytes, hipStream_t stream) {
  switch (choose_tiles<MODE>(p, sizeof(T) == 2, WIDTH)) {
    case kFew:
      if constexpr (MODE != kMatrix) return launch_few<T, MODE, WIDTH>(p, stream);
      break;
    case kTiles64: return launch_tiles<T, MODE, WIDTH, 64, 128, 2, 2>(p, ws, ws_bytes, stream);
    case kTiles128: return launch_tiles<T, MODE, WIDTH, 128, 128, 2, 2>(p, ws, ws_bytes, stream);
    case kTiles256:
      if constexpr (sizeof(T) == 2 && WIDTH != 0)
        return launch_tiles<T, MODE, WIDTH, kLarge, kLarge, 2, 4>(p, ws, ws_bytes, stream);
  }
  return fail(FS_E_INVALID, "fs_expert_product: no tiles");
}

// Workspace for any alignment of the operands.
template <int MODE>
size_t product_workspace(const ProductArgs& p, bool half) {
  size_t most = 0;
  for (int width : {16, 4, 0}) {
    size_t need = 0;
    switch (choose_tiles<MODE>(p, half, width)) {
      case kFew: break;
      case kTiles64: need = parts_bytes<MODE, 64, 128>(p); break;
      case kTiles128: need = parts_bytes<MODE, 128, 128>(p); break;
      case kTiles256: need = parts_bytes<MODE, kLarge, kLarge>(p);
    }
    most = std::max(most, need);
  }
  return most;
}

template <class T, int MODE>
int launch_product(const ProductArgs& p, void* ws, size_t ws_bytes, hipStream_t stream) {
  // straight to LDS: rows and ends of rows on whole loads, and offsets within a
  // step that fit
  const int64_t s = sizeof(T), reach = MODE == kMatrix ? kRowBytes / s : kLarge;
  auto whole = [&](int64_t width) {
    const int64_t ends = (MODE == kMatrix ? p.m : p.k) | (MODE == kRowsTrans ? p.k : p.n);
    const int64_t starts = (int64_t)(uintptr_t)p.a | (int64_t)(uintptr_t)p.b;
    return ((starts | (p.lda | p.ldb | p.b_expert | ends) * s) & (width - 1)) == 0;
  };
  const bool near = reach * std::max(p.lda, p.ldb) * s < (int64_t)kInBuffer;
  if (near && whole(16)) return launch_product<T, MODE, 16>(p, ws, ws_bytes, stream);
  if (near && whole(4)) return launch_product<T, MODE, 4>(p, ws, ws_bytes, stream);
  return launch_product<T, MODE, 0>(p, ws, ws_bytes, stream);
}

template <int MODE>
int launch_product_type(int val_t, const ProductArgs& p, void* ws, size_t ws_bytes, hipStream_t stream) {
  switch (val_t) {
    case FS_F16: return launch_product<_Float16, MODE>(p, ws, ws_bytes, stream);
    case FS_BF16: return launch_product<__bf16, MODE>(p, ws, ws_bytes, stream);
    case FS_F32: return launch_product<float, MODE>(p, ws, ws_bytes, stream);
  }
  return fail(FS_E_INVALID, "fs_expert_product: value types are FS_F16, FS_BF16 and FS_F32");
}

int check_product(const char* who, int64_t n_rows, int64_t n_experts, int64_t a, int64_t b, int trans) {
  if (n_rows < 0 || n_rows > INT32_MAX || n_experts < 1 || n_experts > INT32_MAX || a < 0 || b < 0 ||
      a > INT32_MAX || b > INT32_MAX || (trans != 0 && trans != 1))
    return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
  return FS_OK;
}

// Compute units of the current device (cached per device id; threads that ask
// at once store the same value).
int compute_units() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
  int v = cached[dev].load(std::memory_order_relaxed);
  if (v == 0) {
    if (hipDeviceGetAttribute(&v, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || v <= 0) v = 256;
    cached[dev].store(v, std::memory_order_relaxed);
  }
  return v;
}

ProductArgs product_sizes(int trans, int64_t n_rows, int64_t n_experts, int64_t inner, int64_t outer, bool matrix) {
  ProductArgs p{};
  p.n_rows = n_rows;
  p.n_experts = (int)n_experts;
  p.m = trans ? outer : inner;
  p.n = matrix && trans ? inner : outer;
  p.k = inner;
  p.cus = compute_units();
  p.turn = n_rows / n_experts <= 256;
  return p;
}

}  // namespace
}  // namespace fs

extern "C" size_t fs_expert_product_workspace_bytes(int val_t, int trans, int64_t n_rows, int64_t n_experts,
                                                    int64_t inner, int64_t outer) {
  using namespace fs;
  if (check_product("", n_rows, n_experts, inner, outer, trans) != FS_OK || n_rows == 0 || outer == 0) return 0;
  const ProductArgs p = product_sizes(trans, n_rows, n_experts, inner, outer, false);
  const bool half = val_t == FS_F16 || val_t == FS_BF16;
  return trans ? product_workspace<kRowsTrans>(p, half) : product_workspace<kRowsNon>(p, half);
}

extern "C" int fs_expert_product(int val_t, int trans, int64_t n_rows, int64_t n_experts, int64_t inner, int64_t outer,
                                 const void* rows, int64_t ldr, const void* matrices, const int32_t* offsets, void* out,
                                 void* ws, size_t ws_bytes, hipStream_t stream) {
  using namespace fs;
  if (int rc = check_product("fs_expert_product", n_rows, n_experts, inner, outer, trans)) return rc;
  if (n_rows == 0 || outer == 0) return FS_OK;
  if (!offsets || !out || ldr < 0 || (inner > 0 && (!rows || !matrices)))
    return fail(FS_E_INVALID, "fs_expert_product: bad pointer or stride");
  ProductArgs p = product_sizes(trans, n_rows, n_experts, inner, outer, false);
  p.a = rows;
  p.b = matrices;
  p.c = out;
  p.offsets = offsets;
  p.lda = ldr;
  p.ldb = trans ? inner : outer;
  p.ldc = outer;
  p.b_expert = inner * outer;
  return trans ? launch_product_type<kRowsTrans>(val_t, p, ws, ws_bytes, stream)
               : launch_product_type<kRowsNon>(val_t, p, ws, ws_bytes, stream);
}

extern "C" size_t fs_expert_product_grad_matrices_workspace_bytes(int val_t, int trans, int64_t n_rows,
                                                                  int64_t n_experts, int64_t inner, int64_t outer) {
  using namespace fs;
  if (check_product("", n_rows, n_experts, inner, outer, trans) != FS_OK || inner == 0 || outer == 0) return 0;
  const ProductArgs p = product_sizes(trans, n_rows, n_experts, inner, outer, true);
  return product_workspace<kMatrix>(p, val_t == FS_F16 || val_t == FS_BF16);
}

extern "C" int fs_expert_product_grad_matrices(int val_t, int trans, int64_t n_rows, int64_t n_experts, int64_t inner,
                                               int64_t outer, const void* grad, int64_t ldg, const void* rows,
                                               int64_t ldr, const int32_t* offsets, void* grad_matrices, void* ws,
                                               size_t ws_bytes, hipStream_t stream) {
  using namespace fs;
  if (int rc = check_product("fs_expert_product_grad_matrices", n_rows, n_experts, inner, outer, trans)) return rc;
  if (inner == 0 || outer == 0) return FS_OK;
  if (!offsets || !grad_matrices || ldg < 0 || ldr < 0 || (n_rows > 0 && (!grad || !rows)))
    return fail(FS_E_INVALID, "fs_expert_product_grad_matrices: bad pointer or stride");
  ProductArgs p = product_sizes(trans, n_rows, n_experts, inner, outer, true);
  p.a = trans ? grad : rows;
  p.lda = trans ? ldg : ldr;
  p.b = trans ? rows : grad;
  p.ldb = trans ? ldr : ldg;
  p.c = grad_matrices;
  p.ldc = p.n;
  p.c_expert = inner * outer;
  p.offsets = offsets;
  return launch_product_type<kMatrix>(val_t, p, ws, ws_bytes, stream);
}
