// embedding.hip — embedding lookup with scaling, and its gradient.
//
// out[t] = scale * table[ids[t]], a product with a selection matrix of one
// entry a row; ids outside the table give a zero row.  The gradient is the
// transposed product, grad_table[v] = scale * sum over the t with ids[t] = v of
// grad[t]: positions sorted by token (select_sort.hip, stable), then one sum a
// table row over its segment, in position order, so results do not change from
// run to run.  Rows without tokens are written as zeros in the same pass, of few
// tokens beside their sort.
//
// A row of up to 64 tokens is summed at once.  A longer segment (tokens
// follow a Zipf law: the first ones occur thousands of times in a batch) is cut
// at multiples of 64 sorted positions; each chunk sums its part into the
// workspace, and in a second launch each of four waves adds every fourth of a
// row's parts, and one the four sums, in a fixed order.
#include <type_traits>

#include "select_rows.hpp"

namespace fs {
namespace {

constexpr int kLong = 64;  // tokens of a row that are summed at once, and positions a chunk

// Bound by the rows' bytes: lpr lanes a row (a power of two, up to the
// workgroup), so that short rows fill waves too, and one pass in 16-byte slices.
// 32768 tokens of a Zipf law, rows of 4096 bf16: 82 us, 4.4 TB/s of distinct rows
// read and rows written, 6.6 TB/s counting repeated ones, which come from the
// caches.  One token: a launch, 3 us.
template <class V, class Id>
__global__ __launch_bounds__(256) void embedding_kernel(const V* __restrict__ table, int64_t ldt, int64_t n_rows,
                                                        const Id* __restrict__ ids, int64_t n, int64_t width, int lpr,
                                                        typename Elem<V>::acc scale, V* __restrict__ out) {
  constexpr int E = Slice<V>::n;
  const int lane = threadIdx.x & (lpr - 1);
  const int64_t t = row_block() * (256 / lpr) + threadIdx.x / lpr;
  if (t >= n) return;
  const int64_t id = (int64_t)ids[t];
  const bool in = (uint64_t)id < (uint64_t)n_rows;
  const V* row = table + (in ? id : 0) * ldt;
  V* o = out + t * width;
  const int64_t slices = slices_of<V>(width);
#pragma unroll 2
  for (int64_t c = lane; c < slices; c += lpr) {
    const int64_t h = slice_start<V>(c, width);
    Slice<V> s{};
    if (in) s = load_slice(row + h);
#pragma unroll
    for (int e = 0; e < E; ++e) s.v[e] = in ? (V)(widen(s.v[e]) * scale) : (V)0;
    store_slice(o + h, s);
  }
  for (int64_t h = slices > 0 ? width : lane; h < width; h += lpr) o[h] = in ? (V)(widen(row[h]) * scale) : (V)0;
}

// First index with keys[i] >= key (n if none), by the whole wave: 64 probes a step.
__device__ inline int64_t wave_lower_bound(const uint32_t* __restrict__ keys, int64_t n, uint32_t key, int lane) {
  int64_t lo = 0, hi = n;
  while (hi - lo > 64) {
    const int64_t step = (hi - lo + 63) / 64, p = lo + step * (lane + 1) - 1;
    const int below = __popcll(__ballot(p < hi && keys[p < hi ? p : lo] < key));
    lo += step * below;
    hi = lo + step < hi ? lo + step : hi;
  }
  if (lo > hi) lo = hi;
  const int64_t p = lo + lane;
  return lo + __popcll(__ballot(p < hi && keys[p < hi ? p : 0] < key));
}

// Sum over the positions t0..t1 (held by the lanes) of the rows' slices from
// element h, in position order, the loads of several rows in flight: six of
// 16-bit values, for which eight leave registers for 5 waves a SIMD (65536 tokens
// x 2048, inputs not in cache: 214 and 224 us; sixteen 549), eight of others.
template <class V>
__device__ inline void sum_slices(const V* __restrict__ grad, int64_t ldg, int pos, int t0, int t1, int64_t h,
                                  typename Elem<V>::acc (&acc)[Slice<V>::n]) {
  constexpr int E = Slice<V>::n, kAtOnce = sizeof(V) == 2 ? 6 : 8;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0;
  auto row = [&](int t) { return load_slice(grad + (int64_t)__builtin_amdgcn_readlane(pos, t) * ldg + h); };
  auto add = [&](const Slice<V>& s) {
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += widen(s.v[e]);
  };
  int t = t0;
  for (; t + kAtOnce <= t1; t += kAtOnce) {
    Slice<V> s[kAtOnce];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) s[q] = row(t + q);
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) add(s[q]);
  }
  if (t < t1) {
    Slice<V> s[kAtOnce];
#pragma unroll
    for (int q = 0; q < kAtOnce - 1; ++q)
      if (t + q < t1) s[q] = row(t + q);
#pragma unroll
    for (int q = 0; q < kAtOnce - 1; ++q)
      if (t + q < t1) add(s[q]);
  }
}
// The same of one element, for rows shorter than a slice.
template <class V>
__device__ inline typename Elem<V>::acc sum_element(const V* __restrict__ grad, int64_t ldg, int pos, int t0, int t1,
                                                    int64_t h, bool in) {
  typename Elem<V>::acc a = 0;
  for (int t = t0; t < t1; ++t) {
    const V* row = grad + (int64_t)__builtin_amdgcn_readlane(pos, t) * ldg;
    if (in) a += widen(row[h]);
  }
  return a;
}

// O = V, or float for 16-bit V: a slice of sums leaves as one or two stores.
template <class V, bool PAST, class O, class A>
__device__ inline void store_sums(O* p, const A (&acc)[Slice<V>::n], A scale) {
  constexpr int E = Slice<V>::n, EO = Slice<O>::n;
#pragma unroll
  for (int k = 0; k < E / EO; ++k) {
    Slice<O> s;
#pragma unroll
    for (int e = 0; e < EO; ++e) s.v[e] = (O)(acc[k * EO + e] * scale);
    store_slice<PAST>(p + k * EO, s);
  }
}

// A wave's share of one sum of rows: slices first, first + stride, ...  A sum of
// no rows is zero whatever the scale: infinite, NaN or negative ones give no NaN
// and no -0 in table rows without tokens.
template <bool PAST, class V, class O>
__device__ inline void sum_rows(const V* __restrict__ grad, int64_t ldg, int pos, int t0, int t1, int64_t width,
                                int64_t first, int64_t stride, int lane, typename Elem<V>::acc scale, O* out) {
  const int64_t slices = slices_of<V>(width);
  if (t0 >= t1) scale = 0;
  typename Elem<V>::acc acc[Slice<V>::n];
  for (int64_t c = first; c < slices; c += stride) {  // (the same number of times for the lanes that go on)
    const int64_t h = slice_start<V>(c + lane < slices ? c + lane : slices - 1, width);
    sum_slices(grad, ldg, pos, t0, t1, h, acc);
    store_sums<V, PAST>(out + h, acc, scale);
  }
  if (slices == 0 && first == 0) {
    const auto a = sum_element(grad, ldg, pos, t0, t1, lane, lane < width);
    if (lane < width) out[lane] = (O)(a * scale);
  }
}

// wpr waves share a row (or a chunk), 64 slices each at a time, and go through
// block_rows rows one after the other.  Bound by the bytes where the table is
// large: 65536 tokens of a Zipf law, 131072 rows of 2048 bf16, 806 MB, 179 us of
// the call's 213 (4.5 TB/s; sort 22, join 11); 4095 tokens, 20011 rows of 1001
// float32, 97 MB, 33 us in all (the sort and its zeros, the rows with tokens, join 4).
// FILLED: rows below `filled` hold zeros already.
template <class V, class O, bool PAST, bool FILLED>
__global__ __launch_bounds__(256) void embedding_grad_kernel(
    const V* __restrict__ grad, int64_t ldg, const uint32_t* __restrict__ keys, const int32_t* __restrict__ order,
    int64_t n, int64_t n_rows, int64_t width, typename Elem<V>::acc scale, int64_t padding, int wpr, int block_rows,
    int64_t chunk_blocks, int64_t n_chunks, int64_t filled, O* __restrict__ out,
    typename Elem<V>::acc* __restrict__ parts) {
  using A = typename Elem<V>::acc;
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t first = (int64_t)(w % wpr) * 64, stride = (int64_t)wpr * 64;
  const int groups = 4 / wpr;

  const int64_t block = row_block();
  if (block < chunk_blocks) {  // parts of long segments
    const int64_t chunk = block * groups + w / wpr;
    if (chunk >= n_chunks) return;
    const int64_t c0 = chunk * kLong;
    const int cnt = (int)(n - c0 < kLong ? n - c0 : kLong);
    const uint32_t kk = lane < cnt ? keys[c0 + lane] : 0xffffffffu;
    const int pos = lane < cnt ? order[c0 + lane] : 0;
    const uint32_t kl = (uint32_t)__builtin_amdgcn_readfirstlane((int)kk);
    const uint32_t kr = (uint32_t)__builtin_amdgcn_readlane((int)kk, cnt - 1);
    const uint64_t at_l = __ballot(kk == kl), at_r = __ballot(kk == kr);
    int64_t start = c0;
    if (c0 > 0) start = c0 - __popcll(__ballot(keys[c0 - 64 + lane] == kl));  // (c0 is a multiple of 64)
    const bool enters = start < c0;
    auto is_summed = [&](uint32_t k) { return (int64_t)k < n_rows && (int64_t)k != padding; };
    auto is_long = [&](int64_t s, uint32_t k) { return is_summed(k) && s + kLong < n && keys[s + kLong] == k; };
    const bool left = enters && (start == c0 - 64 ? is_summed(kl) : is_long(start, kl));
    const int f = __builtin_ctzll(at_r);
    const bool right = (f > 0 || !enters) && is_long(c0 + f, kr);
    A* part = parts + chunk * 2 * width;
    if (left) sum_rows<PAST>(grad, ldg, pos, 0, __popcll(at_l), width, first, stride, lane, (A)1, part);
    if (right) sum_rows<PAST>(grad, ldg, pos, f, cnt, width, first, stride, lane, (A)1, part + width);
    return;
  }

  const int64_t v0 = ((block - chunk_blocks) * groups + w / wpr) * block_rows;
  if (v0 >= n_rows) return;
  // a window of 64 sorted positions from the first row's on
  int64_t wb = wave_lower_bound(keys, n, (uint32_t)v0, lane);
  uint32_t kk;
  int pos;
  auto window = [&] {
    kk = wb + lane < n ? keys[wb + lane] : 0xffffffffu;
    pos = wb + lane < n ? order[wb + lane] : 0;
  };
  window();
  for (int r = 0; r < block_rows && v0 + r < n_rows; ++r) {
    const uint32_t v = (uint32_t)(v0 + r);
    while (__ballot(kk < v) == ~0ull) {
      wb += 64;
      window();
    }
    uint64_t m = __ballot(kk == v);
    if (FILLED && m == 0 && (int64_t)v < filled) continue;
    if (m >> 63) {  // the window may cut the segment: begin it there
      wb += __builtin_ctzll(m);
      window();
      m = __ballot(kk == v);
      if (m == ~0ull && wb + kLong < n && keys[wb + kLong] == v) {
        // a long segment: the chunks sum it, or nobody
        if ((int64_t)v == padding)
          sum_rows<PAST>(grad, ldg, pos, 0, 0, width, first, stride, lane, scale, out + (int64_t)v * width);
        wb = wave_lower_bound(keys, n, v + 1, lane);
        window();
        continue;
      }
    }
    const int t0 = m != 0 ? __builtin_ctzll(m) : 0;
    const int t1 = (int64_t)v == padding ? t0 : t0 + __popcll(m);
    sum_rows<PAST>(grad, ldg, pos, t0, t1, width, first, stride, lane, scale, out + (int64_t)v * width);
  }
}

// Rows of long segments: the chunk in which one starts adds its parts, the
// first chunk's second slot and the first slots of the chunks after it.  The
// waves of a workgroup take every kJoinWaves-th part of 256 columns, eight
// loads in flight, and are added in wave order.
constexpr int kJoinWaves = 4;
template <class O, class A>
__global__ __launch_bounds__(64 * kJoinWaves) void embedding_grad_join_kernel(
    const uint32_t* __restrict__ keys, int64_t n, int64_t n_rows, int64_t width, A scale, int64_t padding,
    const A* __restrict__ parts, O* __restrict__ out) {
  constexpr int C = 4, kAtOnce = 8;
  __shared__ A s_sum[kJoinWaves - 1][C][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t chunk = (int64_t)blockIdx.z * gridDim.x + blockIdx.x, c0 = chunk * kLong;
  if (c0 + kLong >= n) return;  // the last chunk starts none that leaves it
  const uint32_t kr = keys[c0 + kLong - 1];
  if (keys[c0 + kLong] != kr || (int64_t)kr >= n_rows || (int64_t)kr == padding) return;
  if (c0 > 0 && keys[c0 - 1] == kr) return;  // starts before
  const int f = __builtin_ctzll(__ballot(keys[c0 + lane] == kr));
  if (c0 + f + kLong >= n || keys[c0 + f + kLong] != kr) return;  // summed at once
  const int64_t end = wave_lower_bound(keys, n, kr + 1, lane);
  const int64_t count = (end - 1) / kLong - chunk + 1;  // chunks that hold it
  int64_t h[C];
#pragma unroll
  for (int u = 0; u < C; ++u) {
    const int64_t own = (int64_t)blockIdx.y * 64 * C + u * 64 + lane;
    h[u] = own < width ? own : width - 1;
  }
  auto part = [&](int64_t k) { return parts + ((chunk + k) * 2 + (k == 0 ? 1 : 0)) * width; };
  A sum[C] = {};
  for (int64_t k = w; k < count; k += kJoinWaves * kAtOnce) {
    A v[kAtOnce][C];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q)
      if (k + q * kJoinWaves < count)
#pragma unroll
        for (int u = 0; u < C; ++u) v[q][u] = part(k + q * kJoinWaves)[h[u]];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q)
      if (k + q * kJoinWaves < count)
#pragma unroll
        for (int u = 0; u < C; ++u) sum[u] += v[q][u];
  }
  if (w > 0)
#pragma unroll
    for (int u = 0; u < C; ++u) s_sum[w - 1][u][lane] = sum[u];
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int u = 0; u < C; ++u) {
    A total = sum[u];
#pragma unroll
    for (int k = 0; k < kJoinWaves - 1; ++k) total += s_sum[k][u][lane];
    out[(int64_t)kr * width + h[u]] = (O)(total * scale);
  }
}

struct GradLayout {
  size_t sort, keys, order, parts, bytes;
};
GradLayout grad_layout(int val_t, int64_t n, int64_t n_rows, int64_t width) {
  auto up = [](size_t b) { return (b + 255) / 256 * 256; };
  GradLayout l{};
  l.sort = 0;
  l.keys = up(select_sort_bytes(n, n_rows));
  l.order = l.keys + up((size_t)n * 4);
  l.parts = l.order + up((size_t)n * 4);
  l.bytes = l.parts;
  if (n > kLong) l.bytes += (size_t)ceil_div(n, kLong) * 2 * (size_t)width * (val_t == FS_F64 ? 8 : 4);
  return l;
}

int check_sizes(const char* who, int64_t n, int64_t n_rows, int64_t width) {
  if (n < 0 || n > INT32_MAX || n_rows < 0 || n_rows >= INT32_MAX || width < 0 || width > 65535 * 256)
    return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
  return FS_OK;
}

}  // namespace
}  // namespace fs

extern "C" int fs_embedding(int val_t, int id_t, int64_t n, int64_t n_rows, int64_t width, const void* table,
                            int64_t ldt, const void* ids, double scale, void* out, hipStream_t stream) {
  using namespace fs;
  if (int rc = check_sizes("fs_embedding", n, n_rows, width)) return rc;
  if (id_t != FS_I32 && id_t != FS_I64) return fail(FS_E_INVALID, "fs_embedding: bad type code");
  if (n == 0 || width == 0) return FS_OK;
  if ((n_rows > 0 && !table) || !ids || !out || ldt < 0)
    return fail(FS_E_INVALID, "fs_embedding: bad pointer or stride");
  return with_value_type(val_t, "fs_embedding", [&](auto v) -> int {
    using V = decltype(v);
    using A = typename Elem<V>::acc;
    const int lpr = lanes_per_row(slices_of<V>(width));
    const dim3 grid = row_grid(ceil_div(n, 256 / lpr));
    auto launch = [&](auto id) {
      using Id = decltype(id);
      hipLaunchKernelGGL((embedding_kernel<V, Id>), grid, dim3(256), 0, stream, (const V*)table, ldt, n_rows,
                         (const Id*)ids, n, width, lpr, (A)scale, (V*)out);
    };
    if (id_t == FS_I64) launch(int64_t(0));
    else launch(int32_t(0));
    FS_CHECK_MAIN_LAUNCH("embedding_kernel");
    return FS_OK;
  });
}

extern "C" size_t fs_embedding_grad_workspace_bytes(int val_t, int64_t n, int64_t n_rows, int64_t width) {
  if (n <= 0 || n > INT32_MAX || n_rows <= 0 || n_rows >= INT32_MAX || width <= 0) return 0;
  return fs::grad_layout(val_t, n, n_rows, width).bytes;
}

extern "C" int fs_embedding_grad(int val_t, int out_t, int id_t, int64_t n, int64_t n_rows, int64_t width,
                                 const void* grad, int64_t ldg, const void* ids, double scale, int64_t padding,
                                 void* out, void* ws, size_t ws_bytes, hipStream_t stream) {
  using namespace fs;
  if (int rc = check_sizes("fs_embedding_grad", n, n_rows, width)) return rc;
  if (id_t != FS_I32 && id_t != FS_I64) return fail(FS_E_INVALID, "fs_embedding_grad: bad type code");
  if (out_t != val_t && !(out_t == FS_F32 && (val_t == FS_F16 || val_t == FS_BF16)))
    return fail(FS_E_INVALID, "fs_embedding_grad: the result has the gradient's type or float32");
  if (n_rows == 0 || width == 0) return FS_OK;
  if (!out || (n > 0 && (!grad || !ids)) || ldg < 0)
    return fail(FS_E_INVALID, "fs_embedding_grad: bad pointer or stride");
  const GradLayout l = grad_layout(val_t, n, n_rows, width);
  if (n > 0 && (ws == nullptr || ws_bytes < l.bytes))
    return fail(FS_E_WORKSPACE, "fs_embedding_grad: workspace too small");
  uint8_t* w = static_cast<uint8_t*>(ws);
  uint32_t* keys = n > 0 ? reinterpret_cast<uint32_t*>(w + l.keys) : nullptr;
  int32_t* order = n > 0 ? reinterpret_cast<int32_t*>(w + l.order) : nullptr;
  if (const int rc = with_value_type(val_t, "fs_embedding_grad", [](auto) -> int { return FS_OK; })) return rc;
  int64_t filled = 0;  // rows that the sort's launches write zeros to
  if (n > 0) {
    const int64_t row_bytes = width * (out_t == FS_F64 ? 8 : out_t == FS_F32 ? 4 : 2);
    filled = std::min(n_rows, select_sort_fill_bytes(n) / row_bytes);
    const int rc = select_sort(ids, id_t, n, n_rows, keys, order, nullptr, nullptr, w, stream, out, filled * row_bytes);
    if (rc != FS_OK) return rc;
  }
  return with_value_type(val_t, "fs_embedding_grad", [&](auto v) -> int {
    using V = decltype(v);
    using A = typename Elem<V>::acc;
    auto run = [&](auto o) -> int {
      using O = decltype(o);
      A* parts = n > 0 ? reinterpret_cast<A*>(w + l.parts) : nullptr;
      const int64_t chunks = n > kLong ? ceil_div(n, kLong) : 0, slices = slices_of<V>(width);
      const int wpr = slices <= 64 ? 1 : slices <= 128 ? 2 : 4;
      // rows a workgroup, so that workgroups fill the chip (us with 16, 8, 4 and 2: 131072
      // tokens of 2000 x 2048 bf16 204, 177, 166, 163, 20000 of 8000 x 1024 53, 46, 42, 41,
      // 65536 of 131072 x 2048 214, 214, 236, 269); of few tokens, found at once, up to 4
      // (1 of 262144 x 1024 118, 125, 103, 128)
      const int64_t most = n <= 4096 ? 4 : 16;
      const int block_rows = (int)std::min(most, std::max<int64_t>(2, n_rows / (2048 * (4 / wpr))));
      const int64_t chunk_blocks = ceil_div(chunks, 4 / wpr);
      const dim3 grid = row_grid(chunk_blocks + ceil_div(n_rows, (4 / wpr) * block_rows));
      auto launch = [&](auto past, auto some) {
        hipLaunchKernelGGL((embedding_grad_kernel<V, O, decltype(past)::value, decltype(some)::value>), grid,
                           dim3(256), 0, stream, (const V*)grad, ldg, keys, order, n, n_rows, width, (A)scale,
                           padding, wpr, block_rows, chunk_blocks, chunks, filled, (O*)out, parts);
      };
      // past the caches only where a wave's slices leave as whole lines: a 32-bit result
      // of 16-bit values leaves as every second 16 bytes at a time (us so and past the
      // caches: 65536 tokens of 131072 x 2048 372 and 562, one token 201 and 527)
      using Past = std::integral_constant<bool, sizeof(O) == sizeof(V)>;
      const int64_t bytes = (n * (int64_t)sizeof(V) + n_rows * (int64_t)sizeof(O)) * width;
      if (Past::value && store_past_caches(bytes, width * sizeof(O)))
        filled > 0 ? launch(Past{}, std::true_type{}) : launch(Past{}, std::false_type{});
      else filled > 0 ? launch(std::false_type{}, std::true_type{}) : launch(std::false_type{}, std::false_type{});
      FS_CHECK_MAIN_LAUNCH("embedding_grad_kernel");
      if (chunks > 0) {
        const dim3 x = row_grid(chunks);
        hipLaunchKernelGGL((embedding_grad_join_kernel<O, A>), dim3(x.x, (uint32_t)ceil_div(width, 256), x.y),
                           dim3(64 * kJoinWaves), 0, stream, keys, n, n_rows, width, (A)scale, padding, parts, (O*)out);
        FS_CHECK_LAUNCH("embedding_grad_join_kernel");
      }
      return FS_OK;
    };
    if constexpr (sizeof(V) == 2) {
      if (out_t == FS_F32) return run(0.0f);
    }
    return run(v);
  });
}
