// embedding.hip — embedding lookup with scaling, and its gradient.
//
// out[t] = scale * table[ids[t]], a product with a selection matrix of one
// entry a row; ids outside the table give a zero row.  The gradient is the
// transposed product, grad_table[v] = scale * sum over the t with ids[t] = v of
// grad[t]: positions sorted by token (select_sort.hip, stable), then one sum a
// table row over its segment, in position order, so results do not change from
// run to run.  Rows without tokens are written as zeros in the same pass.
//
// A row of up to 64 tokens is summed by one wave.  A longer segment (tokens
// follow a Zipf law: the first ones occur thousands of times in a batch) is cut
// at multiples of 64 sorted positions; each chunk sums its part into the
// workspace and a second launch adds a row's parts in order.
#include "select_rows.hpp"

namespace fs {
namespace {

constexpr int kLong = 64;       // tokens of a row that one wave sums, and positions a chunk
constexpr int kRowsPerWave = 4; // table rows of a wave
constexpr int kU = 4;           // slices a lane sums at a time

template <class V, class Id, bool ALIGNED>
__global__ __launch_bounds__(256) void embedding_kernel(const V* __restrict__ table, int64_t ldt, int64_t n_rows,
                                                        const Id* __restrict__ ids, int64_t n, int64_t width, int lpr,
                                                        typename Elem<V>::acc scale, V* __restrict__ out) {
  constexpr int E = Slice<V>::n;
  const int lane = threadIdx.x & (lpr - 1);
  const int64_t t = (int64_t)blockIdx.x * (256 / lpr) + threadIdx.x / lpr;
  if (t >= n) return;
  const int64_t id = (int64_t)ids[t];
  const bool in = (uint64_t)id < (uint64_t)n_rows;
  const V* row = table + (in ? id : 0) * ldt;
  V* o = out + t * width;
  const int64_t full = width / E;
  for (int64_t c = lane; c < full; c += lpr) {
    Slice<V> s;
    if (in) s = load_slice<ALIGNED>(row + c * E);
#pragma unroll
    for (int e = 0; e < E; ++e) s.v[e] = in ? (V)(widen(s.v[e]) * scale) : (V)0;
    store_slice<ALIGNED>(o + c * E, s);
  }
  for (int64_t h = full * E + lane; h < width; h += lpr) o[h] = in ? (V)(widen(row[h]) * scale) : (V)0;
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

// acc[u] = sum over positions t0..t1 (held by the lanes) of the lane's slices
// c0 + u * 64 of the rows, two rows' loads in flight.
template <class V, bool ALIGNED>
__device__ inline void sum_slices(const V* __restrict__ grad, int64_t ldg, int pos, int t0, int t1, int64_t c0,
                                  int64_t full, typename Elem<V>::acc (&acc)[kU][Slice<V>::n]) {
  constexpr int E = Slice<V>::n;
#pragma unroll
  for (int u = 0; u < kU; ++u)
#pragma unroll
    for (int e = 0; e < E; ++e) acc[u][e] = 0;
  auto load = [&](int t, Slice<V> (&s)[kU]) {
    const V* row = grad + (int64_t)__builtin_amdgcn_readlane(pos, t) * ldg;
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (c0 + u * 64 < full) s[u] = load_slice<ALIGNED>(row + (c0 + u * 64) * E);
  };
  auto add = [&](const Slice<V> (&s)[kU]) {
#pragma unroll
    for (int u = 0; u < kU; ++u)
      if (c0 + u * 64 < full)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[u][e] += widen(s[u].v[e]);
  };
  int t = t0;
  for (; t + 1 < t1; t += 2) {
    Slice<V> a[kU], b[kU];
    load(t, a);
    load(t + 1, b);
    add(a);
    add(b);
  }
  if (t < t1) {
    Slice<V> a[kU];
    load(t, a);
    add(a);
  }
}
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
template <bool ALIGNED, class V, class O, class A>
__device__ inline void store_sums(O* p, const A (&acc)[Slice<V>::n], A scale) {
  constexpr int E = Slice<V>::n, EO = Slice<O>::n;
#pragma unroll
  for (int k = 0; k < E / EO; ++k) {
    Slice<O> s;
#pragma unroll
    for (int e = 0; e < EO; ++e) s.v[e] = (O)(acc[k * EO + e] * scale);
    store_slice<ALIGNED>(p + k * EO, s);
  }
}

template <class V, class O, bool ALIGNED>
__global__ __launch_bounds__(256) void embedding_grad_kernel(
    const V* __restrict__ grad, int64_t ldg, const uint32_t* __restrict__ keys, const int32_t* __restrict__ order,
    int64_t n, int64_t n_rows, int64_t width, typename Elem<V>::acc scale, int64_t padding, uint32_t chunk_blocks,
    int64_t n_chunks, O* __restrict__ out, typename Elem<V>::acc* __restrict__ parts) {
  using A = typename Elem<V>::acc;
  constexpr int E = Slice<V>::n;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t full = width / E;
  A acc[kU][E];

  if (blockIdx.x < chunk_blocks) {  // parts of long segments, a wave a chunk
    const int64_t chunk = (int64_t)blockIdx.x * 4 + w;
    if (chunk >= n_chunks) return;
    const int64_t c0 = chunk * kLong;
    const int cnt = (int)(n - c0 < kLong ? n - c0 : kLong);
    const uint32_t kk = lane < cnt ? keys[c0 + lane] : 0xffffffffu;
    const uint32_t kl = (uint32_t)__builtin_amdgcn_readfirstlane((int)kk);
    const uint32_t kr = (uint32_t)__builtin_amdgcn_readlane((int)kk, cnt - 1);
    const uint64_t at_l = __ballot(kk == kl), at_r = __ballot(kk == kr);
    int64_t start = c0;
    if (c0 > 0) {  // (c0 is a multiple of 64)
      const uint64_t before = __ballot(keys[c0 - 64 + lane] == kl);
      start = c0 - __popcll(before);
    }
    const bool enters = start < c0;
    auto is_long = [&](int64_t s, uint32_t k) {
      return (int64_t)k < n_rows && (int64_t)k != padding && s + kLong < n && keys[s + kLong] == k;
    };
    const bool left = enters && (start == c0 - 64 ? (int64_t)kl < n_rows && (int64_t)kl != padding : is_long(start, kl));
    const int f = __builtin_ctzll(at_r);
    const bool right = (f > 0 || !enters) && is_long(c0 + f, kr);
    if (!left && !right) return;
    const int pos = lane < cnt ? order[c0 + lane] : 0;
    for (int side = 0; side < 2; ++side) {
      if (side == 0 ? !left : !right) continue;
      const int t0 = side == 0 ? 0 : f, t1 = side == 0 ? __popcll(at_l) : cnt;
      A* part = parts + (chunk * 2 + side) * width;
      for (int64_t c = lane; c - lane < full; c += 64 * kU) {
        sum_slices<V, ALIGNED>(grad, ldg, pos, t0, t1, c, full, acc);
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (c + u * 64 < full) store_sums<ALIGNED, V>(part + (c + u * 64) * E, acc[u], (A)1);
      }
      const int64_t h = full * E + lane;
      const A a = sum_element(grad, ldg, pos, t0, t1, h, h < width);
      if (h < width) part[h] = a;
    }
    return;
  }

  const int64_t v0 = ((int64_t)(blockIdx.x - chunk_blocks) * 4 + w) * kRowsPerWave;
  if (v0 >= n_rows) return;
  int64_t wb = wave_lower_bound(keys, n, (uint32_t)v0, lane);
  uint32_t kk = wb + lane < n ? keys[wb + lane] : 0xffffffffu;
  for (int r = 0; r < kRowsPerWave && v0 + r < n_rows; ++r) {
    const uint32_t v = (uint32_t)(v0 + r);
    while (__ballot(kk < v) == ~0ull) {
      wb += 64;
      kk = wb + lane < n ? keys[wb + lane] : 0xffffffffu;
    }
    uint64_t m = __ballot(kk == v);
    if (m >> 63) {  // the window may cut the segment: begin it there
      wb += __builtin_ctzll(m);
      kk = wb + lane < n ? keys[wb + lane] : 0xffffffffu;
      m = __ballot(kk == v);
      if (m == ~0ull && wb + kLong < n && keys[wb + kLong] == v) {
        if ((int64_t)v != padding) {  // a long segment: the chunks sum it
          wb = wave_lower_bound(keys, n, v + 1, lane);
          kk = wb + lane < n ? keys[wb + lane] : 0xffffffffu;
          continue;
        }
      }
    }
    const int t0 = m != 0 ? __builtin_ctzll(m) : 0;
    const int t1 = (int64_t)v == padding ? t0 : t0 + __popcll(m);
    const int pos = lane >= t0 && lane < t1 ? order[wb + lane] : 0;
    O* o = out + (int64_t)v * width;
    for (int64_t c = lane; c - lane < full; c += 64 * kU) {
      sum_slices<V, ALIGNED>(grad, ldg, pos, t0, t1, c, full, acc);
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (c + u * 64 < full) store_sums<ALIGNED, V>(o + (c + u * 64) * E, acc[u], scale);
    }
    const int64_t h = full * E + lane;
    const A a = sum_element(grad, ldg, pos, t0, t1, h, h < width);
    if (h < width) o[h] = (O)(a * scale);
  }
}

// Rows of long segments: the chunk in which one starts adds its parts, the
// first chunk's second slot and the first slots of the chunks after it.  The 4
// waves of a workgroup take every fourth part of 256 columns and are added in
// wave order.
template <class O, class A>
__global__ __launch_bounds__(256) void embedding_grad_join_kernel(const uint32_t* __restrict__ keys, int64_t n,
                                                                  int64_t n_rows, int64_t width, A scale,
                                                                  int64_t padding, const A* __restrict__ parts,
                                                                  O* __restrict__ out) {
  constexpr int C = 4;
  __shared__ A s_sum[3][C][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t c0 = (int64_t)blockIdx.x * kLong;
  if (c0 + kLong >= n) return;  // the last chunk starts none that leaves it
  const uint32_t kr = keys[c0 + kLong - 1];
  if (keys[c0 + kLong] != kr || (int64_t)kr >= n_rows || (int64_t)kr == padding) return;
  if (c0 > 0 && keys[c0 - 1] == kr) return;  // starts before
  const int f = __builtin_ctzll(__ballot(keys[c0 + lane] == kr));
  if (c0 + f + kLong >= n || keys[c0 + f + kLong] != kr) return;  // one wave summed it
  const int64_t end = wave_lower_bound(keys, n, kr + 1, lane);
  const int64_t count = (end - 1) / kLong - blockIdx.x + 1;  // chunks that hold it
  const int64_t h0 = (int64_t)blockIdx.y * 64 * C + lane;
  A sum[C] = {};
#pragma unroll 8
  for (int64_t k = w; k < count; k += 4) {
    const A* p = parts + ((blockIdx.x + k) * 2 + (k == 0 ? 1 : 0)) * width;
#pragma unroll
    for (int u = 0; u < C; ++u)
      if (h0 + u * 64 < width) sum[u] += p[h0 + u * 64];
  }
  if (w > 0)
    for (int u = 0; u < C; ++u) s_sum[w - 1][u][lane] = sum[u];
  __syncthreads();
  if (w > 0) return;
#pragma unroll
  for (int u = 0; u < C; ++u) {
    const A total = sum[u] + s_sum[0][u][lane] + s_sum[1][u][lane] + s_sum[2][u][lane];
    if (h0 + u * 64 < width) out[(int64_t)kr * width + h0 + u * 64] = (O)(total * scale);
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
  if (n < 0 || n > INT32_MAX || n_rows < 0 || n_rows >= INT32_MAX || width < 0)
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
  if ((n_rows > 0 && !table) || !ids || !out || ldt < 0) return fail(FS_E_INVALID, "fs_embedding: bad pointer or stride");
  return with_value_type(val_t, "fs_embedding", [&](auto v) -> int {
    using V = decltype(v);
    using A = typename Elem<V>::acc;
    const int64_t s = sizeof(V);
    const int lpr = lanes_per_row(width / Slice<V>::n);
    const dim3 grid((uint32_t)ceil_div(n, 256 / lpr));
    auto launch = [&](auto id, auto al) {
      using Id = decltype(id);
      hipLaunchKernelGGL((embedding_kernel<V, Id, decltype(al)::value>), grid, dim3(256), 0, stream, (const V*)table,
                         ldt, n_rows, (const Id*)ids, n, width, lpr, (A)scale, (V*)out);
    };
    const bool al = aligned16(table, ldt * s) && aligned16(out, width * s);
    if (id_t == FS_I64) al ? launch(int64_t(0), std::true_type{}) : launch(int64_t(0), std::false_type{});
    else al ? launch(int32_t(0), std::true_type{}) : launch(int32_t(0), std::false_type{});
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
  if (n > 0) {
    const int rc = select_sort(ids, id_t, n, n_rows, keys, order, nullptr, nullptr, w, stream);
    if (rc != FS_OK) return rc;
  }
  return with_value_type(val_t, "fs_embedding_grad", [&](auto v) -> int {
    using V = decltype(v);
    using A = typename Elem<V>::acc;
    auto run = [&](auto o) -> int {
      using O = decltype(o);
      A* parts = n > 0 ? reinterpret_cast<A*>(w + l.parts) : nullptr;
      const int64_t chunks = n > kLong ? ceil_div(n, kLong) : 0;
      const uint32_t chunk_blocks = (uint32_t)ceil_div(chunks, 4);
      const dim3 grid(chunk_blocks + (uint32_t)ceil_div(n_rows, 4 * kRowsPerWave));
      // (parts: rows of `width` sums from a 256-byte boundary)
      const bool al = aligned16(grad, ldg * sizeof(V)) && aligned16(out, width * sizeof(O)) &&
                      aligned16(parts, width * sizeof(A));
      if (al)
        hipLaunchKernelGGL((embedding_grad_kernel<V, O, true>), grid, dim3(256), 0, stream, (const V*)grad, ldg, keys,
                           order, n, n_rows, width, (A)scale, padding, chunk_blocks, chunks, (O*)out, parts);
      else
        hipLaunchKernelGGL((embedding_grad_kernel<V, O, false>), grid, dim3(256), 0, stream, (const V*)grad, ldg, keys,
                           order, n, n_rows, width, (A)scale, padding, chunk_blocks, chunks, (O*)out, parts);
      FS_CHECK_MAIN_LAUNCH("embedding_grad_kernel");
      if (chunks > 0) {
        hipLaunchKernelGGL((embedding_grad_join_kernel<O, A>), dim3((uint32_t)chunks, (uint32_t)ceil_div(width, 256)),
                           dim3(256), 0, stream, keys, n, n_rows, width, (A)scale, padding, parts, (O*)out);
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
