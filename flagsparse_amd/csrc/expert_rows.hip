// expert_rows.hip — token rows into expert order and back.
//
// With inverse[t, j] the place of slot j of token t and `routed` the number of
// slots that name an expert (places from there on belong to none):
//   dispatch      rows[inverse[t, j]] = x[t], 0 for slots of no expert
//   combine       out[t] = sum_j w[t, j] rows[inverse[t, j]] over routed slots
//                 (w = 1: the gradient of dispatch)
//   combine_grad  grad_rows[inverse[t, j]] = w[t, j] grad[t];
//                 grad_w[t, j] = sum_h grad[t, h] rows[inverse[t, j], h]
// Products with the routing matrix, tokens by rows, and its transpose; all are
// bound by the rows' bytes.  Sums run in slot order in 32 bits (64 for float64)
// and are rounded once; a slot of no expert is left out, whatever its row holds.
#include <type_traits>

#include "select_rows.hpp"

namespace fs {
namespace {

// A token's row is read once and written once a slot, lpr lanes a row.  Nearly all
// of it is writing: 16384 x 8 slots, rows of 2048 bf16, 604 MB: 103 us, 5.9 TB/s (a
// fill reaches 6.9, a copy 5.1).
template <class V, bool PAST>
__global__ __launch_bounds__(256) void expert_dispatch_kernel(const V* __restrict__ x, int64_t ldx, int64_t n_tokens,
                                                              int slots, int64_t width, int lpr,
                                                              const int32_t* __restrict__ inverse,
                                                              const int32_t* __restrict__ routed_at,
                                                              V* __restrict__ out) {
  const int lane = threadIdx.x & (lpr - 1);
  const int64_t t = row_block() * (256 / lpr) + threadIdx.x / lpr;
  if (t >= n_tokens) return;
  const int routed = *routed_at;
  const V* row = x + t * ldx;
  const int32_t* inv = inverse + t * slots;
  const int64_t slices = slices_of<V>(width);
  for (int64_t c = lane; c < slices; c += lpr) {
    const int64_t h = slice_start<V>(c, width);
    uint4 s;  // (selected word by word: a choice between two slices went through memory)
    __builtin_memcpy(&s, row + h, 16);
#pragma unroll 4
    for (int j = 0; j < slots; ++j) {
      const bool in = inv[j] < routed;
      const uint4 words = make_uint4(in ? s.x : 0u, in ? s.y : 0u, in ? s.z : 0u, in ? s.w : 0u);
      Slice<V> o;
      __builtin_memcpy(&o, &words, 16);
      store_slice<PAST>(out + inv[j] * width + h, o);
    }
  }
  for (int64_t h = slices > 0 ? width : lane; h < width; h += lpr)
    for (int j = 0; j < slots; ++j) out[inv[j] * width + h] = inv[j] < routed ? row[h] : (V)0;
}

// The rows of a token's slots are in flight together (16384 x 8 slots, rows of
// 2048 bf16, 604 MB: 109 us, 5.5 TB/s; 16 tokens x 4: a launch, 4 us).
// (a slot of no expert has a place, whose row is read and left out)
template <class V, bool PAST>
__global__ __launch_bounds__(256) void expert_combine_kernel(const V* __restrict__ rows, int64_t ldr, int64_t n_tokens,
                                                             int slots, int64_t width, int lpr,
                                                             const int32_t* __restrict__ inverse,
                                                             const int32_t* __restrict__ routed_at,
                                                             const typename Elem<V>::acc* __restrict__ weights,
                                                             V* __restrict__ out) {
  using A = typename Elem<V>::acc;
  constexpr int E = Slice<V>::n, kAtOnce = 4;
  const int lane = threadIdx.x & (lpr - 1);
  const int64_t t = row_block() * (256 / lpr) + threadIdx.x / lpr;
  if (t >= n_tokens) return;
  const int routed = *routed_at;
  const int32_t* inv = inverse + t * slots;
  const A* wt = weights != nullptr ? weights + t * slots : nullptr;
  const int64_t slices = slices_of<V>(width);
  for (int64_t c = lane; c < slices; c += lpr) {
    const int64_t h = slice_start<V>(c, width);
    A acc[E] = {};
    auto add = [&](int j, const Slice<V>& s) {
      const A w = wt != nullptr ? wt[j] : (A)1;
      if (inv[j] < routed)
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] += w * widen(s.v[e]);
    };
    int j = 0;
    for (; j + kAtOnce <= slots; j += kAtOnce) {
      Slice<V> s[kAtOnce];
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) s[q] = load_slice(rows + inv[j + q] * ldr + h);
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) add(j + q, s[q]);
    }
    for (; j < slots; ++j) add(j, load_slice(rows + inv[j] * ldr + h));
    Slice<V> o;
#pragma unroll
    for (int e = 0; e < E; ++e) o.v[e] = (V)acc[e];
    store_slice<PAST>(out + t * width + h, o);
  }
  for (int64_t h = slices > 0 ? width : lane; h < width; h += lpr) {
    A acc = 0;
    for (int j = 0; j < slots; ++j)
      if (inv[j] < routed) acc += (wt != nullptr ? wt[j] : (A)1) * widen(rows[inv[j] * ldr + h]);
    out[t * width + h] = (V)acc;
  }
}

// x * y rounded to A before it is rounded to a value type.  (Left to itself the
// compiler turns some of a slice's products into instructions that round to 16
// bits at once and others not, differently in each form of a kernel.)
template <class A>
__device__ inline A product(A x, A y) {
  A p = x * y;
  asm("" : "+v"(p));
  return p;
}

// One wave a slot: the token's gradient row, read by its slots in turn, comes
// from cache after the first.  The row of the gradient is written in the pass that
// sums the weight's: 8191 x 8 slots, rows of 2560 f16, 714 MB, 138 us, 5.2 TB/s, the
// rate of a copy.  ROWS, DOTS: which of the two gradients are wanted; the rows are
// read for the weights' alone, the weights for the rows' alone.
template <class V, bool PAST, bool ROWS, bool DOTS>
__global__ __launch_bounds__(256) void expert_combine_grad_kernel(
    const V* __restrict__ grad, int64_t ldg, const V* __restrict__ rows, int64_t ldr, int64_t n, int slots,
    int64_t width, const int32_t* __restrict__ inverse, const int32_t* __restrict__ routed_at,
    const typename Elem<V>::acc* __restrict__ weights, V* __restrict__ grad_rows,
    typename Elem<V>::acc* __restrict__ grad_w) {
  using A = typename Elem<V>::acc;
  constexpr int E = Slice<V>::n;
  const int lane = threadIdx.x & 63;
  const int64_t i = row_block() * 4 + (threadIdx.x >> 6);
  if (i >= n) return;
  const int at = inverse[i];
  const bool in = at < *routed_at;
  const A w = ROWS && in ? weights[i] : (A)0;
  const V* g = grad + i / slots * ldg;
  const V* y = DOTS ? rows + at * ldr : nullptr;
  V* o = ROWS ? grad_rows + at * width : nullptr;
  // (no overlapping slice at the end: an element counts once in the dot product)
  const int64_t full = width / E;
  A dot = 0;
  if (in) {
    // (two slices' loads in flight)
    auto one = [&](int64_t c, const Slice<V>& sg, const Slice<V>& sy) {
      Slice<V> out;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const A ge = widen(sg.v[e]);
        if constexpr (DOTS) dot += ge * widen(sy.v[e]);
        if constexpr (ROWS) out.v[e] = (V)product(w, ge);
      }
      if constexpr (ROWS) store_slice<PAST>(o + c * E, out);
    };
    auto of_grad = [&](int64_t c) { return load_slice(g + c * E); };
    auto of_row = [&](int64_t c) { return DOTS ? load_slice(y + c * E) : Slice<V>{}; };
    int64_t c = lane;
    for (; c + 64 < full; c += 128) {
      const Slice<V> g0 = of_grad(c), y0 = of_row(c), g1 = of_grad(c + 64), y1 = of_row(c + 64);
      one(c, g0, y0);
      one(c + 64, g1, y1);
    }
    if (c < full) one(c, of_grad(c), of_row(c));
    for (int64_t h = full * E + lane; h < width; h += 64) {
      if constexpr (DOTS) dot += widen(g[h]) * widen(y[h]);
      if constexpr (ROWS) o[h] = (V)product(w, widen(g[h]));
    }
  } else if constexpr (ROWS) {
    for (int64_t c = lane; c < full; c += 64) store_slice<PAST>(o + c * E, Slice<V>{});
    for (int64_t h = full * E + lane; h < width; h += 64) o[h] = (V)0;
  }
  if constexpr (DOTS) {
    dot = wave_sum(dot);
    if (lane == 0) grad_w[i] = dot;
  }
}

int check_rows(const char* who, int64_t n_tokens, int slots, int64_t width, int64_t n_experts) {
  if (n_tokens < 0 || slots < 1 || width < 0 || n_experts < 1 || n_tokens > INT32_MAX / slots)
    return fail(FS_E_INVALID, std::string(who) + ": sizes out of range");
  return FS_OK;
}

}  // namespace
}  // namespace fs

extern "C" int fs_expert_dispatch(int val_t, int64_t n_tokens, int slots, int64_t width, int64_t n_experts,
                                  const void* x, int64_t ldx, const int32_t* inverse, const int32_t* offsets,
                                  void* out, hipStream_t stream) {
  using namespace fs;
  if (int rc = check_rows("fs_expert_dispatch", n_tokens, slots, width, n_experts)) return rc;
  if (n_tokens == 0 || width == 0) return FS_OK;
  if (!x || !inverse || !offsets || !out || ldx < 0)
    return fail(FS_E_INVALID, "fs_expert_dispatch: bad pointer or stride");
  return with_value_type(val_t, "fs_expert_dispatch", [&](auto v) -> int {
    using V = decltype(v);
    const int lpr = lanes_per_row(slices_of<V>(width));
    const dim3 grid = row_grid(ceil_div(n_tokens, 256 / lpr));
    auto launch = [&](auto past) {
      hipLaunchKernelGGL((expert_dispatch_kernel<V, decltype(past)::value>), grid, dim3(256), 0, stream,
                         (const V*)x, ldx, n_tokens, slots, width, lpr, inverse, offsets + n_experts, (V*)out);
    };
    const int64_t row_bytes = width * (int64_t)sizeof(V);
    if (store_past_caches(n_tokens * (slots + 1) * row_bytes, row_bytes)) launch(std::true_type{});
    else launch(std::false_type{});
    FS_CHECK_MAIN_LAUNCH("expert_dispatch_kernel");
    return FS_OK;
  });
}

extern "C" int fs_expert_combine(int val_t, int64_t n_tokens, int slots, int64_t width, int64_t n_experts,
                                 const void* rows, int64_t ldr, const int32_t* inverse, const int32_t* offsets,
                                 const void* weights, void* out, hipStream_t stream) {
  using namespace fs;
  if (int rc = check_rows("fs_expert_combine", n_tokens, slots, width, n_experts)) return rc;
  if (n_tokens == 0 || width == 0) return FS_OK;
  if (!rows || !inverse || !offsets || !out || ldr < 0)
    return fail(FS_E_INVALID, "fs_expert_combine: bad pointer or stride");
  return with_value_type(val_t, "fs_expert_combine", [&](auto v) -> int {
    using V = decltype(v);
    using A = typename Elem<V>::acc;
    const int lpr = lanes_per_row(slices_of<V>(width));
    const dim3 grid = row_grid(ceil_div(n_tokens, 256 / lpr));
    auto launch = [&](auto past) {
      hipLaunchKernelGGL((expert_combine_kernel<V, decltype(past)::value>), grid, dim3(256), 0, stream,
                         (const V*)rows, ldr, n_tokens, slots, width, lpr, inverse, offsets + n_experts,
                         (const A*)weights, (V*)out);
    };
    const int64_t row_bytes = width * (int64_t)sizeof(V);
    if (store_past_caches(n_tokens * (slots + 1) * row_bytes, row_bytes)) launch(std::true_type{});
    else launch(std::false_type{});
    FS_CHECK_MAIN_LAUNCH("expert_combine_kernel");
    return FS_OK;
  });
}

extern "C" int fs_expert_combine_grad(int val_t, int64_t n_tokens, int slots, int64_t width, int64_t n_experts,
                                      const void* grad, int64_t ldg, const void* rows, int64_t ldr,
                                      const int32_t* inverse, const int32_t* offsets, const void* weights,
                                      void* grad_rows, void* grad_weights, hipStream_t stream) {
  using namespace fs;
  if (int rc = check_rows("fs_expert_combine_grad", n_tokens, slots, width, n_experts)) return rc;
  if (n_tokens == 0) return FS_OK;
  // (of no columns the rows' gradient is empty, and may be null where it is wanted)
  const bool of_rows = grad_rows != nullptr, of_weights = grad_weights != nullptr;
  if (!inverse || !offsets || ldg < 0 || ldr < 0 || (of_rows && !weights) ||
      (width > 0 && (!grad || (of_weights && !rows) || (!of_rows && !of_weights))))
    return fail(FS_E_INVALID, "fs_expert_combine_grad: bad pointer or stride");
  if (width == 0 && !of_weights) return FS_OK;
  return with_value_type(val_t, "fs_expert_combine_grad", [&](auto v) -> int {
    using V = decltype(v);
    using A = typename Elem<V>::acc;
    const int64_t n = n_tokens * slots;
    const dim3 grid = row_grid(ceil_div(n, 4));
    auto launch = [&](auto past, auto want_rows, auto want_weights) {
      hipLaunchKernelGGL((expert_combine_grad_kernel<V, decltype(past)::value, decltype(want_rows)::value,
                                                     decltype(want_weights)::value>),
                         grid, dim3(256), 0, stream, (const V*)grad, ldg, (const V*)rows, ldr, n, slots, width,
                         inverse, offsets + n_experts, (const A*)weights, (V*)grad_rows, (A*)grad_weights);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    const int64_t moved = n_tokens + (of_rows ? n : 0) + (of_weights ? n : 0);
    const bool past = store_past_caches(moved * width * (int64_t)sizeof(V), width * sizeof(V));
    if (!of_rows) launch(No{}, No{}, Yes{});
    else if (of_weights) past ? launch(Yes{}, Yes{}, Yes{}) : launch(No{}, Yes{}, Yes{});
    else past ? launch(Yes{}, Yes{}, No{}) : launch(No{}, Yes{}, No{});
    FS_CHECK_MAIN_LAUNCH("expert_combine_grad_kernel");
    return FS_OK;
  });
}
