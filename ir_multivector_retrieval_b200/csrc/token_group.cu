// token_group.cu — rows sorted by group (expert, centroid, token id) and back,
// with weights applied, and their gradients. include/mvr.h states what each
// call computes.
#include "token_ops.cuh"

namespace mvr {
namespace tok {
namespace {

// ---- rows into sorted order and back ---------------------------------------
//
// Bound by memory as well: with C choices a token, spreading reads a row and
// writes C, collecting reads C and writes one. Without the weights' gradient
// the work is cut as for the lookup. With it a group of lanes has a row, for
// the dot products.

// dst[slot[i, c]] = w[i, c] * src[i]: a token's row is read once. KU choices'
// places are asked for at once, beside the rows. 1,521,797 x 2 choices x 64
// f32: 187 us (6.3 TB/s; 215 us with 16 bytes a lane, 222 us with the places
// read one after the other).
template <class T, int V, int UR, int KU>
__global__ void __launch_bounds__(256)
spread_kernel(Flat F, const T* __restrict__ src, uint64_t ss, uint32_t columns, uint64_t pairs,
              const uint32_t* __restrict__ slot, const float* __restrict__ w, T* __restrict__ dst, uint64_t ds) {
  const FlatBlock<UR> B(F);
  src += B.row0 * ss;
  slot += B.row0 * columns;
  if (w) w += B.row0 * columns;
  uint32_t i[UR], c[UR];
  Raw<T, V> x[UR];
#pragma unroll
  for (int j = 0; j < UR; ++j) B.place(j, &i[j], &c[j]);  // (0, 0) behind the end: read, not written
#pragma unroll
  for (int j = 0; j < UR; ++j) x[j].load(src + i[j] * ss + c[j] * V);
  for (uint32_t k0 = 0; k0 < columns; k0 += KU) {
    uint32_t p[UR][KU];
    float f[UR][KU];
#pragma unroll
    for (int j = 0; j < UR; ++j)
#pragma unroll
      for (int k = 0; k < KU; ++k)
        p[j][k] = k0 + k < columns && B.in(j) ? slot[(uint64_t)i[j] * columns + k0 + k] : kNoSlot;
    if (w)
#pragma unroll
      for (int j = 0; j < UR; ++j)
#pragma unroll
        for (int k = 0; k < KU; ++k) f[j][k] = p[j][k] < pairs ? w[(uint64_t)i[j] * columns + k0 + k] : 0.f;
#pragma unroll
    for (int j = 0; j < UR; ++j)
#pragma unroll
      for (int k = 0; k < KU; ++k) {
        if (p[j][k] >= pairs) continue;
        Raw<T, V> r = x[j];
        if (w) {
          float y[V];
#pragma unroll
          for (int v = 0; v < V; ++v) y[v] = f[j][k] * x[j].get(v);
          r.set(y);
        }
        r.store(dst + p[j][k] * ds + c[j] * V);
      }
  }
}

// dst[i] = sum_c w[i, c] * src[slot[i, c]]: KU choices' rows in flight, four at
// most (4093 x 8 x 2048 f16: 26 us, with eight 28). 1,521,797 x 2 x 64 f32: 185
// us (6.3 TB/s; 230 us with 16 bytes a lane).
template <class T, int V, int KU>
__global__ void __launch_bounds__(256)
collect_kernel(Flat F, const T* __restrict__ src, uint64_t ss, uint32_t columns, uint64_t pairs,
               const uint32_t* __restrict__ slot, const float* __restrict__ w, T* __restrict__ dst, uint64_t ds) {
  const FlatBlock<1> B(F);
  if (!B.in(0)) return;
  uint32_t from, c;
  B.place(0, &from, &c);
  const uint64_t i = B.row0 + from;
  float acc[V];
#pragma unroll
  for (int v = 0; v < V; ++v) acc[v] = 0.f;
  for (uint32_t k0 = 0; k0 < columns; k0 += KU) {
    Raw<T, V> x[KU];
    float f[KU];
    uint32_t p[KU];
#pragma unroll
    for (int k = 0; k < KU; ++k) p[k] = k0 + k < columns ? slot[i * columns + k0 + k] : kNoSlot;
#pragma unroll
    for (int k = 0; k < KU; ++k) {
      if (p[k] < pairs) {
        x[k].load(src + p[k] * ss + (uint64_t)c * V);
        f[k] = w ? w[i * columns + k0 + k] : 1.f;
      } else {
        x[k].zero();
        f[k] = 0.f;
      }
    }
#pragma unroll
    for (int k = 0; k < KU; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(f[k], x[k].get(v), acc[v]);
  }
  Raw<T, V> r;
  r.set(acc);
  r.store(dst + i * ds + (uint64_t)c * V);
}

// The pair's two rows in one pass: dst[slot] = w * src[token], dw = <src[token],
// other[slot]>. A group of L lanes has a pair, so a token's row is read once
// from memory and again from the caches for its other choices. Rows that L
// lanes hold at once are taken PU at a time, longer ones CU chunks at a time.
// 8192 x 8 x 2048 bf16: 88 us (6.4 TB/s); 1,521,797 x 2 x 64 f32: 312 us (6.2
// TB/s; 800 us with one pair at a time).
template <class T, int V, int PU, int CU, bool DST>
__global__ void __launch_bounds__(256)
spread_dot_kernel(uint32_t L, uint32_t chunks, const T* __restrict__ src, uint64_t ss, uint32_t columns,
                  uint64_t pairs, const uint32_t* __restrict__ slot, const float* __restrict__ w,
                  T* __restrict__ dst, uint64_t ds, const T* __restrict__ other, uint64_t other_s,
                  float* __restrict__ dw) {
  __shared__ float s_sum[8];
  const uint32_t l = threadIdx.x & (L - 1), G = 256 / L;
  const uint64_t first = (uint64_t)blockIdx.x * (G * PU) + threadIdx.x / L;
  uint32_t p[PU];
  float f[PU], dot[PU];
#pragma unroll
  for (int q = 0; q < PU; ++q) {
    const uint64_t pair = first + q * G;
    p[q] = pair < pairs ? slot[pair] : kNoSlot;
    dot[q] = 0.f;
  }
#pragma unroll
  for (int q = 0; q < PU; ++q) f[q] = w && p[q] < pairs ? w[first + q * G] : 1.f;
  for (uint32_t c0 = l; c0 < chunks; c0 += CU * L) {
    Raw<T, V> x[PU][CU], o[PU][CU];
#pragma unroll
    for (int q = 0; q < PU; ++q)
#pragma unroll
      for (int u = 0; u < CU; ++u) {
        x[q][u].zero();
        o[q][u].zero();
        const uint32_t c = c0 + u * L;
        if (p[q] < pairs && c < chunks) {
          x[q][u].load(src + (first + q * G) / columns * ss + (uint64_t)c * V);
          o[q][u].load(other + p[q] * other_s + (uint64_t)c * V);
        }
      }
#pragma unroll
    for (int q = 0; q < PU; ++q)
#pragma unroll
      for (int u = 0; u < CU; ++u) {
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          dot[q] = fmaf(x[q][u].get(v), o[q][u].get(v), dot[q]);
          y[v] = f[q] * x[q][u].get(v);
        }
        if constexpr (DST) {
          const uint32_t c = c0 + u * L;
          if (p[q] < pairs && c < chunks) {
            if (w) x[q][u].set(y);
            x[q][u].store(dst + p[q] * ds + (uint64_t)c * V);
          }
        }
      }
  }
  if constexpr (PU == 1) {
    dot[0] = group_sum(dot[0], L, s_sum);
    if (l == 0 && first < pairs) dw[first] = dot[0];
  } else {  // L is at most a warp here
    const GroupSums<PU> sums(dot, L, l);
    if (sums.writes)
#pragma unroll 1
      for (int k = 0; k < sums.values; ++k) {
        const uint64_t pair = first + (sums.which + k) * G;
        if (pair < pairs) dw[pair] = sums.at(dot, k);
      }
  }
}

template <class T, int V, bool DST>
int spread_dot(Ctx* c, uint32_t chunks, const T* src, uint64_t ss, uint32_t columns, uint64_t pairs,
               const uint32_t* slot, const float* w, T* dst, uint64_t ds, const T* other, uint64_t os, float* dw) {
  constexpr int U = sizeof(T) * V == 32 ? 2 : 4;
  const uint32_t L = lanes_of(c, pairs, chunks);
  const bool narrow = chunks <= L && L <= 32;
  const auto kernel = narrow ? spread_dot_kernel<T, V, U, 1, DST> : spread_dot_kernel<T, V, 1, U, DST>;
  kernel<<<blocks_of(pairs, narrow ? 256 / L * U : 256 / L), 256, 0, c->stream>>>(L, chunks, src, ss, columns, pairs,
                                                                                 slot, w, dst, ds, other, os, dw);
  MVR_CUDA(c, cudaGetLastError());
  return MVR_OK;
}

// dst[i] = sum_c w * src[slot] and dw = <other[i], src[slot]> in one pass, for
// at most KU choices: a group of lanes has a token. 1,521,797 x 2 x 64 f32: 245
// us (6.4 TB/s); 8192 x 4 x 1024 bf16 out of memory: 19 us (5.2 TB/s).
template <class T, int V, int KU>
__global__ void __launch_bounds__(256, 4)
collect_dot_kernel(uint32_t L, uint32_t chunks, const T* __restrict__ src, uint64_t ss, uint64_t n, uint32_t columns,
                   const uint32_t* __restrict__ slot, const float* __restrict__ w, T* __restrict__ dst, uint64_t ds,
                   const T* __restrict__ other, uint64_t other_s, float* __restrict__ dw) {
  __shared__ float s_sum[8];
  const uint64_t pairs = n * columns;
  const uint32_t l = threadIdx.x & (L - 1);
  const uint64_t i = (uint64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  uint32_t p[KU];
  float f[KU], dot[KU];
#pragma unroll
  for (int k = 0; k < KU; ++k) {
    const bool in = i < n && (uint32_t)k < columns;
    p[k] = in ? slot[i * columns + k] : kNoSlot;
    f[k] = p[k] < pairs ? (w ? w[i * columns + k] : 1.f) : 0.f;
    dot[k] = 0.f;
  }
  constexpr int U = KU <= 2 && sizeof(T) * V < 32 ? 2 : 1;  // chunks at once
  if (i < n)
    for (uint32_t c0 = l; c0 < chunks; c0 += U * L) {
      Raw<T, V> o[U], x[U][KU];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t c = c0 + u * L;
        o[u].zero();
        if (c < chunks) o[u].load(other + i * other_s + (uint64_t)c * V);
#pragma unroll
        for (int k = 0; k < KU; ++k) {
          x[u][k].zero();
          if (p[k] < pairs && c < chunks) x[u][k].load(src + p[k] * ss + (uint64_t)c * V);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t c = c0 + u * L;
        float acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = 0.f;
#pragma unroll
        for (int k = 0; k < KU; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const float xv = x[u][k].get(v);
            acc[v] = fmaf(f[k], xv, acc[v]);
            dot[k] = fmaf(o[u].get(v), xv, dot[k]);
          }
        if (c < chunks) {
          o[u].set(acc);
          o[u].store(dst + i * ds + (uint64_t)c * V);
        }
      }
    }
  // a choice that names no row met only zeros, but zero times an infinity is none
  if constexpr (KU <= 4)  // eight at once would not stay in registers
    if (L <= 32) {
#pragma unroll
      for (int k = 0; k < KU; ++k)
        if (p[k] >= pairs) dot[k] = 0.f;
      const GroupSums<KU> sums(dot, L, l);
      if (sums.writes && i < n)
#pragma unroll 1
        for (uint32_t k = 0; k < (uint32_t)sums.values; ++k)
          if (sums.which + k < columns) dw[i * columns + sums.which + k] = sums.at(dot, k);
      return;
    }
#pragma unroll
  for (int k = 0; k < KU; ++k) {
    if ((uint32_t)k >= columns) break;  // the same for the whole grid
    const float d = group_sum(dot[k], L, s_sum);
    if (l == 0 && i < n) dw[i * columns + k] = p[k] < pairs ? d : 0.f;
  }
}

int spread(Ctx* c, const void* src, int dtype, uint64_t ss, uint64_t n, uint32_t columns, uint32_t dim,
           const uint32_t* slot, const float* w, void* dst, uint64_t ds, const void* other, uint64_t os, float* dw) {
  if (n == 0) return MVR_OK;
  DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  const uint64_t pairs = n * columns;
  if (dw) {
    const int width = vec_of(dtype, dim, {{src, ss}, {dst, ds}, {other, os}}, 32);
    return by_type(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      return by_vec<T, 32>(width, [&](auto vec) {
        constexpr int V = decltype(vec)::value;
        return spread_dot<T, V, true>(c, dim / V, (const T*)src, ss, columns, pairs, slot, w, (T*)dst, ds,
                                      (const T*)other, os, dw);
      });
    });
  }
  const int width = vec_of(dtype, dim, {{src, ss}, {dst, ds}}, 32);
  return by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return by_vec<T, 32>(width, [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      constexpr int kMany = sizeof(T) * V == 32 ? 2 : 4;
      const Flat F = flat_of(n, dim / V);
      const bool several = F.total >= (uint64_t)kMany * 2048 * c->sm_count;
      const auto kernel = several ? (columns <= 2 ? spread_kernel<T, V, kMany, 2> : spread_kernel<T, V, 2, 8>)
                                  : (columns <= 2 ? spread_kernel<T, V, 1, 2> : spread_kernel<T, V, 1, 8>);
      const int per = several ? (columns <= 2 ? 256 * kMany : 512) : 256;
      kernel<<<blocks_of(F.total, per), 256, 0, c->stream>>>(F, (const T*)src, ss, columns, pairs, slot, w, (T*)dst,
                                                             ds);
      MVR_CUDA(c, cudaGetLastError());
      return (int)MVR_OK;
    });
  });
}

// Choices whose dot products a lane holds at once.
constexpr uint32_t kDotColumns = 8;

int collect(Ctx* c, const void* src, int dtype, uint64_t ss, uint64_t n, uint32_t columns, uint32_t dim,
            const uint32_t* slot, const float* w, void* dst, uint64_t ds, const void* other, uint64_t os, float* dw) {
  if (n == 0) return MVR_OK;
  DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  const uint64_t pairs = n * columns;
  if (dw && columns <= kDotColumns) {
    // one or two rows beside the token's own: 32 bytes of each a lane (245 us, with 16 396 us, at 1,521,797 x 2 x
    // 64 f32); more of them are enough in flight with 16 (66 us, with 32 77 us, at 8192 x 8 x 2048 bf16)
    const int most = columns <= 2 ? 32 : 16;
    const int width = vec_of(dtype, dim, {{src, ss}, {dst, ds}, {other, os}}, most);
    return by_type(dtype, [&](auto* t) {
      using T = std::remove_pointer_t<decltype(t)>;
      auto launch = [&](auto kernel, uint32_t chunks) {
        const uint32_t L = lanes_of(c, n, chunks);
        kernel<<<blocks_of(n, 256 / L), 256, 0, c->stream>>>(L, chunks, (const T*)src, ss, n, columns, slot, w, (T*)dst,
                                                             ds, (const T*)other, os, dw);
        MVR_CUDA(c, cudaGetLastError());
        return (int)MVR_OK;
      };
      if (columns <= 2)
        return by_vec<T, 32>(width, [&](auto vec) {
          constexpr int V = decltype(vec)::value;
          return launch(collect_dot_kernel<T, V, 2>, dim / V);
        });
      return by_vec<T>(width, [&](auto vec) {
        constexpr int V = decltype(vec)::value;
        return launch(columns <= 4 ? collect_dot_kernel<T, V, 4> : collect_dot_kernel<T, V, kDotColumns>, dim / V);
      });
    });
  }
  const int width = vec_of(dtype, dim, {{src, ss}, {dst, ds}}, 32);
  MVR_TRY(by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return by_vec<T, 32>(width, [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      const Flat F = flat_of(n, dim / V);
      const auto kernel = columns <= 2 ? collect_kernel<T, V, 2> : collect_kernel<T, V, 4>;
      kernel<<<blocks_of(F.total, 256), 256, 0, c->stream>>>(F, (const T*)src, ss, columns, pairs, slot, w, (T*)dst,
                                                             ds);
      MVR_CUDA(c, cudaGetLastError());
      return (int)MVR_OK;
    });
  }));
  if (!dw) return MVR_OK;
  // more choices than a lane holds dot products of: those on their own, src once more
  const int dot_width = vec_of(dtype, dim, {{src, ss}, {other, os}}, 32);
  return by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return by_vec<T, 32>(dot_width, [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      return spread_dot<T, V, false>(c, dim / V, (const T*)other, os, columns, pairs, slot, nullptr, nullptr, 0,
                                     (const T*)src, ss, dw);
    });
  });
}

}  // namespace
}  // namespace tok
}  // namespace mvr

using mvr::Ctx;

extern "C" {

int mvr_group_rows_device(mvr_ctx* h, const void* d_x, int dtype, uint64_t x_stride, uint64_t n, uint32_t columns,
                          uint32_t dim, const uint32_t* d_slot, const float* d_weights, void* d_out,
                          uint64_t out_stride) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::tok::check_slots(c, n, columns, d_slot, d_weights));
  MVR_TRY(mvr::tok::check_rows(c, "x", d_x, dtype, n, dim, x_stride, false));
  MVR_TRY(mvr::tok::check_rows(c, "out", d_out, dtype, n, dim, out_stride, true));
  return mvr::tok::spread(c, d_x, dtype, x_stride, n, columns, dim, d_slot, d_weights, d_out, out_stride, nullptr, 0,
                     nullptr);
}

int mvr_ungroup_rows_grad_device(mvr_ctx* h, const void* d_dout, int dtype, uint64_t dout_stride, uint64_t n,
                                 uint32_t columns, uint32_t dim, const uint32_t* d_slot, const float* d_weights,
                                 const void* d_xs, uint64_t xs_stride, void* d_dxs, uint64_t dxs_stride,
                                 float* d_dweights) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::tok::check_slots(c, n, columns, d_slot, d_weights));
  MVR_TRY(mvr::tok::check_rows(c, "dout", d_dout, dtype, n, dim, dout_stride, false));
  MVR_TRY(mvr::tok::check_rows(c, "dxs", d_dxs, dtype, n, dim, dxs_stride, true));
  MVR_TRY(mvr::tok::check_f32(c, "dweights", d_dweights));
  if (d_dweights) MVR_TRY(mvr::tok::check_rows(c, "xs", d_xs, dtype, n, dim, xs_stride, false));
  return mvr::tok::spread(c, d_dout, dtype, dout_stride, n, columns, dim, d_slot, d_weights, d_dxs, dxs_stride, d_xs,
                     xs_stride, d_dweights);
}

int mvr_ungroup_rows_device(mvr_ctx* h, const void* d_xs, int dtype, uint64_t xs_stride, uint64_t n, uint32_t columns,
                            uint32_t dim, const uint32_t* d_slot, const float* d_weights, void* d_out,
                            uint64_t out_stride) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::tok::check_slots(c, n, columns, d_slot, d_weights));
  MVR_TRY(mvr::tok::check_rows(c, "xs", d_xs, dtype, n, dim, xs_stride, false));
  MVR_TRY(mvr::tok::check_rows(c, "out", d_out, dtype, n, dim, out_stride, true));
  return mvr::tok::collect(c, d_xs, dtype, xs_stride, n, columns, dim, d_slot, d_weights, d_out, out_stride, nullptr, 0,
                      nullptr);
}

int mvr_group_rows_grad_device(mvr_ctx* h, const void* d_dout, int dtype, uint64_t dout_stride, uint64_t n,
                               uint32_t columns, uint32_t dim, const uint32_t* d_slot, const float* d_weights,
                               const void* d_x, uint64_t x_stride, void* d_dx, uint64_t dx_stride,
                               float* d_dweights) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::tok::check_slots(c, n, columns, d_slot, d_weights));
  MVR_TRY(mvr::tok::check_rows(c, "dout", d_dout, dtype, n, dim, dout_stride, false));
  MVR_TRY(mvr::tok::check_rows(c, "dx", d_dx, dtype, n, dim, dx_stride, true));
  MVR_TRY(mvr::tok::check_f32(c, "dweights", d_dweights));
  if (d_dweights) MVR_TRY(mvr::tok::check_rows(c, "x", d_x, dtype, n, dim, x_stride, false));
  return mvr::tok::collect(c, d_dout, dtype, dout_stride, n, columns, dim, d_slot, d_weights, d_dx, dx_stride, d_x,
                      x_stride, d_dweights);
}

}  // extern "C"
