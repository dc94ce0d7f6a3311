// token_ops.cu — token operators on the GPU: a table read by token id with
// scaling and its gradient by sorted tokens; rows sorted by group (expert,
// centroid, token id) and back, with weights applied, and their gradients.
// No reference counterpart. include/mvr.h states what each call computes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "../../include/mvr.h"
#include "km_engine.h"
#include "mvr_device.cuh"
#include "mvr_internal.h"

namespace mvr {
namespace {

constexpr uint32_t kNoSlot = MVR_NO_SLOT;
constexpr uint64_t kMaxIds = 0x7FFFFFFFull;   // pairs of a plan: places fit 31 bits
constexpr uint64_t kMaxRows = 0x7FFFFFFEull;  // rows + 1 offsets, and `rows` itself is the key of no row

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// The row an id names, or `rows` where it names none (negative ids are large
// as unsigned values).
__device__ __forceinline__ uint32_t row_of(const void* ids, int id_bytes, uint64_t i, uint32_t rows) {
  const uint64_t v = id_bytes == 8 ? static_cast<const uint64_t*>(ids)[i]
                                   : (uint64_t) static_cast<const uint32_t*>(ids)[i];
  return v < rows ? (uint32_t)v : rows;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---- lookup ----------------------------------------------------------------

// One warp per row.
template <class T>
__global__ void __launch_bounds__(256)
lookup_kernel(const T* __restrict__ table, uint32_t rows, uint32_t dim, uint64_t ts, const void* __restrict__ ids,
              int id_bytes, uint64_t n, const float* __restrict__ scale, float alpha, T* __restrict__ out,
              uint64_t os) {
  const int lane = threadIdx.x & 31;
  for (uint64_t i = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (uint64_t)gridDim.x * 8) {
    const uint32_t r = row_of(ids, id_bytes, i, rows);
    const float f = scale ? alpha * scale[i] : alpha;
    for (uint32_t d = lane; d < dim; d += 32)
      out[i * os + d] = r < rows ? from_f32<T>(f * to_f32(table[r * ts + d])) : from_f32<T>(0.f);
  }
}

// ---- plan ------------------------------------------------------------------

__global__ void __launch_bounds__(256)
plan_keys_kernel(const void* __restrict__ ids, int id_bytes, uint32_t n, uint32_t rows, uint32_t* __restrict__ keys) {
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i < n) keys[i] = row_of(ids, id_bytes, i, rows);
}

// offsets[v] = first place whose key is >= v, by bisection.
__global__ void __launch_bounds__(256)
plan_offsets_kernel(const uint32_t* __restrict__ keys, uint32_t n, uint32_t rows, uint32_t* __restrict__ offsets) {
  const uint32_t v = blockIdx.x * 256u + threadIdx.x;
  if (v > rows) return;
  uint32_t lo = 0, hi = n;
  while (lo < hi) {
    const uint32_t mid = lo + ((hi - lo) >> 1);
    if (keys[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  offsets[v] = lo;
}

__global__ void __launch_bounds__(256)
plan_finish_kernel(const uint32_t* __restrict__ keys, const uint32_t* __restrict__ vals, uint32_t n, uint32_t rows,
                   uint32_t* __restrict__ keys_out, uint32_t* __restrict__ order, uint32_t* __restrict__ slot) {
  const uint32_t p = blockIdx.x * 256u + threadIdx.x;
  if (p >= n) return;
  keys_out[p] = keys[p];
  order[p] = vals[p];
  slot[vals[p]] = keys[p] < rows ? p : kNoSlot;
}

// ---- lookup gradients ------------------------------------------------------

// One warp per table row: its tokens' gradients in sorted order.
template <class T, class O>
__global__ void __launch_bounds__(256)
lookup_grad_kernel(const T* __restrict__ grad, uint64_t gs, uint32_t n, uint32_t rows, uint32_t dim,
                   const uint32_t* __restrict__ offsets, const uint32_t* __restrict__ order,
                   const float* __restrict__ scale, float alpha, O* __restrict__ dtable, uint64_t ds, int accumulate) {
  const int lane = threadIdx.x & 31;
  for (uint64_t v = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); v < rows; v += (uint64_t)gridDim.x * 8) {
    const uint32_t lo = min(offsets[v], n), hi = min(offsets[v + 1], n);
    if (accumulate && lo >= hi) continue;
    for (uint32_t d = lane; d < dim; d += 32) {
      float acc = 0.f;
      for (uint32_t p = lo; p < hi; ++p) {
        const uint32_t i = order[p];
        if (i < n) acc += (scale ? alpha * scale[i] : alpha) * to_f32(grad[i * gs + d]);
      }
      O* o = dtable + v * ds + d;
      *o = from_f32<O>(accumulate ? to_f32(*o) + acc : acc);
    }
  }
}

// One warp per token; its table row is the key at its place.
template <class T>
__global__ void __launch_bounds__(256)
lookup_dscale_kernel(const T* __restrict__ grad, uint64_t gs, uint32_t n, uint32_t rows, uint32_t dim,
                     const uint32_t* __restrict__ keys, const uint32_t* __restrict__ slot, float alpha,
                     const T* __restrict__ table, uint64_t ts, float* __restrict__ dscale) {
  const int lane = threadIdx.x & 31;
  for (uint64_t i = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (uint64_t)gridDim.x * 8) {
    const uint32_t p = slot[i], r = p < n ? keys[p] : rows;
    float acc = 0.f;
    if (r < rows)
      for (uint32_t d = lane; d < dim; d += 32) acc = fmaf(to_f32(grad[i * gs + d]), to_f32(table[r * ts + d]), acc);
    acc = warp_sum(acc);
    if (lane == 0) dscale[i] = alpha * acc;
  }
}

// ---- rows into sorted order and back ---------------------------------------

// spread: one warp per token, dst[slot] = w * src[token]; with dw also the
// dot of src[token] and other[slot].
template <class T>
__global__ void __launch_bounds__(256)
spread_kernel(const T* __restrict__ src, uint64_t ss, uint64_t n, uint32_t columns, uint32_t dim,
              const uint32_t* __restrict__ slot, const float* __restrict__ w, T* __restrict__ dst, uint64_t ds,
              const T* __restrict__ other, uint64_t other_s, float* __restrict__ dw) {
  const int lane = threadIdx.x & 31;
  const uint64_t pairs = n * columns;
  for (uint64_t i = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (uint64_t)gridDim.x * 8) {
    for (uint32_t c = 0; c < columns; ++c) {
      const uint32_t p = slot[i * columns + c];
      const bool ok = p < pairs;
      const float f = w ? w[i * columns + c] : 1.f;
      float acc = 0.f;
      if (ok)
        for (uint32_t d = lane; d < dim; d += 32) {
          const float x = to_f32(src[i * ss + d]);
          dst[p * ds + d] = from_f32<T>(f * x);
          if (dw) acc = fmaf(x, to_f32(other[p * other_s + d]), acc);
        }
      if (dw) {
        acc = warp_sum(acc);
        if (lane == 0) dw[i * columns + c] = acc;
      }
    }
  }
}

// collect: one warp per token, dst[token] = sum_c w * src[slot]; with dw also
// the dot of other[token] and src[slot].
template <class T>
__global__ void __launch_bounds__(256)
collect_kernel(const T* __restrict__ src, uint64_t ss, uint64_t n, uint32_t columns, uint32_t dim,
               const uint32_t* __restrict__ slot, const float* __restrict__ w, T* __restrict__ dst, uint64_t ds,
               const T* __restrict__ other, uint64_t other_s, float* __restrict__ dw) {
  const int lane = threadIdx.x & 31;
  const uint64_t pairs = n * columns;
  for (uint64_t i = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < n; i += (uint64_t)gridDim.x * 8) {
    for (uint32_t d = lane; d < dim; d += 32) {
      float acc = 0.f;
      for (uint32_t c = 0; c < columns; ++c) {
        const uint32_t p = slot[i * columns + c];
        if (p < pairs) acc = fmaf(w ? w[i * columns + c] : 1.f, to_f32(src[p * ss + d]), acc);
      }
      dst[i * ds + d] = from_f32<T>(acc);
    }
    if (dw)
      for (uint32_t c = 0; c < columns; ++c) {
        const uint32_t p = slot[i * columns + c];
        float acc = 0.f;
        if (p < pairs)
          for (uint32_t d = lane; d < dim; d += 32)
            acc = fmaf(to_f32(other[i * other_s + d]), to_f32(src[p * ss + d]), acc);
        acc = warp_sum(acc);
        if (lane == 0) dw[i * columns + c] = acc;
      }
  }
}

// ---- host side ---------------------------------------------------------------

size_t elem_size(int dtype) { return dtype == MVR_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == MVR_F32 || dtype == MVR_BF16 || dtype == MVR_F16; }
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
uint64_t up256(uint64_t v) { return (v + 255) & ~(uint64_t)255; }
unsigned warp_grid(Ctx* c, uint64_t n) {
  return (unsigned)std::min<uint64_t>((n + 7) / 8, (uint64_t)c->sm_count * 32);
}

// Calls f with a null pointer of the element type.
template <class F>
int by_type(int dtype, F&& f) {
  switch (dtype) {
    case MVR_F32: return f(static_cast<float*>(nullptr));
    case MVR_BF16: return f(static_cast<__nv_bfloat16*>(nullptr));
    default: return f(static_cast<__half*>(nullptr));
  }
}

int bad(Ctx* c, const char* msg) { return fail(c, MVR_E_INVALID_ARGUMENT, msg); }

int check_ids(Ctx* c, const void* ids, int id_bytes, uint64_t n, uint64_t rows) {
  if (id_bytes != 4 && id_bytes != 8) return bad(c, "id_bytes must be 4 or 8");
  if (rows == 0 || rows > kMaxRows) return bad(c, "rows must be in [1, 2^31 - 2]");
  if (n && !ids) return bad(c, "null pointer: ids");
  if (!aligned(ids, id_bytes)) return bad(c, "ids are not aligned to their type");
  return MVR_OK;
}

int check_rows(Ctx* c, const char* what, const void* p, int dtype, uint64_t n, uint32_t dim, uint64_t stride,
               bool output) {
  if (!known(dtype)) return bad(c, "unknown element type");
  if (dim == 0) return fail(c, MVR_E_DIM_MISMATCH, "dim == 0");
  if (n && !p) return fail(c, MVR_E_INVALID_ARGUMENT, std::string("null pointer: ") + what);
  if (!aligned(p, elem_size(dtype)))
    return fail(c, MVR_E_INVALID_ARGUMENT, std::string(what) + " is not aligned to its element type");
  if (output && stride < dim) return fail(c, MVR_E_INVALID_ARGUMENT, std::string(what) + ": stride below dim");
  return MVR_OK;
}

int check_f32(Ctx* c, const char* what, const void* p) {
  if (!aligned(p, 4)) return fail(c, MVR_E_INVALID_ARGUMENT, std::string(what) + " is not aligned to its type");
  return MVR_OK;
}

int check_workspace(Ctx* c, const void* p, uint64_t bytes, uint64_t need) {
  if (need == 0) return MVR_OK;
  if (!p || bytes < need) return bad(c, "workspace below the size asked for");
  if (!aligned(p, 16)) return bad(c, "workspace is not 16-byte aligned");
  return MVR_OK;
}

int check_slots(Ctx* c, uint64_t n, uint32_t columns, const uint32_t* slot, const float* w) {
  if (columns == 0) return bad(c, "columns == 0");
  if (n > kMaxIds / columns) return bad(c, "more than 2^31 - 1 ids");
  if (n && !slot) return bad(c, "null pointer: slot");
  if (!aligned(slot, 4) || !aligned(w, 4)) return bad(c, "slot or weights are not aligned to their type");
  return MVR_OK;
}

// Workspace of the plan: keys, two pairs of (keys, order) for the radix
// passes, and the passes' counts.
struct PlanSpace {
  uint64_t keys, k0, v0, k1, v1, scratch, total;
  explicit PlanSpace(uint64_t n) {
    uint64_t off = 0;
    auto take = [&](uint64_t words) {
      const uint64_t o = off;
      off += up256(words * 4);
      return o;
    };
    keys = take(n);
    k0 = take(n);
    v0 = take(n);
    k1 = take(n);
    v1 = take(n);
    scratch = take(radix_pairs_scratch_words(n));
    total = off;
  }
};

int spread(Ctx* c, const void* src, int dtype, uint64_t ss, uint64_t n, uint32_t columns, uint32_t dim,
           const uint32_t* slot, const float* w, void* dst, uint64_t ds, const void* other, uint64_t os, float* dw) {
  if (n == 0) return MVR_OK;
  DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  return by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    spread_kernel<T><<<warp_grid(c, n), 256, 0, c->stream>>>((const T*)src, ss, n, columns, dim, slot, w, (T*)dst, ds,
                                                             (const T*)other, os, dw);
    MVR_CUDA(c, cudaGetLastError());
    return (int)MVR_OK;
  });
}

int collect(Ctx* c, const void* src, int dtype, uint64_t ss, uint64_t n, uint32_t columns, uint32_t dim,
            const uint32_t* slot, const float* w, void* dst, uint64_t ds, const void* other, uint64_t os, float* dw) {
  if (n == 0) return MVR_OK;
  DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  return by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    collect_kernel<T><<<warp_grid(c, n), 256, 0, c->stream>>>((const T*)src, ss, n, columns, dim, slot, w, (T*)dst, ds,
                                                              (const T*)other, os, dw);
    MVR_CUDA(c, cudaGetLastError());
    return (int)MVR_OK;
  });
}

}  // namespace
}  // namespace mvr

using mvr::Ctx;

extern "C" {

int mvr_lookup_device(mvr_ctx* h, const void* d_table, int dtype, uint64_t rows, uint32_t dim, uint64_t table_stride,
                      const void* d_ids, int id_bytes, uint64_t n, const float* d_scale, float alpha, void* d_out,
                      uint64_t out_stride) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::check_rows(c, "table", d_table, dtype, rows, dim, table_stride, false));
  MVR_TRY(mvr::check_ids(c, d_ids, id_bytes, n, rows));
  MVR_TRY(mvr::check_rows(c, "out", d_out, dtype, n, dim, out_stride, true));
  MVR_TRY(mvr::check_f32(c, "scale", d_scale));
  if (n == 0) return MVR_OK;
  mvr::DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  return mvr::by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    mvr::lookup_kernel<T><<<mvr::warp_grid(c, n), 256, 0, c->stream>>>(
        (const T*)d_table, (uint32_t)rows, dim, table_stride, d_ids, id_bytes, n, d_scale, alpha, (T*)d_out,
        out_stride);
    MVR_CUDA(c, cudaGetLastError());
    return (int)MVR_OK;
  });
}

int mvr_token_plan_bytes(uint64_t n_ids, uint64_t rows, uint64_t* bytes) {
  if (!bytes || n_ids > mvr::kMaxIds || rows == 0 || rows > mvr::kMaxRows) return MVR_E_INVALID_ARGUMENT;
  *bytes = n_ids ? mvr::PlanSpace(n_ids).total : 0;
  return MVR_OK;
}

int mvr_token_plan_device(mvr_ctx* h, const void* d_ids, int id_bytes, uint64_t n_ids, uint64_t rows,
                          uint32_t* d_offsets, uint32_t* d_order, uint32_t* d_keys, uint32_t* d_slot,
                          void* d_workspace, uint64_t workspace_bytes) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::check_ids(c, d_ids, id_bytes, n_ids, rows));
  if (n_ids > mvr::kMaxIds) return mvr::bad(c, "more than 2^31 - 1 ids");
  if (!d_offsets || (n_ids && (!d_order || !d_keys || !d_slot))) return mvr::bad(c, "null pointer");
  if (!mvr::aligned(d_offsets, 4) || !mvr::aligned(d_order, 4) || !mvr::aligned(d_keys, 4) || !mvr::aligned(d_slot, 4))
    return mvr::bad(c, "an output is not aligned to its type");
  uint64_t need = 0;
  MVR_TRY(mvr_token_plan_bytes(n_ids, rows, &need));
  MVR_TRY(mvr::check_workspace(c, d_workspace, workspace_bytes, need));
  mvr::DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  cudaStream_t st = c->stream;
  const uint32_t n = (uint32_t)n_ids, v = (uint32_t)rows;
  const unsigned gn = (n + 255) / 256, gv = v / 256 + 1;
  if (n == 0) {
    MVR_CUDA(c, cudaMemsetAsync(d_offsets, 0, (rows + 1) * 4, st));
    return MVR_OK;
  }
  const mvr::PlanSpace ws(n_ids);
  auto at = [&](uint64_t off) { return reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(d_workspace) + off); };
  int bits = 1;
  while ((rows >> bits) != 0) ++bits;  // keys are 0 .. rows
  mvr::plan_keys_kernel<<<gn, 256, 0, st>>>(d_ids, id_bytes, n, v, at(ws.keys));
  const uint32_t *ko, *vo;
  MVR_TRY(mvr::radix_sort_pairs(c, st, at(ws.keys), nullptr, n, bits, at(ws.k0), at(ws.v0), at(ws.k1), at(ws.v1),
                                at(ws.scratch), &ko, &vo));
  mvr::plan_finish_kernel<<<gn, 256, 0, st>>>(ko, vo, n, v, d_keys, d_order, d_slot);
  mvr::plan_offsets_kernel<<<gv, 256, 0, st>>>(ko, n, v, d_offsets);
  MVR_CUDA(c, cudaGetLastError());
  return MVR_OK;
}

int mvr_lookup_grad_bytes(uint64_t n_ids, uint32_t dim, uint64_t* bytes) {
  if (!bytes || n_ids > mvr::kMaxIds || dim == 0) return MVR_E_INVALID_ARGUMENT;
  *bytes = 0;
  return MVR_OK;
}

int mvr_lookup_grad_device(mvr_ctx* h, const void* d_grad, int dtype, uint64_t grad_stride, uint64_t n_ids,
                           uint64_t rows, uint32_t dim, const uint32_t* d_offsets, const uint32_t* d_order,
                           const uint32_t* d_keys, const uint32_t* d_slot, const float* d_scale, float alpha,
                           const void* d_table, uint64_t table_stride, void* d_dtable, int dtable_dtype,
                           uint64_t dtable_stride, int accumulate, float* d_dscale, void* d_workspace,
                           uint64_t workspace_bytes) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::check_rows(c, "grad", d_grad, dtype, n_ids, dim, grad_stride, false));
  if (rows == 0 || rows > mvr::kMaxRows) return mvr::bad(c, "rows must be in [1, 2^31 - 2]");
  if (n_ids > mvr::kMaxIds) return mvr::bad(c, "more than 2^31 - 1 ids");
  if (dtable_dtype != dtype && dtable_dtype != MVR_F32) return mvr::bad(c, "dtable must have grad's type or f32");
  MVR_TRY(mvr::check_rows(c, "dtable", d_dtable, dtable_dtype, rows, dim, dtable_stride, true));
  if (!d_offsets || (n_ids && (!d_order || !d_keys || !d_slot))) return mvr::bad(c, "null pointer: plan");
  if (!mvr::aligned(d_offsets, 4) || !mvr::aligned(d_order, 4) || !mvr::aligned(d_keys, 4) || !mvr::aligned(d_slot, 4))
    return mvr::bad(c, "the plan is not aligned to its type");
  MVR_TRY(mvr::check_f32(c, "scale", d_scale));
  MVR_TRY(mvr::check_f32(c, "dscale", d_dscale));
  if (d_dscale) MVR_TRY(mvr::check_rows(c, "table", d_table, dtype, rows, dim, table_stride, false));
  uint64_t need = 0;
  MVR_TRY(mvr_lookup_grad_bytes(n_ids, dim, &need));
  MVR_TRY(mvr::check_workspace(c, d_workspace, workspace_bytes, need));
  mvr::DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  cudaStream_t st = c->stream;
  const uint32_t n = (uint32_t)n_ids, v = (uint32_t)rows;
  return mvr::by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    if (dtable_dtype == MVR_F32)
      mvr::lookup_grad_kernel<T, float><<<mvr::warp_grid(c, v), 256, 0, st>>>(
          (const T*)d_grad, grad_stride, n, v, dim, d_offsets, d_order, d_scale, alpha, (float*)d_dtable,
          dtable_stride, accumulate);
    else
      mvr::lookup_grad_kernel<T, T><<<mvr::warp_grid(c, v), 256, 0, st>>>((const T*)d_grad, grad_stride, n, v, dim,
                                                                          d_offsets, d_order, d_scale, alpha,
                                                                          (T*)d_dtable, dtable_stride, accumulate);
    if (d_dscale && n)
      mvr::lookup_dscale_kernel<T><<<mvr::warp_grid(c, n), 256, 0, st>>>((const T*)d_grad, grad_stride, n, v, dim,
                                                                         d_keys, d_slot, alpha, (const T*)d_table,
                                                                         table_stride, d_dscale);
    MVR_CUDA(c, cudaGetLastError());
    return (int)MVR_OK;
  });
}

int mvr_group_rows_device(mvr_ctx* h, const void* d_x, int dtype, uint64_t x_stride, uint64_t n, uint32_t columns,
                          uint32_t dim, const uint32_t* d_slot, const float* d_weights, void* d_out,
                          uint64_t out_stride) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::check_slots(c, n, columns, d_slot, d_weights));
  MVR_TRY(mvr::check_rows(c, "x", d_x, dtype, n, dim, x_stride, false));
  MVR_TRY(mvr::check_rows(c, "out", d_out, dtype, n, dim, out_stride, true));
  return mvr::spread(c, d_x, dtype, x_stride, n, columns, dim, d_slot, d_weights, d_out, out_stride, nullptr, 0,
                     nullptr);
}

int mvr_ungroup_rows_grad_device(mvr_ctx* h, const void* d_dout, int dtype, uint64_t dout_stride, uint64_t n,
                                 uint32_t columns, uint32_t dim, const uint32_t* d_slot, const float* d_weights,
                                 const void* d_xs, uint64_t xs_stride, void* d_dxs, uint64_t dxs_stride,
                                 float* d_dweights) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::check_slots(c, n, columns, d_slot, d_weights));
  MVR_TRY(mvr::check_rows(c, "dout", d_dout, dtype, n, dim, dout_stride, false));
  MVR_TRY(mvr::check_rows(c, "dxs", d_dxs, dtype, n, dim, dxs_stride, true));
  MVR_TRY(mvr::check_f32(c, "dweights", d_dweights));
  if (d_dweights) MVR_TRY(mvr::check_rows(c, "xs", d_xs, dtype, n, dim, xs_stride, false));
  return mvr::spread(c, d_dout, dtype, dout_stride, n, columns, dim, d_slot, d_weights, d_dxs, dxs_stride, d_xs,
                     xs_stride, d_dweights);
}

int mvr_ungroup_rows_device(mvr_ctx* h, const void* d_xs, int dtype, uint64_t xs_stride, uint64_t n, uint32_t columns,
                            uint32_t dim, const uint32_t* d_slot, const float* d_weights, void* d_out,
                            uint64_t out_stride) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::check_slots(c, n, columns, d_slot, d_weights));
  MVR_TRY(mvr::check_rows(c, "xs", d_xs, dtype, n, dim, xs_stride, false));
  MVR_TRY(mvr::check_rows(c, "out", d_out, dtype, n, dim, out_stride, true));
  return mvr::collect(c, d_xs, dtype, xs_stride, n, columns, dim, d_slot, d_weights, d_out, out_stride, nullptr, 0,
                      nullptr);
}

int mvr_group_rows_grad_device(mvr_ctx* h, const void* d_dout, int dtype, uint64_t dout_stride, uint64_t n,
                               uint32_t columns, uint32_t dim, const uint32_t* d_slot, const float* d_weights,
                               const void* d_x, uint64_t x_stride, void* d_dx, uint64_t dx_stride,
                               float* d_dweights) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::check_slots(c, n, columns, d_slot, d_weights));
  MVR_TRY(mvr::check_rows(c, "dout", d_dout, dtype, n, dim, dout_stride, false));
  MVR_TRY(mvr::check_rows(c, "dx", d_dx, dtype, n, dim, dx_stride, true));
  MVR_TRY(mvr::check_f32(c, "dweights", d_dweights));
  if (d_dweights) MVR_TRY(mvr::check_rows(c, "x", d_x, dtype, n, dim, x_stride, false));
  return mvr::collect(c, d_dout, dtype, dout_stride, n, columns, dim, d_slot, d_weights, d_dx, dx_stride, d_x,
                      x_stride, d_dweights);
}

}  // extern "C"
