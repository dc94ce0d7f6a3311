// token_ops.cuh — what the token operators share: rows read up to 32 bytes a
// lane, work numbered through rows, argument checks and dispatch by element
// type and width.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "../../include/mvr.h"
#include "mvr_device.cuh"
#include "mvr_internal.h"

namespace mvr {
namespace tok {

constexpr uint32_t kNoSlot = MVR_NO_SLOT;
constexpr uint64_t kMaxIds = 0x7FFFFFFFull;   // pairs of a plan: places fit 31 bits
constexpr uint64_t kMaxElems = 1ull << 38;    // of one tensor: fewer than 2^31 blocks of 256 threads
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

// V consecutive elements of a row as they lie in memory: 2 to 32 bytes, aligned
// to that size, so that each is one access. Rows in flight are kept in this
// form.
template <class T, int V>
struct Raw {
  static constexpr int kBytes = (int)sizeof(T) * V;
  static constexpr int kWords = (kBytes + 3) / 4;
  static_assert(kBytes <= 32, "one access");
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* __restrict__ p) {
    if constexpr (kBytes == 32) {
      asm volatile("ld.global.nc.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                   : "l"(p));
    } else if constexpr (kBytes == 16) {
      const uint4 r = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = r.x;
      w[1] = r.y;
      w[2] = r.z;
      w[3] = r.w;
    } else if constexpr (kBytes == 8) {
      const uint2 r = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = r.x;
      w[1] = r.y;
    } else if constexpr (kBytes == 4) {
      w[0] = __ldg(reinterpret_cast<const uint32_t*>(p));
    } else {
      w[0] = __ldg(reinterpret_cast<const unsigned short*>(p));
    }
  }

  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes == 32) {
      asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                   "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
    } else if constexpr (kBytes == 16) {
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    } else {
      *reinterpret_cast<unsigned short*>(p) = (unsigned short)w[0];
    }
  }

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }

  __device__ __forceinline__ float get(int v) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[v]);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
      return __uint_as_float(v & 1 ? w[v / 2] & 0xFFFF0000u : w[v / 2] << 16);
    } else {
      return __half2float(__ushort_as_half((unsigned short)(v & 1 ? w[v / 2] >> 16 : w[v / 2] & 0xFFFFu)));
    }
  }

  // rounds each to the element type
  __device__ __forceinline__ void set(const float (&x)[V]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int v = 0; v < V; ++v) w[v] = __float_as_uint(x[v]);
    } else if constexpr (V == 1) {
      const T t = from_f32<T>(x[0]);
      w[0] = *reinterpret_cast<const unsigned short*>(&t);
    } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
};

// The row an id names, or `rows` where it names none (negative ids are large
// as unsigned values).
template <class I>
__device__ __forceinline__ uint32_t row_of(const I* ids, uint64_t i, uint32_t rows) {
  const I id = ids[i];
  return id < rows ? (uint32_t)id : rows;
}

// Sum of x over the lanes of a group (L a power of two up to 256), in lane 0.
// s: one value a warp; every thread of the block calls it.
__device__ __forceinline__ float group_sum(float x, uint32_t L, float* s) {
  for (uint32_t o = min(L, 32u) >> 1; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (L > 32) {
    const uint32_t warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0) s[warp] = x;
    __syncthreads();
    if ((threadIdx.x & (L - 1)) == 0)
      for (uint32_t q = 1; q < L / 32; ++q) x += s[warp + q];
    __syncthreads();
  }
  return x;
}

// Sums of U values over the L lanes of a group, all at once: while a lane has
// several values, it gives half of them to the lane across and takes the other
// half's, so they take U - 1 + log2(L / U) exchanges instead of U log2(L).
template <int U>
struct GroupSums {
  uint32_t which = 0;  // x[k] has become the sum of value which + k, k < values
  int values = U;      // one unless the group has fewer lanes than U
  bool writes;         // whether this lane is the one to write them
  __device__ __forceinline__ GroupSums(float (&x)[U], uint32_t L, uint32_t l) {
    uint32_t o = L >> 1;
#pragma unroll
    for (int half = U >> 1; half > 0; half >>= 1) {
      if (o == 0) continue;  // the same for all lanes
      const bool up = l & o;
#pragma unroll
      for (int k = 0; k < half; ++k) {
        const float give = up ? x[k] : x[k + half];
        const float keep = up ? x[k + half] : x[k];
        x[k] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
      which += up ? half : 0;
      values = half;
      o >>= 1;
    }
    writes = o == 0 || (l & (2 * o - 1)) == 0;
    for (; o > 0; o >>= 1) x[0] += __shfl_xor_sync(0xffffffffu, x[0], o);
  }
  static __device__ __forceinline__ float at(const float (&x)[U], int k) {
    float r = x[0];
#pragma unroll
    for (int q = 1; q < U; ++q) r = k == q ? x[q] : r;
    return r;
  }
};

// Where element `e` of the outputs lies: row and chunk of a row. `shift` is
// log2(chunks) or -1.
struct Flat {
  uint64_t total;  // rows x chunks
  uint32_t chunks;
  int shift;
};

template <int UR>
struct FlatBlock {
  uint64_t first, row0;
  uint32_t rem0;
  const Flat F;
  __device__ __forceinline__ explicit FlatBlock(const Flat& f) : F(f) {
    first = (uint64_t)blockIdx.x * (256 * UR);
    row0 = F.shift >= 0 ? first >> F.shift : first / F.chunks;
    rem0 = (uint32_t)(first - row0 * F.chunks);
  }
  __device__ __forceinline__ bool in(int j) const { return first + (j * 256 + threadIdx.x) < F.total; }
  // the row from row0 on, and the chunk; (0, 0) behind the end
  __device__ __forceinline__ void place(int j, uint32_t* row, uint32_t* chunk) const {
    const uint32_t x = rem0 + j * 256 + threadIdx.x;
    const uint32_t q = F.shift >= 0 ? x >> F.shift : x / F.chunks;
    *row = in(j) ? q : 0;
    *chunk = in(j) ? x - q * F.chunks : 0;
  }
};

inline size_t elem_size(int dtype) { return dtype == MVR_F32 ? 4 : 2; }
inline bool known(int dtype) { return dtype == MVR_F32 || dtype == MVR_BF16 || dtype == MVR_F16; }
inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline uint64_t up256(uint64_t v) { return (v + 255) & ~(uint64_t)255; }

// Largest number of elements, at most `most` bytes, by which the row length, the
// strides and the addresses can all be divided: how wide a lane reads.
struct Rows {
  const void* p;
  uint64_t stride;
};
inline int vec_of(int dtype, uint32_t dim, std::initializer_list<Rows> all, uint64_t most = 16) {
  const uint64_t e = elem_size(dtype);
  uint64_t bits = most / e | dim;
  for (const Rows& r : all)
    if (r.p) bits |= r.stride | reinterpret_cast<uintptr_t>(r.p) / e;
  return (int)(bits & (~bits + 1));
}

inline uint32_t pow2_ceil(uint32_t v) {
  uint32_t p = 1;
  while (p < v) p <<= 1;
  return p;
}

inline Flat flat_of(uint64_t n, uint32_t chunks) {
  int shift = -1;
  if ((chunks & (chunks - 1)) == 0)
    for (shift = 0; (1u << shift) < chunks;) ++shift;
  return {n * chunks, chunks, shift};
}

// Lanes of a row for the dot products: a warp where the row fills one (fewer
// would read pieces of lines, more have to meet in shared memory), several
// while that leaves an SM short of 1024 threads.
inline uint32_t lanes_of(Ctx* c, uint64_t n, uint32_t chunks) {
  uint32_t L = std::min(256u, pow2_ceil(chunks));
  while (L > 32 && n * (L / 2) >= 1024ull * c->sm_count) L /= 2;
  return L;
}

// Blocks of a launch: fewer than 2^31 for all that the checks let through.
inline unsigned blocks_of(uint64_t items, uint64_t per_block) {
  return (unsigned)((items + per_block - 1) / per_block);
}

// Calls f with the width as a compile-time number, at most MOST bytes.
template <class T, int MOST = 16, class F>
int by_vec(int v, F&& f) {
  if constexpr (MOST / sizeof(T) >= 16)
    if (v >= 16) return f(std::integral_constant<int, 16>());
  if constexpr (MOST / sizeof(T) >= 8)
    if (v >= 8) return f(std::integral_constant<int, 8>());
  if (v >= 4) return f(std::integral_constant<int, 4>());
  if (v >= 2) return f(std::integral_constant<int, 2>());
  return f(std::integral_constant<int, 1>());
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

inline int bad(Ctx* c, const char* msg) { return fail(c, MVR_E_INVALID_ARGUMENT, msg); }

inline int check_ids(Ctx* c, const void* ids, int id_bytes, uint64_t n, uint64_t rows) {
  if (id_bytes != 4 && id_bytes != 8) return bad(c, "id_bytes must be 4 or 8");
  if (rows == 0 || rows > kMaxRows) return bad(c, "rows must be in [1, 2^31 - 2]");
  if (n && !ids) return bad(c, "null pointer: ids");
  if (!aligned(ids, id_bytes)) return bad(c, "ids are not aligned to their type");
  return MVR_OK;
}

inline int check_rows(Ctx* c, const char* what, const void* p, int dtype, uint64_t n, uint32_t dim,
                      uint64_t stride, bool output) {
  if (!known(dtype)) return bad(c, "unknown element type");
  if (dim == 0) return fail(c, MVR_E_DIM_MISMATCH, "dim == 0");
  if (dim > MVR_MAX_ROW_DIM) return bad(c, "dim above MVR_MAX_ROW_DIM");
  if (n && !p) return fail(c, MVR_E_INVALID_ARGUMENT, std::string("null pointer: ") + what);
  if (n > kMaxElems / dim) return fail(c, MVR_E_INVALID_ARGUMENT, std::string(what) + ": more than 2^38 elements");
  if (!aligned(p, elem_size(dtype)))
    return fail(c, MVR_E_INVALID_ARGUMENT, std::string(what) + " is not aligned to its element type");
  if (stride >> 32) return fail(c, MVR_E_INVALID_ARGUMENT, std::string(what) + ": stride above 2^32 - 1");
  if (output && stride < dim) return fail(c, MVR_E_INVALID_ARGUMENT, std::string(what) + ": stride below dim");
  return MVR_OK;
}

inline int check_f32(Ctx* c, const char* what, const void* p) {
  if (!aligned(p, 4)) return fail(c, MVR_E_INVALID_ARGUMENT, std::string(what) + " is not aligned to its type");
  return MVR_OK;
}

inline int check_workspace(Ctx* c, const void* p, uint64_t bytes, uint64_t need) {
  if (need == 0) return MVR_OK;
  if (!p || bytes < need) return bad(c, "workspace below the size asked for");
  if (!aligned(p, 16)) return bad(c, "workspace is not 16-byte aligned");
  return MVR_OK;
}

inline int check_slots(Ctx* c, uint64_t n, uint32_t columns, const uint32_t* slot, const float* w) {
  if (columns == 0) return bad(c, "columns == 0");
  if (n > kMaxIds / columns) return bad(c, "more than 2^31 - 1 ids");
  if (n && !slot) return bad(c, "null pointer: slot");
  if (!aligned(slot, 4) || !aligned(w, 4)) return bad(c, "slot or weights are not aligned to their type");
  return MVR_OK;
}

}  // namespace tok
}  // namespace mvr
