// token_ops.cu — token operators on the GPU: a table read by token id with
// scaling and its gradient by sorted tokens; rows sorted by group (expert,
// centroid, token id) and back, with weights applied, and their gradients.
// No reference counterpart. include/mvr.h states what each call computes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "../../include/mvr.h"
#include "km_engine.h"
#include "mvr_device.cuh"
#include "mvr_internal.h"

namespace mvr {
namespace {

constexpr uint32_t kNoSlot = MVR_NO_SLOT;
constexpr uint64_t kMaxIds = 0x7FFFFFFFull;   // pairs of a plan: places fit 31 bits
constexpr uint64_t kMaxElems = 1ull << 38;
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

// V consecutive elements of a row as they lie in memory: 2 to 16 bytes (32
// for f32 sums beside 8 16-bit elements), aligned to that size up to 16, so
// each is one access or two. Rows in flight are kept in this form.
template <class T, int V>
struct Raw {
  static constexpr int kBytes = (int)sizeof(T) * V;
  static constexpr int kWords = (kBytes + 3) / 4;
  static_assert(kBytes <= 32, "one or two accesses");
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* __restrict__ p) {
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int h = 0; h < kBytes / 16; ++h) {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(p) + h);
        w[h * 4] = r.x;
        w[h * 4 + 1] = r.y;
        w[h * 4 + 2] = r.z;
        w[h * 4 + 3] = r.w;
      }
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
    if constexpr (kBytes >= 16) {
#pragma unroll
      for (int h = 0; h < kBytes / 16; ++h)
        reinterpret_cast<uint4*>(p)[h] = make_uint4(w[h * 4], w[h * 4 + 1], w[h * 4 + 2], w[h * 4 + 3]);
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
__device__ __forceinline__ uint32_t row_of(const void* ids, int id_bytes, uint64_t i, uint32_t rows) {
  const uint64_t v = id_bytes == 8 ? static_cast<const uint64_t*>(ids)[i]
                                   : (uint64_t) static_cast<const uint32_t*>(ids)[i];
  return v < rows ? (uint32_t)v : rows;
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

// ---- lookup ----------------------------------------------------------------
//
// Bound by memory: the table's rows that are named are read, every output row
// is written. One thread per V elements, numbered through the whole output,
// so that a warp writes one run of memory whatever the row length; four of
// them a thread, the block's stride apart, when there is work for all SMs.

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
  // false behind the end
  __device__ __forceinline__ bool at(int j, uint64_t* row, uint32_t* chunk) const {
    const uint32_t local = j * 256 + threadIdx.x;
    if (first + local >= F.total) return false;
    const uint32_t x = rem0 + local;
    const uint32_t q = F.shift >= 0 ? x >> F.shift : x / F.chunks;
    *row = row0 + q;
    *chunk = x - q * F.chunks;
    return true;
  }
};

template <class T, int V, int UR>
__global__ void __launch_bounds__(256)
lookup_kernel(Flat F, const T* __restrict__ table, uint32_t rows, uint64_t ts, const void* __restrict__ ids,
              int id_bytes, const float* __restrict__ scale, float alpha, T* __restrict__ out, uint64_t os) {
  const FlatBlock<UR> B(F);
  uint64_t i[UR];
  uint32_t c[UR], r[UR];
  float f[UR];
  Raw<T, V> x[UR];
#pragma unroll
  for (int j = 0; j < UR; ++j) {
    r[j] = rows;
    f[j] = alpha;
    if (B.at(j, &i[j], &c[j])) {
      r[j] = row_of(ids, id_bytes, i[j], rows);
      if (scale) f[j] = alpha * scale[i[j]];
    } else {
      i[j] = ~0ull;
    }
  }
#pragma unroll
  for (int j = 0; j < UR; ++j) {
    x[j].zero();
    if (r[j] < rows) x[j].load(table + r[j] * ts + (uint64_t)c[j] * V);
  }
#pragma unroll
  for (int j = 0; j < UR; ++j) {
    if (i[j] == ~0ull) continue;
    if (r[j] < rows) {
      float y[V];
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = f[j] * x[j].get(v);
      x[j].set(y);
    }
    x[j].store(out + i[j] * os + (uint64_t)c[j] * V);
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
//
// dtable is a sum over the sorted places of each key. The places are cut into
// tiles of one size whatever the keys are, so a key with a seventh of all
// tokens costs no more time than one with few: a group of L lanes sums Tg
// consecutive places in registers, 16 bytes of the row a lane, and writes the
// rows of the keys that begin and end among them. What a key has in a group
// it does not begin or end in goes through shared memory to the block's other
// groups, and what it has in a block it does not begin or end in through the
// workspace to lookup_grad_join_kernel. Every sum's order is fixed by the
// places, so results do not depend on which block runs first.

// Chunks a lane holds: V elements of a row are at most 16 bytes; rows that
// cannot be read 16 bytes at a time take several.
template <class T, int V>
constexpr int chunks_per_lane() {
  return (int)sizeof(T) * V >= 16 ? 1 : (int)sizeof(T) * V >= 8 ? 2 : 4;
}

struct GradShape {
  uint32_t n, rows, dim;
  uint32_t lanes;     // L: lanes of a group, a power of two
  uint32_t per_group;  // Tg: places of a group, a multiple of 8
  uint64_t gs, ts, ds;  // row strides of grad, table, dtable
};

template <class T, class O, int V>
struct GradArgs {
  GradShape s;
  const T* grad;
  const uint32_t *offsets, *order, *keys;
  const float* scale;
  float alpha;
  const T* table;
  O* dtable;
  int accumulate;
  float* dscale;
  float* part;  // [tile][2][dim]: 0 the end of a key that began before the tile, 1 what goes on behind it
};

template <class O, int V>
__device__ __forceinline__ void put_sum(O* p, const float (&sum)[V], int accumulate) {
  Raw<O, V> r;
  if (accumulate) {
    float x[V];
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = to_f32(p[v]) + sum[v];
    r.set(x);
  } else {
    r.set(sum);
  }
  r.store(p);
}

template <class T, class O, int V, bool DSCALE>
__global__ void __launch_bounds__(256)
lookup_grad_tile_kernel(const GradArgs<T, O, V> A) {
  constexpr int NCH = chunks_per_lane<T, V>();
  constexpr int U = DSCALE ? 4 : 8;  // rows in flight a lane
  __shared__ float s_head[256 * NCH * V], s_tail[256 * NCH * V];
  __shared__ uint8_t s_hkind[256], s_has_tail[256];  // head: 0 none, 1 ends here, 2 goes on
  __shared__ uint32_t s_hkey[256], s_tkey[256];
  const GradShape& S = A.s;
  const uint32_t L = S.lanes, G = 256 / L;
  const uint32_t g = threadIdx.x / L, l = threadIdx.x & (L - 1);
  const uint32_t valid = min(A.offsets[S.rows], S.n);
  const uint32_t tile = G * S.per_group;
  const uint64_t tile0 = (uint64_t)blockIdx.x * tile;
  if constexpr (DSCALE) {  // the tokens behind the last place name no row
    const uint64_t end = min((uint64_t)S.n, tile0 + tile);
    for (uint64_t p = max((uint64_t)valid, tile0) + threadIdx.x; p < end; p += 256)
      if (A.order[p] < S.n) A.dscale[A.order[p]] = 0.f;
  }
  if (tile0 >= valid) return;
  const uint32_t a = (uint32_t)min((uint64_t)valid, tile0 + (uint64_t)g * S.per_group);
  const uint32_t b = (uint32_t)min((uint64_t)valid, tile0 + (uint64_t)(g + 1) * S.per_group);
  uint32_t col[NCH];
  bool on[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    col[k] = ((blockIdx.y * NCH + k) * L + l) * V;
    on[k] = col[k] < S.dim;
  }
  float acc[NCH][V];
  auto clear = [&]() {
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[k][v] = 0.f;
  };
  clear();

  bool started = a < b && (a == 0 || A.keys[a - 1] != A.keys[a]);
  uint32_t cur = a < b ? A.keys[a] : S.rows;
  uint32_t hkind = 0;
  auto stage = [&](float* where) {
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) where[((g * NCH + k) * V + v) * L + l] = acc[k][v];
  };
  auto write = [&](uint32_t key) {
    if (key < S.rows)
#pragma unroll
      for (int k = 0; k < NCH; ++k)
        if (on[k]) put_sum(A.dtable + (uint64_t)key * S.ds + col[k], acc[k], A.accumulate);
  };

  const uint32_t steps = (S.per_group + U - 1) / U;  // the same for all lanes: shuffles inside
  for (uint32_t step = 0; step < steps; ++step) {
    const uint32_t p0 = a + step * U;
    if (__all_sync(0xffffffffu, p0 >= b)) break;
    uint32_t key[U], tok[U];
    float f[U];
    Raw<T, V> row[U][NCH], trow[DSCALE ? U : 1][NCH];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = p0 + u < b;
      key[u] = in ? A.keys[p0 + u] : S.rows;
      tok[u] = in ? A.order[p0 + u] : S.n;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool in = tok[u] < S.n && key[u] < S.rows;
      f[u] = in ? (A.scale ? A.alpha * A.scale[tok[u]] : A.alpha) : 0.f;
#pragma unroll
      for (int k = 0; k < NCH; ++k) {
        row[u][k].zero();
        if (in && on[k]) row[u][k].load(A.grad + tok[u] * S.gs + col[k]);
        if constexpr (DSCALE) {
          trow[u][k].zero();
          if (in && on[k]) trow[u][k].load(A.table + key[u] * S.ts + col[k]);
        }
      }
    }
    if constexpr (DSCALE) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float dot = 0.f;
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v) dot = fmaf(row[u][k].get(v), trow[u][k].get(v), dot);
        for (uint32_t o = L >> 1; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (l == 0 && tok[u] < S.n) A.dscale[tok[u]] = A.alpha * dot;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (p0 + u < b) {
        if (key[u] != cur) {
          if (started) {
            write(cur);
          } else {
            stage(s_head);
            hkind = 1;
            if (l == 0) s_hkey[g] = cur;
          }
          started = true;
          cur = key[u];
          clear();
        }
#pragma unroll
        for (int k = 0; k < NCH; ++k)
#pragma unroll
          for (int v = 0; v < V; ++v) acc[k][v] = fmaf(f[u], row[u][k].get(v), acc[k][v]);
      }
    }
  }
  bool has_tail = false;
  if (a < b) {
    const bool ends = b == valid || A.keys[b] != cur;
    if (started && ends) {
      write(cur);
    } else if (!started) {
      stage(s_head);
      hkind = ends ? 1 : 2;
      if (l == 0) s_hkey[g] = cur;
    } else {
      stage(s_tail);
      has_tail = true;
      if (l == 0) s_tkey[g] = cur;
    }
  }
  if (l == 0) {
    s_hkind[g] = (uint8_t)hkind;
    s_has_tail[g] = has_tail;
  }
  __syncthreads();

  // a group that began a key which goes on adds what the next groups have of
  // it; the first group does the same for a key that began in an earlier block
  const bool from_before = g == 0 && s_hkind[0] != 0;
#pragma unroll
  for (int turn = 0; turn < 2; ++turn) {
    if (turn == 0 ? !from_before : !s_has_tail[g]) continue;
    const uint32_t key = turn == 0 ? s_hkey[0] : s_tkey[g];
    const float* first = turn == 0 ? s_head : s_tail;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[k][v] = first[((g * NCH + k) * V + v) * L + l];
    bool open = turn == 1 || s_hkind[0] == 2;
    for (uint32_t q = g + 1; open && q < G && s_hkind[q] != 0; ++q) {
#pragma unroll
      for (int k = 0; k < NCH; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) acc[k][v] += s_head[((q * NCH + k) * V + v) * L + l];
      open = s_hkind[q] == 2;
    }
    if (turn == 1 && !open) {
      write(key);
    } else {
      float* out = A.part + ((uint64_t)blockIdx.x * 2 + (open ? 1 : 0)) * S.dim;
#pragma unroll
      for (int k = 0; k < NCH; ++k)
        if (on[k])
#pragma unroll
          for (int v = 0; v < V; ++v) out[col[k] + v] = acc[k][v];
    }
  }
}

// Rows without a token become zeros (blocks from `joins` on), and block t <
// joins sums the key that crosses the border of tiles t and t + 1 and has
// crossed no earlier one: what it left behind the tiles, in their order, then
// its end.
template <class O, int V>
__global__ void __launch_bounds__(256)
lookup_grad_join_kernel(GradShape S, uint32_t tile, uint32_t joins, const uint32_t* __restrict__ offsets,
                        const uint32_t* __restrict__ keys, const float* __restrict__ part, O* __restrict__ dtable,
                        int accumulate) {
  if (blockIdx.x >= joins) {
    if (accumulate) return;
    const uint32_t chunks = S.dim / V;
    const uint64_t total = (uint64_t)S.rows * chunks;
    for (uint64_t e = (uint64_t)(blockIdx.x - joins) * 256 + threadIdx.x; e < total;
         e += (uint64_t)(gridDim.x - joins) * 256) {
      const uint32_t v = (uint32_t)(e / chunks), c = (uint32_t)(e - (uint64_t)v * chunks);
      if (offsets[v] == offsets[v + 1]) {
        Raw<O, V> z;
        z.zero();
        z.store(dtable + v * S.ds + c * V);
      }
    }
    return;
  }
  const uint32_t valid = min(offsets[S.rows], S.n);
  const uint64_t border = (uint64_t)(blockIdx.x + 1) * tile;
  if (border >= valid) return;
  const uint32_t key = keys[border];
  if (key >= S.rows || keys[border - 1] != key) return;
  const uint32_t first = offsets[key] / tile, last = (min(offsets[key + 1], valid) - 1) / tile;
  if (first != blockIdx.x) return;
  __shared__ float s_sum[256];
  // 32 columns at a time, 8 warps over the tiles
  const uint32_t w = threadIdx.x >> 5, l = threadIdx.x & 31;
  for (uint32_t c0 = 0; c0 < S.dim; c0 += 32) {
    const uint32_t c = c0 + l;
    float acc = 0.f;
    if (c < S.dim) {
#pragma unroll 8
      for (uint32_t t = first + w; t < last; t += 8) acc += part[((uint64_t)t * 2 + 1) * S.dim + c];
    }
    s_sum[threadIdx.x] = acc;
    __syncthreads();
    if (w == 0 && c < S.dim) {
#pragma unroll
      for (int q = 1; q < 8; ++q) acc += s_sum[q * 32 + l];
      acc += part[(uint64_t)last * 2 * S.dim + c];
      O* o = dtable + (uint64_t)key * S.ds + c;
      *o = from_f32<O>(accumulate ? to_f32(*o) + acc : acc);
    }
    __syncthreads();
  }
}

// dscale where a row's parts lie in several blocks of the sums: a group of L
// lanes per token, its table row is the key at its place.
template <class T, int V>
__global__ void __launch_bounds__(256)
lookup_dscale_kernel(uint32_t L, uint32_t chunks, const T* __restrict__ grad, uint64_t gs, uint32_t n, uint32_t rows,
                     const uint32_t* __restrict__ keys, const uint32_t* __restrict__ slot, float alpha,
                     const T* __restrict__ table, uint64_t ts, float* __restrict__ dscale) {
  constexpr int U = 4;
  __shared__ float s_sum[8];
  const uint32_t l = threadIdx.x & (L - 1);
  const uint64_t i = (uint64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const uint32_t p = i < n ? slot[i] : kNoSlot, r = p < n ? keys[p] : rows;
  float dot = 0.f;
  if (r < rows) {
    const T* a = grad + i * gs;
    const T* b = table + r * ts;
    for (uint32_t c0 = l; c0 < chunks; c0 += U * L) {
      Raw<T, V> x[U], o[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u].zero();
        o[u].zero();
        const uint32_t c = c0 + u * L;
        if (c < chunks) {
          x[u].load(a + (uint64_t)c * V);
          o[u].load(b + (uint64_t)c * V);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) dot = fmaf(x[u].get(v), o[u].get(v), dot);
    }
  }
  dot = group_sum(dot, L, s_sum);
  if (l == 0 && i < n) dscale[i] = alpha * dot;
}

// ---- rows into sorted order and back ---------------------------------------
//
// Bound by memory as well: with C choices a token, spreading reads a row and
// writes C, collecting reads C and writes one. Without the weights' gradient
// the work is cut as for the lookup. With it a group of lanes has a row, for
// the dot products.

// dst[slot[i, c]] = w[i, c] * src[i]: a token's row is read once.
template <class T, int V, int UR>
__global__ void __launch_bounds__(256)
spread_kernel(Flat F, const T* __restrict__ src, uint64_t ss, uint32_t columns, uint64_t pairs,
              const uint32_t* __restrict__ slot, const float* __restrict__ w, T* __restrict__ dst, uint64_t ds) {
  const FlatBlock<UR> B(F);
  uint64_t i[UR];
  uint32_t c[UR];
  Raw<T, V> x[UR];
#pragma unroll
  for (int j = 0; j < UR; ++j) {
    if (B.at(j, &i[j], &c[j]))
      x[j].load(src + i[j] * ss + (uint64_t)c[j] * V);
    else
      i[j] = ~0ull;
  }
#pragma unroll
  for (int j = 0; j < UR; ++j) {
    if (i[j] == ~0ull) continue;
    for (uint32_t k = 0; k < columns; ++k) {
      const uint32_t p = slot[i[j] * columns + k];
      if (p >= pairs) continue;
      Raw<T, V> r = x[j];
      if (w) {
        const float f = w[i[j] * columns + k];
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) y[v] = f * x[j].get(v);
        r.set(y);
      }
      r.store(dst + p * ds + (uint64_t)c[j] * V);
    }
  }
}

// dst[i] = sum_c w[i, c] * src[slot[i, c]]: KU choices' rows in flight.
template <class T, int V, int KU>
__global__ void __launch_bounds__(256)
collect_kernel(Flat F, const T* __restrict__ src, uint64_t ss, uint32_t columns, uint64_t pairs,
               const uint32_t* __restrict__ slot, const float* __restrict__ w, T* __restrict__ dst, uint64_t ds) {
  const FlatBlock<1> B(F);
  uint64_t i;
  uint32_t c;
  if (!B.at(0, &i, &c)) return;
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
// other[slot]>. A group of lanes has a pair, so a token's row is read once
// from memory and again from the caches for its other choices.
template <class T, int V, bool DST>
__global__ void __launch_bounds__(256)
spread_dot_kernel(uint32_t L, uint32_t chunks, const T* __restrict__ src, uint64_t ss, uint32_t columns,
                  uint64_t pairs, const uint32_t* __restrict__ slot, const float* __restrict__ w,
                  T* __restrict__ dst, uint64_t ds, const T* __restrict__ other, uint64_t other_s,
                  float* __restrict__ dw) {
  constexpr int U = 4;
  __shared__ float s_sum[8];
  const uint32_t l = threadIdx.x & (L - 1);
  const uint64_t pair = (uint64_t)blockIdx.x * (256 / L) + threadIdx.x / L;
  const uint32_t p = pair < pairs ? slot[pair] : kNoSlot;
  float dot = 0.f;
  if (p < pairs) {
    const T* a = src + pair / columns * ss;
    const T* b = other + p * other_s;
    const float f = w ? w[pair] : 1.f;
    for (uint32_t c0 = l; c0 < chunks; c0 += U * L) {
      Raw<T, V> x[U], o[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u].zero();
        o[u].zero();
        const uint32_t c = c0 + u * L;
        if (c < chunks) {
          x[u].load(a + (uint64_t)c * V);
          o[u].load(b + (uint64_t)c * V);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          dot = fmaf(x[u].get(v), o[u].get(v), dot);
          y[v] = f * x[u].get(v);
        }
        if constexpr (DST) {
          const uint32_t c = c0 + u * L;
          if (c < chunks) {
            if (w) x[u].set(y);
            x[u].store(dst + p * ds + (uint64_t)c * V);
          }
        }
      }
    }
  }
  dot = group_sum(dot, L, s_sum);
  if (l == 0 && pair < pairs) dw[pair] = dot;
}

// dst[i] = sum_c w * src[slot] and dw = <other[i], src[slot]> in one pass, for
// at most KU choices: a group of lanes has a token.
template <class T, int V, int KU>
__global__ void __launch_bounds__(256)
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
  if (i < n)
    for (uint32_t c = l; c < chunks; c += L) {
      Raw<T, V> o, x[KU];
      o.load(other + i * other_s + (uint64_t)c * V);
      float acc[V];
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = 0.f;
#pragma unroll
      for (int k = 0; k < KU; ++k) {
        x[k].zero();
        if (p[k] < pairs) x[k].load(src + p[k] * ss + (uint64_t)c * V);
      }
#pragma unroll
      for (int k = 0; k < KU; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) {
          const float xv = x[k].get(v);
          acc[v] = fmaf(f[k], xv, acc[v]);
          dot[k] = fmaf(o.get(v), xv, dot[k]);
        }
      o.set(acc);
      o.store(dst + i * ds + (uint64_t)c * V);
    }
#pragma unroll
  for (int k = 0; k < KU; ++k) {
    if ((uint32_t)k >= columns) break;  // the same for the whole grid
    const float d = group_sum(dot[k], L, s_sum);
    // a choice that names no row met only zeros, but zero times an infinity is none
    if (l == 0 && i < n) dw[i * columns + k] = p[k] < pairs ? d : 0.f;
  }
}

// ---- host side ---------------------------------------------------------------

size_t elem_size(int dtype) { return dtype == MVR_F32 ? 4 : 2; }
bool known(int dtype) { return dtype == MVR_F32 || dtype == MVR_BF16 || dtype == MVR_F16; }
bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
uint64_t up256(uint64_t v) { return (v + 255) & ~(uint64_t)255; }

// Largest number of elements, at most 16 bytes, by which the row length, the
// strides and the addresses can all be divided: how wide a lane reads.
struct Rows {
  const void* p;
  uint64_t stride;
};
int vec_of(int dtype, uint32_t dim, std::initializer_list<Rows> all) {
  const uint64_t e = elem_size(dtype);
  uint64_t bits = 16 / e | dim;
  for (const Rows& r : all)
    if (r.p) bits |= r.stride | reinterpret_cast<uintptr_t>(r.p) / e;
  return (int)(bits & (~bits + 1));
}

uint32_t pow2_ceil(uint32_t v) {
  uint32_t p = 1;
  while (p < v) p <<= 1;
  return p;
}

Flat flat_of(uint64_t n, uint32_t chunks) {
  int shift = -1;
  if ((chunks & (chunks - 1)) == 0)
    for (shift = 0; (1u << shift) < chunks;) ++shift;
  return {n * chunks, chunks, shift};
}

// Four elements a thread when that still fills every SM with threads.
bool many(Ctx* c, const Flat& F) { return F.total >= 4ull * 2048 * c->sm_count; }

// Lanes of a row for the dot products: one chunk a lane when there are few
// rows; as many as four a lane (fewer lanes to sum over) while every SM keeps
// 1024 threads.
uint32_t lanes_of(Ctx* c, uint64_t n, uint32_t chunks) {
  uint32_t L = std::min(256u, pow2_ceil(chunks));
  while (L > 1 && chunks < 4 * L && n * (L / 2) >= 1024ull * c->sm_count) L /= 2;
  return L;
}

// Blocks of a launch: fewer than 2^31 for all that the checks let through.
unsigned blocks_of(uint64_t items, uint64_t per_block) {
  return (unsigned)((items + per_block - 1) / per_block);
}

// Calls f with the width as a compile-time number.
template <class T, class F>
int by_vec(int v, F&& f) {
  if constexpr (sizeof(T) == 2) {
    if (v >= 8) return f(std::integral_constant<int, 8>());
  }
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
  if (dim > MVR_MAX_ROW_DIM) return bad(c, "dim above MVR_MAX_ROW_DIM");
  if (n && !p) return fail(c, MVR_E_INVALID_ARGUMENT, std::string("null pointer: ") + what);
  // what one launch covers: 2^31 - 1 blocks of 256 elements
  if (n > kMaxElems / dim) return fail(c, MVR_E_INVALID_ARGUMENT, std::string(what) + ": more than 2^38 elements");
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

// Smallest block of places, whatever the row length: the workspace is sized
// for it. 8 places a group, 8 groups of 32 lanes at least.
constexpr uint32_t kMinTile = 64;

template <class T, class O, int V>
int lookup_grad_run(Ctx* c, GradArgs<T, O, V> A, const uint32_t* slot) {
  GradShape& S = A.s;
  cudaStream_t st = c->stream;
  constexpr uint32_t NCH = chunks_per_lane<T, V>();
  const uint32_t chunks = S.dim / V;
  S.lanes = std::min(32u, pow2_ceil((chunks + NCH - 1) / NCH));
  const uint32_t slabs = (chunks + S.lanes * NCH - 1) / (S.lanes * NCH);
  const uint32_t groups = 256 / S.lanes;
  // Long groups leave fewer sums to join, short ones more blocks: the longest
  // of 8 to 64 places that still gives every SM eight blocks.
  S.per_group = 64;
  while (S.per_group > 8 &&
         (uint64_t)slabs * ((S.n + (uint64_t)groups * S.per_group - 1) / ((uint64_t)groups * S.per_group)) <
             8ull * c->sm_count)
    S.per_group >>= 1;
  const uint32_t tile = groups * S.per_group;
  const uint32_t tiles = (uint32_t)((S.n + (uint64_t)tile - 1) / tile);
  if (tiles) {
    if (A.dscale && slabs == 1)
      lookup_grad_tile_kernel<T, O, V, true><<<dim3(tiles, slabs), 256, 0, st>>>(A);
    else
      lookup_grad_tile_kernel<T, O, V, false><<<dim3(tiles, slabs), 256, 0, st>>>(A);
    if (A.dscale && slabs > 1) {  // a row's parts lie in several blocks
      const uint32_t L = lanes_of(c, S.n, chunks);
      lookup_dscale_kernel<T, V><<<blocks_of(S.n, 256 / L), 256, 0, st>>>(
          L, chunks, A.grad, S.gs, S.n, S.rows, A.keys, slot, A.alpha, A.table, S.ts, A.dscale);
    }
  }
  const uint32_t joins = tiles ? tiles - 1 : 0;
  const uint64_t fill = A.accumulate ? 0 : std::min<uint64_t>(((uint64_t)S.rows * chunks + 255) / 256, 8ull * c->sm_count);
  if (joins + fill)
    lookup_grad_join_kernel<O, V><<<(unsigned)(joins + fill), 256, 0, st>>>(S, tile, joins, A.offsets, A.keys, A.part,
                                                                           A.dtable, A.accumulate);
  MVR_CUDA(c, cudaGetLastError());
  return MVR_OK;
}

int spread(Ctx* c, const void* src, int dtype, uint64_t ss, uint64_t n, uint32_t columns, uint32_t dim,
           const uint32_t* slot, const float* w, void* dst, uint64_t ds, const void* other, uint64_t os, float* dw) {
  if (n == 0) return MVR_OK;
  DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  const uint64_t pairs = n * columns;
  const int w_ = vec_of(dtype, dim, {{src, ss}, {dst, ds}, {dw ? other : nullptr, os}});
  return by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return by_vec<T>(w_, [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      const uint32_t chunks = dim / V;
      if (dw) {
        const uint32_t L = lanes_of(c, pairs, chunks);
        spread_dot_kernel<T, V, true><<<blocks_of(pairs, 256 / L), 256, 0, c->stream>>>(
            L, chunks, (const T*)src, ss, columns, pairs, slot, w, (T*)dst, ds, (const T*)other, os, dw);
      } else {
        const Flat F = flat_of(n, chunks);
        if (many(c, F))
          spread_kernel<T, V, 4><<<blocks_of(F.total, 1024), 256, 0, c->stream>>>(F, (const T*)src, ss, columns, pairs,
                                                                                  slot, w, (T*)dst, ds);
        else
          spread_kernel<T, V, 1><<<blocks_of(F.total, 256), 256, 0, c->stream>>>(F, (const T*)src, ss, columns, pairs,
                                                                                 slot, w, (T*)dst, ds);
      }
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
  const int w_ = vec_of(dtype, dim, {{src, ss}, {dst, ds}, {dw ? other : nullptr, os}});
  return by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return by_vec<T>(w_, [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      const uint32_t chunks = dim / V;
      const T *s = (const T*)src, *o = (const T*)other;
      if (dw && columns <= kDotColumns) {
        const uint32_t L = lanes_of(c, n, chunks);
        const unsigned blocks = blocks_of(n, 256 / L);
        if (columns <= 2)
          collect_dot_kernel<T, V, 2><<<blocks, 256, 0, c->stream>>>(L, chunks, s, ss, n, columns, slot, w, (T*)dst,
                                                                     ds, o, os, dw);
        else
          collect_dot_kernel<T, V, kDotColumns><<<blocks, 256, 0, c->stream>>>(L, chunks, s, ss, n, columns, slot, w,
                                                                               (T*)dst, ds, o, os, dw);
      } else {
        const Flat F = flat_of(n, chunks);
        if (columns <= 2)
          collect_kernel<T, V, 2><<<blocks_of(F.total, 256), 256, 0, c->stream>>>(F, s, ss, columns, pairs, slot, w,
                                                                                  (T*)dst, ds);
        else
          collect_kernel<T, V, 8><<<blocks_of(F.total, 256), 256, 0, c->stream>>>(F, s, ss, columns, pairs, slot, w,
                                                                                  (T*)dst, ds);
        if (dw) {  // the dots on their own: src once more
          const uint32_t L = lanes_of(c, pairs, chunks);
          spread_dot_kernel<T, V, false><<<blocks_of(pairs, 256 / L), 256, 0, c->stream>>>(
              L, chunks, o, os, columns, pairs, slot, nullptr, nullptr, 0, s, ss, dw);
        }
      }
      MVR_CUDA(c, cudaGetLastError());
      return (int)MVR_OK;
    });
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
  const int w = mvr::vec_of(dtype, dim, {{d_table, table_stride}, {d_out, out_stride}});
  return mvr::by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return mvr::by_vec<T>(w, [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      const mvr::Flat F = mvr::flat_of(n, dim / V);
      if (mvr::many(c, F))
        mvr::lookup_kernel<T, V, 4><<<mvr::blocks_of(F.total, 1024), 256, 0, c->stream>>>(
            F, (const T*)d_table, (uint32_t)rows, table_stride, d_ids, id_bytes, d_scale, alpha, (T*)d_out,
            out_stride);
      else
        mvr::lookup_kernel<T, V, 1><<<mvr::blocks_of(F.total, 256), 256, 0, c->stream>>>(
            F, (const T*)d_table, (uint32_t)rows, table_stride, d_ids, id_bytes, d_scale, alpha, (T*)d_out,
            out_stride);
      MVR_CUDA(c, cudaGetLastError());
      return (int)MVR_OK;
    });
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
  *bytes = (n_ids + mvr::kMinTile - 1) / mvr::kMinTile * 2 * dim * sizeof(float);
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
  const uint32_t n = (uint32_t)n_ids, v = (uint32_t)rows;
  return mvr::by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    auto run = [&](auto* o) {
      using O = std::remove_pointer_t<decltype(o)>;
      int w = mvr::vec_of(dtype, dim, {{d_grad, grad_stride}, {d_dscale ? d_table : nullptr, table_stride}});
      // 8 f32 sums are two 16-byte accesses, so 16-byte alignment serves them too
      const int wo = mvr::vec_of(dtable_dtype, dim, {{d_dtable, dtable_stride}});
      w = std::min(w, sizeof(O) > sizeof(T) && wo == 4 ? 8 : wo);
      return mvr::by_vec<T>(w, [&](auto vec) {
        constexpr int V = decltype(vec)::value;
        mvr::GradArgs<T, O, V> A;
        A.s = {n, v, dim, 0, 0, grad_stride, table_stride, dtable_stride};
        A.grad = (const T*)d_grad;
        A.offsets = d_offsets;
        A.order = d_order;
        A.keys = d_keys;
        A.scale = d_scale;
        A.alpha = alpha;
        A.table = (const T*)d_table;
        A.dtable = (O*)d_dtable;
        A.accumulate = accumulate;
        A.dscale = d_dscale;
        A.part = (float*)d_workspace;
        return mvr::lookup_grad_run(c, A, d_slot);
      });
    };
    if (dtable_dtype == MVR_F32) return run(static_cast<float*>(nullptr));
    return run(t);
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
