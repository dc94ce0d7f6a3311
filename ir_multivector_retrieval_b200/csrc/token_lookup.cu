// token_lookup.cu — a table read by token id with scaling, and its gradients by
// sorted tokens. include/mvr.h states what each call computes.
#include "token_ops.cuh"

namespace mvr {
namespace tok {
namespace {

// ---- lookup ----------------------------------------------------------------
//
// Bound by memory: the table's rows that are named are read, every output row
// is written. One thread per V elements, numbered through the whole output, so
// that a warp writes one run of memory whatever the row length; several of
// them a thread, the block's stride apart, when there is work for all SMs. All
// ids and scales are asked for before the first is used: the chain from an id
// to its row is what a block's time consists of. 1,521,797 x 64 f32 from 32,768
// rows with scales: 71 us (5.6 TB/s) with two accesses of 32 bytes a thread and
// eight blocks an SM, 81 us with four of 16 bytes and six, 93 with eight.
template <class T, class I, int V, int UR, bool SCALE>
__global__ void __launch_bounds__(256, sizeof(T) * V == 32 ? 8 : 6)
lookup_kernel(Flat F, const T* __restrict__ table, uint32_t rows, uint64_t ts, const I* __restrict__ ids,
              const float* __restrict__ scale, float alpha, T* __restrict__ out, uint64_t os) {
  const FlatBlock<UR> B(F);
  ids += B.row0;
  if (SCALE) scale += B.row0;
  out += B.row0 * os;
  uint32_t i[UR], c[UR], r[UR];
  float f[UR];
  Raw<T, V> x[UR];
#pragma unroll
  for (int j = 0; j < UR; ++j) B.place(j, &i[j], &c[j]);  // (0, 0) behind the end: read, not written
#pragma unroll
  for (int j = 0; j < UR; ++j) r[j] = row_of<I>(ids, i[j], rows);
#pragma unroll
  for (int j = 0; j < UR; ++j) f[j] = SCALE ? scale[i[j]] : 1.f;
#pragma unroll
  for (int j = 0; j < UR; ++j) {
    x[j].zero();
    if (r[j] < rows) x[j].load(table + r[j] * ts + c[j] * V);
  }
#pragma unroll
  for (int j = 0; j < UR; ++j) {
    if (!B.in(j)) continue;
    if (r[j] < rows) {
      const float g = SCALE ? alpha * f[j] : alpha;
      float y[V];
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = g * x[j].get(v);
      x[j].set(y);
    }
    x[j].store(out + i[j] * os + c[j] * V);
  }
}

template <class T, class I, int V>
int lookup_run(Ctx* c, uint64_t n, uint32_t chunks, const void* table, uint64_t rows, uint64_t ts, const void* ids,
               const float* scale, float alpha, void* out, uint64_t os) {
  constexpr int kMany = sizeof(T) * V == 32 ? 2 : 4;
  const Flat F = flat_of(n, chunks);
  const bool several = F.total >= (uint64_t)kMany * 2048 * c->sm_count;
  const auto kernel = scale ? (several ? lookup_kernel<T, I, V, kMany, true> : lookup_kernel<T, I, V, 1, true>)
                            : (several ? lookup_kernel<T, I, V, kMany, false> : lookup_kernel<T, I, V, 1, false>);
  kernel<<<blocks_of(F.total, several ? 256 * kMany : 256), 256, 0, c->stream>>>(
      F, (const T*)table, (uint32_t)rows, ts, (const I*)ids, scale, alpha, (T*)out, os);
  MVR_CUDA(c, cudaGetLastError());
  return MVR_OK;
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
//
// Bound: the gradient is read once, in rows of 128 bytes and more at random
// places, which costs no more than reading it in order; the scale's gradient
// comes out of the same pass (its own would read the gradient again). At
// 1,521,797 x 64 f32 over 32,768 rows, a seventh of the tokens in one of them:
// 86 us (4.5 TB/s of gradient), 101 us with the scale's gradient: the tiles, the
// joining launch and, where short keys meet in a block, groups that wait for one
// another. Rows through a ring of asynchronous copies in shared memory, 32 bytes
// a lane, eight rows in flight, 128 threads a block and groups of 32 or 128
// places measured no faster.

// Chunks a lane holds: 16 bytes of a row, in several pieces where its length or
// alignment does not allow one.
template <class T, int V>
constexpr int chunks_per_lane() {
  return (int)sizeof(T) * V >= 16 ? 1 : (int)sizeof(T) * V >= 8 ? 2 : 4;
}

struct GradShape {
  uint32_t n, rows, dim;
  uint32_t lanes;     // L: lanes of a group, a power of two
  uint32_t per_group;  // Tg: places of a group
  uint32_t fills;      // blocks that fill rows without a token, before those with places
  uint32_t tiles;
  uint32_t dots;       // blocks behind them for dscale, where a row's parts lie in several blocks
  uint32_t fill_lanes;  // lanes of a row there, a power of two
  uint32_t gs, ts;  // row strides of grad and table
  uint64_t ds;      // of dtable
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
__device__ __forceinline__ void put_sum(O* p, const float (&sum)[V], float alpha, int accumulate) {
  Raw<O, V> r;
  float x[V];
#pragma unroll
  for (int v = 0; v < V; ++v) x[v] = accumulate ? fmaf(alpha, sum[v], to_f32(p[v])) : alpha * sum[v];
  r.set(x);
  r.store(p);
}

// Zeros for the rows without a token, 64 rows a block, 8 a warp: enough blocks
// for all SMs to write at once.
constexpr uint32_t kFillRows = 64;
template <class O, int V>
__device__ __forceinline__ void fill_empty_rows(const GradShape& S, const uint32_t* __restrict__ offsets,
                                                O* __restrict__ dtable) {
  const uint64_t block = (uint64_t)blockIdx.x * gridDim.y + blockIdx.y;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t v0 = block * kFillRows + (threadIdx.x >> 5) * (kFillRows / 8);
  const uint64_t v = v0 + lane;
  const uint32_t empty =
      __ballot_sync(0xffffffffu, lane < kFillRows / 8 && v < S.rows && offsets[v] == offsets[v + 1]);
  const uint32_t chunks = S.dim / V, L = S.fill_lanes;
  Raw<O, V> z;
  z.zero();
  for (uint32_t j = lane / L; j < kFillRows / 8; j += 32 / L)
    if (empty >> j & 1)
      for (uint32_t c = lane & (L - 1); c < chunks; c += L) z.store(dtable + (v0 + j) * S.ds + (uint64_t)c * V);
}

// dscale of rows whose parts lie in several blocks: a warp per place, beside
// the blocks that sum, whose time is mostly waiting.
template <class T, class O, int V>
__device__ __forceinline__ void scale_dots(const GradArgs<T, O, V>& A) {
  constexpr int U = 4;
  const GradShape& S = A.s;
  const uint64_t block = (uint64_t)(blockIdx.x - S.fills - S.tiles) * gridDim.y + blockIdx.y;
  const uint64_t p = block * 8 + (threadIdx.x >> 5);
  if (p >= S.n) return;
  const uint32_t lane = threadIdx.x & 31, chunks = S.dim / V;
  const uint32_t i = A.order[p], r = A.keys[p];
  if (i >= S.n) return;
  float dot = 0.f;
  if (r < S.rows) {
    const T* a = A.grad + (uint64_t)i * S.gs;
    const T* b = A.table + (uint64_t)r * S.ts;
    for (uint32_t c0 = lane; c0 < chunks; c0 += U * 32) {
      Raw<T, V> x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        x[u].zero();
        y[u].zero();
        const uint32_t c = c0 + u * 32;
        if (c < chunks) {
          x[u].load(a + (uint64_t)c * V);
          y[u].load(b + (uint64_t)c * V);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) dot = fmaf(x[u].get(v), y[u].get(v), dot);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
  if (lane == 0) A.dscale[i] = r < S.rows ? A.alpha * dot : 0.f;
}

// Places of a tile whose plan entries a block keeps in shared memory.
constexpr uint32_t kMaxTile = 2048;
constexpr int kFlight = 4;  // rows a lane takes at once

size_t grad_smem(uint32_t tile) { return (size_t)tile * 12; }

template <class T, class O, int V, bool DSCALE>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 4 : 3)
lookup_grad_tile_kernel(const GradArgs<T, O, V> A) {
  constexpr int NCH = chunks_per_lane<T, V>();
  constexpr int U = kFlight;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ float s_head[256 * NCH * V], s_tail[256 * NCH * V];
  __shared__ uint8_t s_hkind[256], s_has_tail[256];  // head: 0 none, 1 ends here, 2 goes on
  __shared__ uint32_t s_tkey[256];
  grid_dependency_wait();
  const GradShape& S = A.s;
  if (blockIdx.x < S.fills) {
    fill_empty_rows<O, V>(S, A.offsets, A.dtable);
    return;
  }
  if constexpr (!DSCALE) {
    if (blockIdx.x >= S.fills + S.tiles) {
      scale_dots(A);
      return;
    }
  }
  const uint32_t tile_at = blockIdx.x - S.fills;
  const uint32_t L = S.lanes, G = 256 / L;
  const uint32_t g = threadIdx.x / L, l = threadIdx.x & (L - 1);
  const uint32_t valid = min(A.offsets[S.rows], S.n);
  const uint32_t tile = G * S.per_group;
  const uint64_t tile0 = (uint64_t)tile_at * tile;
  if constexpr (DSCALE) {  // the tokens behind the last place name no row
    const uint64_t end = min((uint64_t)S.n, tile0 + tile);
    for (uint64_t p = max((uint64_t)valid, tile0) + threadIdx.x; p < end; p += 256)
      if (A.order[p] < S.n) A.dscale[A.order[p]] = 0.f;
  }
  if (tile0 >= valid) return;
  // the tile's plan: keys, tokens, scales
  uint32_t* s_key = reinterpret_cast<uint32_t*>(smem);
  uint32_t* s_tok = s_key + tile;
  float* s_scale = reinterpret_cast<float*>(s_tok + tile);
  const uint32_t here = (uint32_t)min((uint64_t)tile, valid - tile0);
  for (uint32_t e0 = 0; e0 < here; e0 += 1024) {  // four a thread at once: each loop is one wait for memory
    uint32_t tok[4], key[4];
    float f[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t e = e0 + q * 256 + threadIdx.x;
      tok[q] = e < here ? A.order[tile0 + e] : 0;
      key[q] = e < here ? A.keys[tile0 + e] : 0;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (tok[q] >= S.n) tok[q] = 0;  // in bounds whatever the plan holds
      f[q] = 1.f;
    }
    if (A.scale)
#pragma unroll
      for (int q = 0; q < 4; ++q) f[q] = A.scale[tok[q]];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t e = e0 + q * 256 + threadIdx.x;
      if (e < here) {
        s_key[e] = key[q];
        s_tok[e] = tok[q];
        s_scale[e] = f[q];
      }
    }
  }
  const bool goes_on = tile0 + here < valid && A.keys[tile0 + here] == A.keys[tile0 + here - 1];
  const bool from_before_tile = tile0 && A.keys[tile0 - 1] == A.keys[tile0];
  __syncthreads();

  const uint32_t a = g * S.per_group, b = min(here, a + S.per_group);  // places in the tile: none where a >= b
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
        if (on[k]) put_sum(A.dtable + (uint64_t)key * S.ds + col[k], acc[k], A.alpha, A.accumulate);
  };
  bool started = a < b && (a ? s_key[a - 1] != s_key[a] : !from_before_tile);
  uint32_t cur = a < b ? s_key[a] : S.rows;
  uint32_t hkind = 0;
  Raw<T, V> trow[NCH];  // the table's row of `cur`
  const T* grad[NCH];
#pragma unroll
  for (int k = 0; k < NCH; ++k) grad[k] = A.grad + col[k];
  auto load_grad = [&](Raw<T, V> (&r)[NCH], uint32_t token) {
#pragma unroll
    for (int k = 0; k < NCH; ++k)
      if (on[k]) r[k].load(grad[k] + (uint64_t)token * S.gs);
  };
  auto load_table = [&](Raw<T, V> (&r)[NCH], uint32_t key) {
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      r[k].zero();
      if (key < S.rows && on[k]) r[k].load(A.table + (uint64_t)key * S.ts + col[k]);
    }
  };
  auto add = [&](const Raw<T, V> (&r)[NCH], float f) {
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[k][v] = fmaf(f, r[k].get(v), acc[k][v]);
  };
  auto times = [&](const Raw<T, V> (&x)[NCH], const Raw<T, V> (&y)[NCH]) {
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v) d = fmaf(x[k].get(v), y[k].get(v), d);
    return d;
  };
  if constexpr (DSCALE) load_table(trow, cur);

  Raw<T, V> row[U][NCH];  // zeros for good where the lane is behind the row's end
  float f[U];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < NCH; ++k) row[u][k].zero();
  auto load_step = [&](uint32_t p0) {  // groups begin at multiples of 8 places
#pragma unroll
    for (int u = 0; u < U; u += 4) {
      if (p0 + u >= b) break;
      const uint4 t = *reinterpret_cast<const uint4*>(s_tok + p0 + u);
      load_grad(row[u], t.x);
      if (p0 + u + 1 < b) load_grad(row[u + 1], t.y);
      if (p0 + u + 2 < b) load_grad(row[u + 2], t.z);
      if (p0 + u + 3 < b) load_grad(row[u + 3], t.w);
      const float4 x = *reinterpret_cast<const float4*>(s_scale + p0 + u);
      f[u] = x.x;
      f[u + 1] = x.y;
      f[u + 2] = x.z;
      f[u + 3] = x.w;
    }
  };
  load_step(a);
  const uint32_t steps = (S.per_group + U - 1) / U;  // the same for all lanes: exchanges inside
  for (uint32_t step = 0; step < steps; ++step) {
    const uint32_t p0 = a + step * U;
    if (__all_sync(0xffffffffu, p0 >= b)) break;
    float dot[U];
    // sorted: all of them are of the current key when the last is
    if (p0 + U <= b && s_key[p0 + U - 1] == cur) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        add(row[u], f[u]);
        if constexpr (DSCALE) dot[u] = times(row[u], trow);
      }
    } else {
      uint32_t begins = 0;  // bit u: place p0 + u begins a key
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p0 + u < b && s_key[p0 + u] != (u ? s_key[p0 + u - 1] : cur)) begins |= 1u << u;
      if constexpr (DSCALE) {
        Raw<T, V> other[U][NCH];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          load_table(other[u], p0 + u < b ? s_key[p0 + u] : S.rows);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) dot[u] = times(row[u], other[u]);
#pragma unroll
        for (int k = 0; k < NCH; ++k) trow[k] = other[U - 1][k];  // of the last place's key
      }
      const int count = min((uint32_t)U, b - min(b, p0));
      // the places up to the next key's first, then that key
      for (int from = 0;;) {
        const int to = begins ? __ffs(begins) - 1 : count;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u >= from && u < to) add(row[u], f[u]);
        if (!begins) break;
        if (started) {
          write(cur);
        } else {
          stage(s_head);
          hkind = 1;
        }
        started = true;
        clear();
        cur = s_key[p0 + to];
        begins &= begins - 1;
        from = to;
      }
    }
    load_step(p0 + U);  // on their way during the exchanges
    if constexpr (DSCALE) {
      __syncwarp();
      const GroupSums<U> sums(dot, L, l);
      const uint32_t p = p0 + sums.which;
      if (sums.writes) {
#pragma unroll 1
        for (int k = 0; k < sums.values; ++k)
          if (p + k < b) A.dscale[s_tok[p + k]] = A.alpha * sums.at(dot, k);
      }
    }
  }
  bool has_tail = false;
  if (a < b) {
    const bool ends = b < here ? s_key[b] != cur : !goes_on;
    if (started && ends) {
      write(cur);
    } else if (!started) {
      stage(s_head);
      hkind = ends ? 1 : 2;
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
#pragma unroll 1
  for (int turn = 0; turn < 2; ++turn) {
    if (turn == 0 ? !from_before : !s_has_tail[g]) continue;
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
      write(s_tkey[g]);
    } else {
      float* out = A.part + ((uint64_t)tile_at * 2 + (open ? 1 : 0)) * S.dim;
#pragma unroll
      for (int k = 0; k < NCH; ++k)
        if (on[k])
#pragma unroll
          for (int v = 0; v < V; ++v) out[col[k] + v] = acc[k][v];
    }
  }
}

// Block t sums the key that crosses the border of tiles t and t + 1 and has
// crossed no earlier one: what it left behind the tiles, in their order, then
// its end. L lanes have a tile's sums, W columns each, and the block's groups
// of L lanes take every 512 / L-th tile.
constexpr uint32_t kJoinThreads = 512;
template <class O, int W>
__global__ void __launch_bounds__(kJoinThreads)
lookup_grad_join_kernel(GradShape S, uint32_t L, uint32_t tile, const uint32_t* __restrict__ offsets,
                        const uint32_t* __restrict__ keys, const float* __restrict__ part, O* __restrict__ dtable,
                        float alpha, int accumulate) {
  grid_dependency_wait();
  const uint64_t border = (uint64_t)(blockIdx.x + 1) * tile;
  const uint32_t key = keys[border], before = keys[border - 1];
  if (key >= S.rows || before != key) return;
  const uint32_t first = offsets[key] / tile, last = min((offsets[key + 1] - 1) / tile, S.tiles - 1);
  if (first != blockIdx.x) return;
  __shared__ float s_sum[W][kJoinThreads];
  const uint32_t g = threadIdx.x / L, l = threadIdx.x & (L - 1), G = kJoinThreads / L;
  for (uint32_t c0 = blockIdx.y * (L * W); c0 < S.dim; c0 += gridDim.y * (L * W)) {
    const uint32_t c = c0 + l * W;
    float acc[W];
    Raw<float, W> x;
#pragma unroll
    for (int v = 0; v < W; ++v) acc[v] = 0.f;
    if (c < S.dim) {
#pragma unroll 4
      for (uint32_t t = first + g; t < last; t += G) {
        x.load(part + ((uint64_t)t * 2 + 1) * S.dim + c);
#pragma unroll
        for (int v = 0; v < W; ++v) acc[v] += x.get(v);
      }
    }
#pragma unroll
    for (int v = 0; v < W; ++v) s_sum[v][threadIdx.x] = acc[v];
    __syncthreads();
    if (g == 0 && c < S.dim) {
      x.load(part + (uint64_t)last * 2 * S.dim + c);
      const uint32_t used = min(G, last - first);
#pragma unroll 1
      for (uint32_t q = 1; q < used; ++q)
#pragma unroll
        for (int v = 0; v < W; ++v) acc[v] += s_sum[v][q * L + l];
#pragma unroll
      for (int v = 0; v < W; ++v) {
        const float sum[1] = {acc[v] + x.get(v)};
        put_sum<O, 1>(dtable + (uint64_t)key * S.ds + c + v, sum, alpha, accumulate);
      }
    }
    __syncthreads();
  }
}

// Smallest block of places, whatever the row length: the workspace is sized
// for it. 8 places a group, 8 groups of 32 lanes at least.
constexpr uint32_t kMinTile = 64;

template <class T, class O, int V>
int lookup_grad_run(Ctx* c, GradArgs<T, O, V> A) {
  GradShape& S = A.s;
  cudaStream_t st = c->stream;
  constexpr uint32_t NCH = chunks_per_lane<T, V>();
  const uint32_t chunks = S.dim / V;
  S.lanes = std::min(32u, pow2_ceil((chunks + NCH - 1) / NCH));
  const uint32_t slabs = (chunks + S.lanes * NCH - 1) / (S.lanes * NCH);
  const uint32_t groups = 256 / S.lanes;
  // Few places are one tile, which leaves nothing to join: four steps of a group
  // take no longer than another launch. Otherwise long groups leave fewer sums
  // to join, short ones more blocks: the longest of 8 to 64 places that still
  // gives every SM eight blocks, as long as the tile's plan fits.
  const uint32_t most = kMaxTile / groups;
  S.per_group = (S.n / groups + 8) / 8 * 8;
  if (S.per_group > std::min(16u, most)) {
    S.per_group = std::min(64u, most);
    while (S.per_group > 8 &&
           (uint64_t)slabs * ((S.n + (uint64_t)groups * S.per_group - 1) / ((uint64_t)groups * S.per_group)) <
               8ull * c->sm_count)
      S.per_group >>= 1;
  }
  const uint32_t tile = groups * S.per_group;
  S.tiles = (uint32_t)((S.n + (uint64_t)tile - 1) / tile);
  S.fill_lanes = std::min(32u, pow2_ceil(chunks));
  S.fills = A.accumulate ? 0 : (uint32_t)(((S.rows + kFillRows - 1ull) / kFillRows + slabs - 1) / slabs);
  const bool with_dscale = A.dscale && slabs == 1;
  S.dots = A.dscale && !with_dscale ? (uint32_t)(((S.n + 7ull) / 8 + slabs - 1) / slabs) : 0;
  if (S.tiles + S.fills == 0) return MVR_OK;
  const auto kernel = with_dscale ? lookup_grad_tile_kernel<T, O, V, true> : lookup_grad_tile_kernel<T, O, V, false>;
  const size_t smem = grad_smem(tile);  // with the kernel's own below the 48 KB that need no request
  MVR_CUDA(c, launch_pdl(kernel, dim3(S.fills + S.tiles + S.dots, slabs), 256, smem, st, A));
  if (S.tiles > 1) {  // a block's columns once, while the grid stays small: most blocks have nothing to join
    const uint32_t w = S.dim % 4 == 0 ? 4 : 1, L = std::min(32u, pow2_ceil(S.dim / w));
    const uint32_t columns = (S.dim + L * w - 1) / (L * w);
    const dim3 grid(S.tiles - 1, std::max(1u, std::min(columns, 32768u / S.tiles)));
    const auto join = w == 4 ? lookup_grad_join_kernel<O, 4> : lookup_grad_join_kernel<O, 1>;
    MVR_CUDA(c, launch_pdl(join, grid, kJoinThreads, 0, st, S, L, tile, A.offsets, A.keys, A.part, A.dtable, A.alpha,
                           A.accumulate));
  }
  return MVR_OK;
}

}  // namespace
}  // namespace tok
}  // namespace mvr

using mvr::Ctx;

extern "C" {

int mvr_lookup_device(mvr_ctx* h, const void* d_table, int dtype, uint64_t rows, uint32_t dim, uint64_t table_stride,
                      const void* d_ids, int id_bytes, uint64_t n, const float* d_scale, float alpha, void* d_out,
                      uint64_t out_stride) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::tok::check_rows(c, "table", d_table, dtype, rows, dim, table_stride, false));
  MVR_TRY(mvr::tok::check_ids(c, d_ids, id_bytes, n, rows));
  MVR_TRY(mvr::tok::check_rows(c, "out", d_out, dtype, n, dim, out_stride, true));
  MVR_TRY(mvr::tok::check_f32(c, "scale", d_scale));
  if (n == 0) return MVR_OK;
  mvr::DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  const int w = mvr::tok::vec_of(dtype, dim, {{d_table, table_stride}, {d_out, out_stride}}, 32);
  return mvr::tok::by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    return mvr::tok::by_vec<T, 32>(w, [&](auto vec) {
      constexpr int V = decltype(vec)::value;
      const auto run = id_bytes == 8 ? mvr::tok::lookup_run<T, uint64_t, V> : mvr::tok::lookup_run<T, uint32_t, V>;
      return run(c, n, dim / V, d_table, rows, table_stride, d_ids, d_scale, alpha, d_out, out_stride);
    });
  });
}

int mvr_lookup_grad_bytes(uint64_t n_ids, uint32_t dim, uint64_t* bytes) {
  if (!bytes || n_ids > mvr::tok::kMaxIds || dim == 0) return MVR_E_INVALID_ARGUMENT;
  *bytes = (n_ids + mvr::tok::kMinTile - 1) / mvr::tok::kMinTile * 2 * dim * sizeof(float);
  return MVR_OK;
}

int mvr_lookup_grad_device(mvr_ctx* h, const void* d_grad, int dtype, uint64_t grad_stride, uint64_t n_ids,
                           uint64_t rows, uint32_t dim, const uint32_t* d_offsets, const uint32_t* d_order,
                           const uint32_t* d_keys, const float* d_scale, float alpha, const void* d_table,
                           uint64_t table_stride, void* d_dtable, int dtable_dtype, uint64_t dtable_stride,
                           int accumulate, float* d_dscale, void* d_workspace, uint64_t workspace_bytes) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::tok::check_rows(c, "grad", d_grad, dtype, n_ids, dim, grad_stride, false));
  if (rows == 0 || rows > mvr::tok::kMaxRows) return mvr::tok::bad(c, "rows must be in [1, 2^31 - 2]");
  if (n_ids > mvr::tok::kMaxIds) return mvr::tok::bad(c, "more than 2^31 - 1 ids");
  if (dtable_dtype != dtype && dtable_dtype != MVR_F32) return mvr::tok::bad(c, "dtable must have grad's type or f32");
  MVR_TRY(mvr::tok::check_rows(c, "dtable", d_dtable, dtable_dtype, rows, dim, dtable_stride, true));
  if (!d_offsets || (n_ids && (!d_order || !d_keys))) return mvr::tok::bad(c, "null pointer: plan");
  if (!mvr::tok::aligned(d_offsets, 4) || !mvr::tok::aligned(d_order, 4) || !mvr::tok::aligned(d_keys, 4))
    return mvr::tok::bad(c, "the plan is not aligned to its type");
  MVR_TRY(mvr::tok::check_f32(c, "scale", d_scale));
  MVR_TRY(mvr::tok::check_f32(c, "dscale", d_dscale));
  if (d_dscale) MVR_TRY(mvr::tok::check_rows(c, "table", d_table, dtype, rows, dim, table_stride, false));
  uint64_t need = 0;
  MVR_TRY(mvr_lookup_grad_bytes(n_ids, dim, &need));
  MVR_TRY(mvr::tok::check_workspace(c, d_workspace, workspace_bytes, need));
  mvr::DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  const uint32_t n = (uint32_t)n_ids, v = (uint32_t)rows;
  return mvr::tok::by_type(dtype, [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    auto run = [&](auto* o) {
      using O = std::remove_pointer_t<decltype(o)>;
      int w = mvr::tok::vec_of(dtype, dim, {{d_grad, grad_stride}, {d_dscale ? d_table : nullptr, table_stride}});
      // beside 8 16-bit elements, 8 f32 sums are 32 bytes
      w = std::min(w, mvr::tok::vec_of(dtable_dtype, dim, {{d_dtable, dtable_stride}}, 16 / sizeof(T) * sizeof(O)));
      return mvr::tok::by_vec<T>(w, [&](auto vec) {
        constexpr int V = decltype(vec)::value;
        mvr::tok::GradArgs<T, O, V> A;
        A.s = {n, v, dim, 0, 0, 0, 0, 0, 0, (uint32_t)grad_stride, (uint32_t)table_stride, dtable_stride};
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
        return mvr::tok::lookup_grad_run(c, A);
      });
    };
    if (dtable_dtype == MVR_F32) return run(static_cast<float*>(nullptr));
    return run(t);
  });
}

}  // extern "C"
