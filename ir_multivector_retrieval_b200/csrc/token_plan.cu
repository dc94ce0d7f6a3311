// token_plan.cu — the stable sort of token ids that the table's gradient and
// the grouping of rows read. include/mvr.h states what it gives.
#include <cooperative_groups.h>

#include <utility>

#include "token_ops.cuh"

namespace cg = cooperative_groups;

namespace mvr {
namespace tok {
namespace {

// The sort is by radix, stable: in each pass, least significant digit first, a
// pair goes to (pairs of smaller digits) + (pairs of its digit before it). The
// ids are a few bytes a token beside rows of hundreds, so what costs is the
// number of dependent steps: some thousand pairs go through all passes in
// one launch of one cluster of blocks; above, a pass is two or three launches
// over tiles.

constexpr int kMostBits = 10;  // of a digit
constexpr uint32_t kSmallThreads = 256, kSmallRounds = 8, kSmallBlocks = 8;
constexpr uint32_t kSmallMax = kSmallThreads * kSmallRounds * kSmallBlocks;  // 16,384 pairs
constexpr uint32_t kSmallMaxPasses = kSmallMax / 2;                          // where one pass is not enough
constexpr uint32_t kTileThreads = 256;

struct PlanArgs {
  const void* ids;
  int id_bytes;
  uint32_t n, rows;
  uint32_t *offsets, *order, *keys, *slot;
};

// Where a pass reads its keys: the ids (4 or 8 bytes) or the last pass's.
template <class I>
__device__ __forceinline__ uint32_t key_at(const void* src, uint64_t e, uint32_t rows) {
  if constexpr (std::is_same_v<I, void>) {
    return __ldcg(static_cast<const uint32_t*>(src) + e);
  } else {
    return row_of(static_cast<const I*>(src), e, rows);
  }
}

// Place of a lane's pair among its warp's pairs of the same digit so far; the
// warp's count of the digit goes up by this round's. Lanes with equal digits
// are found by a vote on each bit: 30 cycles of the SM a warp at 8 bits, where
// the match instruction takes 66 when the digits differ.
__device__ __forceinline__ uint32_t place_in(uint32_t* count, uint32_t digit, int bits, bool in) {
  uint32_t m = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < kMostBits; ++b)
    if (b < bits) {
      const bool one = digit >> b & 1;
      const uint32_t v = __ballot_sync(0xffffffffu, one);
      m &= one ? v : ~v;
    }
  const uint32_t below = __popc(m & lanemask_lt());
  uint32_t place = 0;
  if (in) place = count[digit] + below;
  __syncwarp();
  if (in && below == 0) count[digit] += __popc(m);
  __syncwarp();
  return place;
}

// A digit's counts in the warps' rows of s, R apart, become those of the warps
// before; their sum.
__device__ __forceinline__ uint32_t warps_prefix(uint32_t* s, uint32_t R, uint32_t warps) {
  uint32_t run = 0;
#pragma unroll 1
  for (uint32_t q = 0; q < warps; q += 4) {  // warps come in fours
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = s[(q + k) * R];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s[(q + k) * R] = run;
      run += x[k];
    }
  }
  return run;
}

// Exclusive prefix sums of s[0 .. R) by all `threads` threads of the block (a
// multiple of 32, at most 1024). w: one value a warp. These kernels run through
// their code once, so its length is time: loops are kept as loops.
__device__ __forceinline__ void block_prefix(uint32_t* s, uint32_t R, uint32_t threads, uint32_t* w) {
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint32_t per = (R + threads - 1) / threads;
  const uint32_t lo = min(R, t * per), hi = min(R, lo + per);
  uint32_t sum = 0;
#pragma unroll 1
  for (uint32_t k = lo; k < hi; ++k) sum += s[k];
  uint32_t run = sum;
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= (uint32_t)o) run += x;
  }
  if (lane == 31) w[warp] = run;
  __syncthreads();
  if (warp == 0) {
    uint32_t x = lane < threads / 32 ? w[lane] : 0;
#pragma unroll 1
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= (uint32_t)o) x += y;
    }
    w[lane] = x;
  }
  __syncthreads();
  run += (warp ? w[warp - 1] : 0) - sum;
#pragma unroll 1
  for (uint32_t k = lo; k < hi; ++k) {
    const uint32_t x = s[k];
    s[k] = run;
    run += x;
  }
  __syncthreads();
}

// All passes over at most kSmallMax pairs by one cluster. A warp has 32 x
// rounds pairs in order, the blocks read one another's digit counts from shared
// memory. With one pass the digits are the keys, and their prefix sums the
// offsets.
template <class I>
__global__ void __launch_bounds__(kSmallThreads)
plan_small_kernel(PlanArgs A, uint32_t rounds, int digit_bits, int passes, uint32_t* k0, uint32_t* v0, uint32_t* k1,
                  uint32_t* v1) {
  extern __shared__ uint32_t smem[];
  __shared__ uint32_t s_warp[32];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), blocks = cluster.num_blocks();
  const uint32_t threads = blockDim.x, warps = threads / 32;
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint32_t R = 1u << digit_bits;
  uint32_t* s_total = smem;       // [R] the block's pairs of a digit
  uint32_t* s_base = s_total + R;  // [R] first place of the digit
  uint32_t* s_before = s_base + R;  // [R] its pairs in the blocks before
  uint32_t* s_count = s_before + R;  // [warps][R] a warp's; then those of the warps before
  uint32_t* mine = s_count + warp * R;
  const uint32_t first = rank * (rounds * threads) + warp * (rounds * 32) + lane;
  const uint32_t *kin = nullptr, *vin = nullptr;
  uint32_t *kout = k0, *vout = v0;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    const bool last = pass + 1 == passes;
    uint32_t key[kSmallRounds], val[kSmallRounds], place[kSmallRounds];
#pragma unroll
    for (uint32_t j = 0; j < kSmallRounds; ++j) {
      if (j >= rounds) break;
      const uint32_t e = first + j * 32;
      key[j] = val[j] = 0;
      if (e < A.n) {
        key[j] = pass ? key_at<void>(kin, e, 0) : key_at<I>(A.ids, e, A.rows);
        val[j] = pass ? __ldcg(vin + e) : e;
      }
    }
    for (uint32_t e = t; e < warps * R; e += threads) s_count[e] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t j = 0; j < kSmallRounds; ++j) {
      if (j >= rounds) break;
      place[j] = place_in(mine, (key[j] >> shift) & (R - 1), digit_bits, first + j * 32 < A.n);
    }
    __syncthreads();
    for (uint32_t d = t; d < R; d += threads) s_total[d] = warps_prefix(s_count + d, R, warps);
    cluster.sync();
    for (uint32_t d = t; d < R; d += threads) {
      uint32_t before = 0, all = 0;
#pragma unroll 2
      for (uint32_t q = 0; q < blocks; ++q) {
        const uint32_t x = *cluster.map_shared_rank(s_total + d, q);
        if (q < rank) before += x;
        all += x;
      }
      s_base[d] = all;
      s_before[d] = before;
    }
    __syncthreads();
    block_prefix(s_base, R, threads, s_warp);
    if (passes == 1 && rank == 0)
      for (uint32_t d = t; d <= A.rows; d += threads) A.offsets[d] = s_base[d];
#pragma unroll
    for (uint32_t j = 0; j < kSmallRounds; ++j) {
      if (j >= rounds || first + j * 32 >= A.n) break;
      const uint32_t d = (key[j] >> shift) & (R - 1);
      const uint32_t pos = s_base[d] + s_before[d] + mine[d] + place[j];
      if (last) {
        A.keys[pos] = key[j];
        A.order[pos] = val[j];
        A.slot[val[j]] = key[j] < A.rows ? pos : kNoSlot;
      } else {
        __stcg(kout + pos, key[j]);
        __stcg(vout + pos, val[j]);
      }
    }
    cluster.sync();  // the pairs are in place, and nobody reads this block's counts any more
    kin = kout;
    vin = vout;
    kout = kout == k0 ? k1 : k0;
    vout = vout == v0 ? v1 : v0;
  }
}

// Up to so many tiles a scatter sums the counts of the tiles before it itself
// (then hist is [tile][digit]), which saves a launch: 14.9 us for the plan of
// 16,384 ids instead of 18.4, at 65,536 both take 19. Above, plan_scan_kernel
// does it for all.
constexpr uint32_t kDirectTiles = 64;

// Pairs of each digit in a tile: hist[digit][tile].
template <class I, uint32_t ROUNDS>
__global__ void __launch_bounds__(kTileThreads)
plan_hist_kernel(const void* __restrict__ src, uint32_t n, uint32_t rows, int shift, uint32_t R, uint32_t tiles,
                 uint32_t* __restrict__ hist) {
  __shared__ uint32_t s_count[1 << kMostBits];
  grid_dependency_wait();
  const uint32_t t = threadIdx.x;
  for (uint32_t d = t; d < R; d += kTileThreads) s_count[d] = 0;
  __syncthreads();
  const uint64_t first = (uint64_t)blockIdx.x * (kTileThreads * ROUNDS) + t;
  uint32_t key[ROUNDS];
#pragma unroll
  for (uint32_t j = 0; j < ROUNDS; ++j) {
    const uint64_t e = first + j * kTileThreads;
    key[j] = e < n ? key_at<I>(src, e, rows) : ~0u;
  }
#pragma unroll
  for (uint32_t j = 0; j < ROUNDS; ++j)
    if (first + j * kTileThreads < n) atomicAdd(&s_count[(key[j] >> shift) & (R - 1)], 1u);
  __syncthreads();
  const bool direct = tiles <= kDirectTiles;
  for (uint32_t d = t; d < R; d += kTileThreads)
    hist[direct ? (uint64_t)blockIdx.x * R + d : (uint64_t)d * tiles + blockIdx.x] = s_count[d];
}

// A digit's counts become those of the tiles before; its total beside them.
__global__ void __launch_bounds__(256)
plan_scan_kernel(uint32_t tiles, uint32_t* __restrict__ hist, uint32_t* __restrict__ total) {
  __shared__ uint32_t s_part[1024], s_warp[32];
  grid_dependency_wait();
  uint32_t* h = hist + (uint64_t)blockIdx.x * tiles;
  uint32_t run = 0;
  for (uint32_t t0 = 0; t0 < tiles; t0 += 1024) {
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t t = t0 + k * 256 + threadIdx.x;
      s_part[k * 256 + threadIdx.x] = t < tiles ? h[t] : 0;
    }
    __syncthreads();
    const uint32_t end = s_part[1023];
    block_prefix(s_part, 1024, 256, s_warp);
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      const uint32_t t = t0 + k * 256 + threadIdx.x;
      if (t < tiles) h[t] = run + s_part[k * 256 + threadIdx.x];
    }
    run += s_part[1023] + end;
    __syncthreads();
  }
  if (threadIdx.x == 0) total[blockIdx.x] = run;
}

// A tile's pairs, sorted by digit in shared memory first so that each digit's
// run is written in one piece. Blocks of 256 threads that share an SM by fours
// measured best: the plan of 1,521,797 pairs over 32,768 rows takes 48 us, 7 %
// more with six of them, 4 % more with blocks of 512 threads by twos (the same
// at 800,000 and 3,000,000 pairs).
template <class I, uint32_t ROUNDS, bool LAST>
__global__ void __launch_bounds__(kTileThreads, 4)
plan_scatter_kernel(PlanArgs A, const void* __restrict__ src, const uint32_t* __restrict__ vin, int shift,
                    int bits, uint32_t tiles, const uint32_t* __restrict__ hist,
                    const uint32_t* __restrict__ total, uint32_t* __restrict__ kout, uint32_t* __restrict__ vout) {
  constexpr uint32_t kWarps = kTileThreads / 32, kTile = kTileThreads * ROUNDS;
  const uint32_t R = 1u << bits;
  extern __shared__ uint32_t smem[];
  uint32_t* s_start = smem;            // [R] first place of the digit in the tile
  uint32_t* s_glob = s_start + R;      // [R] its first place among all, less s_start
  uint32_t* s_count = s_glob + R;      // [kWarps][R] a warp's; then those of the warps before
  uint32_t* s_key = s_count;           // [kTile] once the places are known
  uint32_t* s_val = s_key + kTile;     // [kTile]
  __shared__ uint32_t s_warp[32];
  grid_dependency_wait();
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const uint64_t tile0 = (uint64_t)blockIdx.x * kTile;
  const uint32_t in_tile = (uint32_t)min((uint64_t)kTile, A.n - tile0);
  const uint32_t first = warp * (ROUNDS * 32) + lane;
  uint32_t key[ROUNDS], place[ROUNDS];
#pragma unroll
  for (uint32_t j = 0; j < ROUNDS; ++j) {
    const uint32_t q = first + j * 32;
    key[j] = q < in_tile ? key_at<I>(src, tile0 + q, A.rows) : 0;
  }
  for (uint32_t e = t; e < kWarps * R; e += kTileThreads) s_count[e] = 0;
  constexpr uint32_t kDigits = (1u << kMostBits) / kTileThreads;  // of a thread
  uint32_t before[kDigits];  // the digit's pairs in the tiles before
#pragma unroll
  for (uint32_t k = 0; k < kDigits; ++k) {
    const uint32_t d = t + k * kTileThreads;
    before[k] = 0;
    if (d >= R) break;
    if (tiles <= kDirectTiles) {
      uint32_t all = 0;
#pragma unroll 8
      for (uint32_t q = 0; q < tiles; ++q) {
        const uint32_t x = hist[q * R + d];
        before[k] += q < blockIdx.x ? x : 0;
        all += x;
      }
      s_glob[d] = all;
    } else {
      before[k] = hist[(uint64_t)d * tiles + blockIdx.x];
      s_glob[d] = total[d];
    }
  }
  __syncthreads();
  uint32_t* mine = s_count + warp * R;
#pragma unroll
  for (uint32_t j = 0; j < ROUNDS; ++j)
    place[j] = place_in(mine, (key[j] >> shift) & (R - 1), bits, first + j * 32 < in_tile);
  block_prefix(s_glob, R, kTileThreads, s_warp);
  for (uint32_t d = t; d < R; d += kTileThreads) s_start[d] = warps_prefix(s_count + d, R, kWarps);
  __syncthreads();
  block_prefix(s_start, R, kTileThreads, s_warp);
#pragma unroll
  for (uint32_t k = 0; k < kDigits; ++k) {
    const uint32_t d = t + k * kTileThreads;
    if (d < R) s_glob[d] += before[k] - s_start[d];
  }
#pragma unroll
  for (uint32_t j = 0; j < ROUNDS; ++j) {
    const uint32_t d = (key[j] >> shift) & (R - 1);
    place[j] += s_start[d] + mine[d];
  }
  __syncthreads();  // the counts' memory holds the pairs from here on
#pragma unroll
  for (uint32_t j = 0; j < ROUNDS; ++j) {
    const uint32_t q = first + j * 32;
    if (q < in_tile) {
      s_key[place[j]] = key[j];
      s_val[place[j]] = std::is_same_v<I, void> ? __ldcg(vin + tile0 + q) : (uint32_t)(tile0 + q);
    }
  }
  __syncthreads();
#pragma unroll
  for (uint32_t j = 0; j < ROUNDS; ++j) {
    const uint32_t q = j * kTileThreads + t;
    if (q >= in_tile) break;
    const uint32_t k = s_key[q], v = s_val[q];
    const uint32_t pos = s_glob[(k >> shift) & (R - 1)] + q;
    if (LAST) {
      A.keys[pos] = k;
      A.order[pos] = v;
      A.slot[v] = k < A.rows ? pos : kNoSlot;
    } else {
      kout[pos] = k;
      vout[pos] = v;
    }
  }
}

// offsets[v] = first place whose key is >= v, for rows far more than places:
// by bisection, a thread a row.
__global__ void __launch_bounds__(256) plan_offsets_kernel(PlanArgs A) {
  grid_dependency_wait();
  const uint32_t v = blockIdx.x * 256u + threadIdx.x;
  if (v > A.rows) return;
  uint32_t lo = 0, hi = A.n;
  while (lo < hi) {
    const uint32_t mid = lo + ((hi - lo) >> 1);
    if (A.keys[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  A.offsets[v] = lo;
}

// The same for rows of the places' number: place p (n included) fills the rows
// behind the key before it up to its own. A warp fills the gaps of its 32
// places as one run of rows, the block one that is longer than kWarpFill.
// Q: places of a thread, several when there are enough blocks anyway.
constexpr uint32_t kWarpFill = 1024;
template <int Q>
__global__ void __launch_bounds__(256) plan_borders_kernel(PlanArgs A) {
  __shared__ uint32_t s_gaps, s_lo[256 * Q], s_hi[256 * Q], s_place[256 * Q];
  grid_dependency_wait();
  if (threadIdx.x == 0) s_gaps = 0;
  __syncthreads();
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t p0 = (uint64_t)blockIdx.x * (256 * Q) + threadIdx.x;
  uint32_t lo[Q], hi[Q];  // rows to fill
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const uint64_t p = p0 + q * 256;
    lo[q] = hi[q] = 0;
    if (p <= A.n) {
      if (p) lo[q] = A.keys[p - 1] + 1;
      hi[q] = p < A.n ? A.keys[p] + 1 : A.rows + 1;
    }
  }
#pragma unroll
  for (int q = 0; q < Q; ++q) {
    const uint32_t p = (uint32_t)(p0 + q * 256);
    uint32_t gap = lo[q] < hi[q] ? hi[q] - lo[q] : 0;
    if (gap > kWarpFill) {
      const uint32_t g = atomicAdd(&s_gaps, 1u);
      s_lo[g] = lo[q];
      s_hi[g] = hi[q];
      s_place[g] = p;
      gap = 0;
    }
    if (gap == 1) {  // the most when there are few rows
      A.offsets[lo[q]] = p;
      gap = 0;
    }
    if (!__any_sync(0xffffffffu, gap != 0)) continue;
    uint32_t end = gap;  // of the gaps up to this lane's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, end, o);
      if (lane >= (uint32_t)o) end += x;
    }
    const uint32_t total = __shfl_sync(0xffffffffu, end, 31);
    for (uint32_t f0 = 0; f0 < total; f0 += 32) {
      const uint32_t f = f0 + lane;
      uint32_t l = 0;  // the lane whose gap has the f-th row: the first whose end is behind f
#pragma unroll
      for (int o = 16; o > 0; o >>= 1)
        if (__shfl_sync(0xffffffffu, end, l + o - 1) <= f) l += o;
      l = min(l, 31u);
      const uint32_t row = __shfl_sync(0xffffffffu, lo[q] + gap - end, l) + f;
      const uint32_t place = __shfl_sync(0xffffffffu, p, l);
      if (f < total) A.offsets[row] = place;
    }
  }
  __syncthreads();
  for (uint32_t g = 0; g < s_gaps; ++g)
    for (uint64_t v = (uint64_t)s_lo[g] + threadIdx.x; v < s_hi[g]; v += 256) A.offsets[v] = s_place[g];
}

int plan_borders(Ctx* c, const PlanArgs& A) {
  const bool four = A.n >= 1024u * 8 * (uint32_t)c->sm_count;
  const unsigned per = four ? 1024 : 256;
  MVR_CUDA(c, launch_pdl(four ? plan_borders_kernel<4> : plan_borders_kernel<1>, A.n / per + 1, 256, 0, c->stream, A));
  return MVR_OK;
}

struct Digits {
  int bits, passes;
  explicit Digits(uint64_t rows) {
    int b = 1;
    while ((rows >> b) != 0) ++b;  // keys are 0 .. rows
    passes = (b + kMostBits - 1) / kMostBits;
    bits = (b + passes - 1) / passes;
  }
};

// Whether one cluster does it. A pass takes it as long as the tiles' two
// launches at some 7,000 pairs: over 32,768 rows 15.2 us against 17.6 at 6,000
// pairs, 17.2 against 14.8 at 8,193 (three passes, 3,000,000 rows: 40 against
// 43, 44 against 42). A single pass has the offsets beside it, which the tiles
// need another launch for: over 800 rows 12.3 against 14.3 us at 12,000 pairs,
// 13.9 against 12.3 at 16,384, the most the cluster holds.
bool is_small(uint64_t n, const Digits& D) { return n <= (D.passes == 1 ? kSmallMax : kSmallMaxPasses); }

// Pairs a thread of a tile: few while the tiles are one wave of four blocks an
// SM, then the most that 64 registers hold. Few give more blocks to wait at
// once, many fewer counts to sum and longer runs to write; the plan over 1,000 /
// 32,768 / 1,000,000 rows in us:
//   450,000 pairs    4 each: 22 / 27 / 43    11 each: 25 / 33 / 48
//   606,209          27 / 31 / 51            25 / 34 / 48
//   800,000          33 / 37 / 64            27 / 35 / 50
//   1,521,797        53 / 57 / 102           37 / 49 / 70
// A workspace is asked for without a device at hand, so the SMs are a number
// here: those of a B200.
constexpr uint32_t kFewRounds = 4, kManyRounds = 11;
bool few_rounds(uint64_t n) { return n <= 148ull * 4 * kFewRounds * kTileThreads; }

// Workspace: two sets of pairs for the passes, and the counts of the tiles.
struct PlanSpace {
  uint64_t k0, v0, k1, v1, hist, sums, total;
  PlanSpace(uint64_t n, uint64_t rows) {
    const Digits D(rows);
    const bool small = is_small(n, D);
    const uint64_t tile = kTileThreads * (few_rounds(n) ? kFewRounds : kManyRounds);
    uint64_t off = 0;
    auto take = [&](uint64_t words) {
      const uint64_t o = off;
      off += up256(words * 4);
      return o;
    };
    k0 = take(D.passes > 1 ? n : 0);
    v0 = take(D.passes > 1 ? n : 0);
    k1 = take(D.passes > 2 ? n : 0);
    v1 = take(D.passes > 2 ? n : 0);
    hist = take(small ? 0 : ((n + tile - 1) / tile) << D.bits);
    sums = take(small ? 0 : 1ull << D.bits);
    total = off;
  }
};

template <class I>
int plan_small(Ctx* c, const PlanArgs& A, const Digits& D, uint32_t* k0, uint32_t* v0, uint32_t* k1, uint32_t* v1) {
  // another block joins for every 256 pairs
  const uint32_t R = 1u << D.bits, threads = kSmallThreads;
  const uint32_t blocks = std::min(kSmallBlocks, pow2_ceil((A.n + 256u - 1) / 256u));
  const uint32_t chunk = (A.n + blocks - 1) / blocks;
  const uint32_t rounds = (chunk + threads - 1) / threads;
  const size_t smem = (3 + (size_t)threads / 32) * R * 4;  // 44 KB at most: needs no request
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = blocks;
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = c->stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  MVR_CUDA(c, cudaLaunchKernelEx(&cfg, plan_small_kernel<I>, A, rounds, D.bits, D.passes, k0, v0, k1, v1));
  return MVR_OK;
}

// One pass over the tiles; I: what it reads its keys from.
template <class I, uint32_t ROUNDS>
int plan_pass_of(Ctx* c, const PlanArgs& A, const void* kin, const uint32_t* vin, int shift, int bits, bool last,
                 uint32_t* kout, uint32_t* vout, uint32_t* hist, uint32_t* sums) {
  cudaStream_t st = c->stream;
  constexpr uint32_t kTile = kTileThreads * ROUNDS;
  const uint32_t tiles = (uint32_t)((A.n + (kTile - 1ull)) / kTile), R = 1u << bits;
  const size_t smem = (2 * R + std::max(kTileThreads / 32 * R, 2 * kTile)) * 4;  // 40 KB at most: needs no request
  const auto count = plan_hist_kernel<I, ROUNDS>;
  MVR_CUDA(c, launch_pdl(count, tiles, kTileThreads, 0, st, kin, A.n, A.rows, shift, R, tiles, hist));
  if (tiles > kDirectTiles) MVR_CUDA(c, launch_pdl(plan_scan_kernel, R, 256, 0, st, tiles, hist, sums));
  const auto scatter = last ? plan_scatter_kernel<I, ROUNDS, true> : plan_scatter_kernel<I, ROUNDS, false>;
  MVR_CUDA(c, launch_pdl(scatter, tiles, kTileThreads, smem, st, A, kin, vin, shift, bits, tiles, hist, sums, kout,
                         vout));
  return MVR_OK;
}
template <class I>
int plan_pass(Ctx* c, const PlanArgs& A, const void* kin, const uint32_t* vin, int shift, int bits, bool last,
              uint32_t* kout, uint32_t* vout, uint32_t* hist, uint32_t* sums) {
  const auto pass = few_rounds(A.n) ? plan_pass_of<I, kFewRounds> : plan_pass_of<I, kManyRounds>;
  return pass(c, A, kin, vin, shift, bits, last, kout, vout, hist, sums);
}

int plan_tiles(Ctx* c, const PlanArgs& A, const Digits& D, uint32_t* k0, uint32_t* v0, uint32_t* k1, uint32_t* v1,
               uint32_t* hist, uint32_t* sums) {
  if (A.id_bytes == 8)
    MVR_TRY(plan_pass<uint64_t>(c, A, A.ids, nullptr, 0, D.bits, D.passes == 1, k0, v0, hist, sums));
  else
    MVR_TRY(plan_pass<uint32_t>(c, A, A.ids, nullptr, 0, D.bits, D.passes == 1, k0, v0, hist, sums));
  for (int pass = 1; pass < D.passes; ++pass) {
    MVR_TRY(plan_pass<void>(c, A, k0, v0, pass * D.bits, D.bits, pass + 1 == D.passes, k1, v1, hist, sums));
    std::swap(k0, k1);
    std::swap(v0, v1);
  }
  return MVR_OK;
}

}  // namespace
}  // namespace tok
}  // namespace mvr

using mvr::Ctx;

extern "C" {

int mvr_token_plan_bytes(uint64_t n_ids, uint64_t rows, uint64_t* bytes) {
  if (!bytes || n_ids > mvr::tok::kMaxIds || rows == 0 || rows > mvr::tok::kMaxRows) return MVR_E_INVALID_ARGUMENT;
  *bytes = n_ids ? mvr::tok::PlanSpace(n_ids, rows).total : 0;
  return MVR_OK;
}

int mvr_token_plan_device(mvr_ctx* h, const void* d_ids, int id_bytes, uint64_t n_ids, uint64_t rows,
                          uint32_t* d_offsets, uint32_t* d_order, uint32_t* d_keys, uint32_t* d_slot,
                          void* d_workspace, uint64_t workspace_bytes) {
  if (!h) return MVR_E_INVALID_ARGUMENT;
  Ctx* c = &h->impl;
  MVR_TRY(mvr::tok::check_ids(c, d_ids, id_bytes, n_ids, rows));
  if (n_ids > mvr::tok::kMaxIds) return mvr::tok::bad(c, "more than 2^31 - 1 ids");
  if (!d_offsets || (n_ids && (!d_order || !d_keys || !d_slot))) return mvr::tok::bad(c, "null pointer");
  if (!mvr::tok::aligned(d_offsets, 4) || !mvr::tok::aligned(d_order, 4) || !mvr::tok::aligned(d_keys, 4) ||
      !mvr::tok::aligned(d_slot, 4))
    return mvr::tok::bad(c, "an output is not aligned to its type");
  uint64_t need = 0;
  MVR_TRY(mvr_token_plan_bytes(n_ids, rows, &need));
  MVR_TRY(mvr::tok::check_workspace(c, d_workspace, workspace_bytes, need));
  mvr::DeviceScope dev_scope(c);
  MVR_TRY(dev_scope.status);
  cudaStream_t st = c->stream;
  if (n_ids == 0) {
    MVR_CUDA(c, cudaMemsetAsync(d_offsets, 0, (rows + 1) * 4, st));
    return MVR_OK;
  }
  const mvr::tok::PlanArgs A = {d_ids,     id_bytes, (uint32_t)n_ids, (uint32_t)rows,
                                d_offsets, d_order,  d_keys,          d_slot};
  const mvr::tok::PlanSpace ws(n_ids, rows);
  auto at = [&](uint64_t off) { return reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(d_workspace) + off); };
  const mvr::tok::Digits D(rows);
  if (mvr::tok::is_small(n_ids, D)) {
    const auto small = id_bytes == 8 ? mvr::tok::plan_small<uint64_t> : mvr::tok::plan_small<uint32_t>;
    MVR_TRY(small(c, A, D, at(ws.k0), at(ws.v0), at(ws.k1), at(ws.v1)));
    if (D.passes == 1) return MVR_OK;  // the offsets came with the counts
  } else {
    MVR_TRY(mvr::tok::plan_tiles(c, A, D, at(ws.k0), at(ws.v0), at(ws.k1), at(ws.v1), at(ws.hist), at(ws.sums)));
  }
  // Walking the places costs one read each, a search some twenty dependent ones
  // a row: the walk is for rows that do not outnumber the places by far.
  if (rows <= 8 * n_ids)
    MVR_TRY(mvr::tok::plan_borders(c, A));
  else
    MVR_CUDA(c, mvr::launch_pdl(mvr::tok::plan_offsets_kernel, (unsigned)(rows / 256 + 1), 256, 0, st, A));
  return MVR_OK;
}

}  // extern "C"
