// Eviction from the uncompressed paged cache by accumulated attention weight
// (lc_paged_evict) and the reordering of beams' pages (lc_paged_reorder).
//
// Eviction, per (sequence, kv head) row of n slots: the `budget` slots with
// the largest (key, lower slot first) stay, key = acc, or above everything
// for the first n_sink and the last n_recent positions. Slots do not move
// for order's sake: attention does not depend on it and pos keeps each
// slot's position, so only the kept slots at or past `budget` move, each
// into a freed slot below it. That is the least that can be copied, the
// sources and targets are disjoint (no order among the copies), and a cache
// held at its budget moves one row a step instead of half of them.
//
// A block owns a row: keys in shared memory, a radix select of the budget-th
// largest over histograms of 11, 11 and 10 bits, and a prefix sum over runs of
// slots for the order. Of long rows a cluster of up to 8 blocks has a range of
// slots each and they read one another's histograms and counts; where a row's
// keys are more than their shared memory takes, keys are in global
// memory. Short lists are moved by the row's own blocks, long ones by a second
// kernel over the whole card.
//
// 128 rows of 1025 slots cut to 1024: 7.0 us, all of it the chain of loads and
// block barriers. 64 rows of 6001 to 8192 cut to 2048: 14.3 us of choosing
// (that chain, a fifth of it waiting for DRAM) and 17.7 of moving 95 MB, 5.4
// TB/s, or 0.82 of what a plain copy of the card's memory reaches.
#include <cooperative_groups.h>

#include <algorithm>

#include "devutil.cuh"
#include "paged.h"

namespace cg = cooperative_groups;

namespace lc {
namespace {

constexpr int kBins = 2048;  // 11 + 11 + 10 bits of the key
constexpr int kEvictMaxCluster = 8;
constexpr int64_t kEvictSmemKeys = 40 * 1024;  // 160 KB of keys a block
constexpr int64_t kEvictBlockSlots = 12288;    // see paged_evict_cluster
constexpr int kFusedMoves = 64;  // longest list that a row's own blocks move (a second launch costs more)
// pairs a warp looks up at a time: 16 and 8 took 35.2 us, 4 took 35.7 (64 rows of up to 8192)
constexpr int kMoveBatch = 16;
constexpr int kHeld = 8;  // slots whose acc and pos a thread holds in registers

// Monotone map to unsigned; NaN below everything, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the block of x (two counts in one word where a caller
// needs two); *total gets the block's sum.
template <int THREADS>
__device__ __forceinline__ uint64_t block_scan(uint64_t x, uint64_t* warp_sum, uint64_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t up = __shfl_up_sync(~0u, inc, o);
    if (lane >= o) inc += up;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  constexpr int W = THREADS / 32;
  uint64_t sums = lane < W ? warp_sum[lane] : 0;
#pragma unroll
  for (int o = 1; o < W; o <<= 1) {
    const uint64_t up = __shfl_up_sync(~0u, sums, o);
    if (lane >= o) sums += up;
  }
  *total = __shfl_sync(~0u, sums, W - 1);
  const uint64_t before = __shfl_sync(~0u, sums, warp > 0 ? warp - 1 : 0);
  return (warp > 0 ? before : 0) + inc - x;
}

// Offset in copy units of slot t's row, or -1 for a page id outside the pool.
__device__ __forceinline__ int64_t page_row(const PagedView& c, int s, int t) {
  const int page = c.tables[(int64_t)s * c.width + t / c.page_tokens];
  if (page < 0 || page >= c.n_pages) {
    c.status[kBadInput] = 1;
    return -1;
  }
  return page * c.page + (int64_t)(t % c.page_tokens) * c.token;
}

// Moves pairs [0, pairs) of a row's list: warp `first` of `warps`, B pairs at
// a time: their lookups by B lanes, then N copies in flight a lane.
template <typename U, int B, int N>
__device__ __forceinline__ void move_pairs(const PagedEvictArgs& a, int row, int pairs, int first, int warps) {
  const int lane = threadIdx.x & 31, s = row / a.c.hkv, h = row - s * a.c.hkv;
  const int* list = a.list + row * 4 * a.list_cap;
  U* kb = static_cast<U*>(a.c.k) + a.layer * a.c.layer + h * a.c.head;
  U* vb = static_cast<U*>(a.c.v) + a.layer * a.c.layer + h * a.c.head;
  const int units = a.c.d;
  for (int p0 = first * B; p0 < pairs; p0 += warps * B) {
    int64_t src = -1, dst = -1;
    if (lane < B && p0 + lane < pairs) {
      const int* pair = list + p0 + lane;
      const int to = pair[0], from = pair[a.list_cap];
      const int acc = pair[2 * a.list_cap], pos = pair[3 * a.list_cap];
      dst = page_row(a.c, s, to);
      src = page_row(a.c, s, from);
      a.acc_out[row * a.stride + to] = __int_as_float(acc);
      a.pos_out[row * a.stride + to] = pos;
      if (src < 0) dst = -1;
    }
    for (int q = 0; q < B && p0 + q < pairs; q += N)
      for (int x0 = 0; x0 < 2 * units; x0 += 32) {
        const int x = x0 + lane;
        U* base = x >= units ? vb + (x - units) : kb + x;
        U got[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int64_t from = __shfl_sync(~0u, src, q + i), to = __shfl_sync(~0u, dst, q + i);
          if (to >= 0 && x < 2 * units) got[i] = base[from];
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int64_t to = __shfl_sync(~0u, dst, q + i);
          if (to >= 0 && x < 2 * units) base[to] = got[i];
        }
      }
  }
}

// CL: the row has a cluster of blocks (else one). U: the unit of a copy, in
// which the view's strides and d are given.
template <typename U, int THREADS, bool CL>
__global__ void __launch_bounds__(THREADS, 1)
    k_paged_evict(const PagedEvictArgs a, const int cl_arg, const int use_smem) {
  extern __shared__ uint32_t smem_keys[];
  __shared__ __align__(16) int hist[3][kBins];
  __shared__ uint64_t warp_sum[THREADS / 32];
  __shared__ uint64_t sh_count;
  __shared__ int sh_max, sh_bin, sh_need, sh_equal, sh_eq;
  cg::cluster_group cluster = cg::this_cluster();
  const int cl = CL ? cl_arg : 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = CL ? blockIdx.x % cl : 0;
  const int row = CL ? blockIdx.x / cl : blockIdx.x, s = row / a.c.hkv, h = row - s * a.c.hkv;
  const int cap = a.c.width * a.c.page_tokens;
  auto sync = [&] {
    if (CL)
      cluster.sync();
    else
      __syncthreads();
  };
  auto remote = [&](auto* p, int r) { return CL ? cluster.map_shared_rank(p, r) : p; };
  const float* acc_in = a.acc_in + row * a.stride;
  const int* pos_in = a.pos_in + row * a.stride;
  float* acc_out = a.acc_out + row * a.stride;
  int* pos_out = a.pos_out + row * a.stride;
#pragma unroll
  for (int i = tid; i < 3 * kBins / 4; i += THREADS) reinterpret_cast<int4*>(hist)[i] = make_int4(0, 0, 0, 0);
  if (tid == 0) sh_max = INT32_MIN;
  pdl_wait();
  float held_acc[kHeld];
  int held_pos[kHeld];
  auto hold = [&](int from, int end) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
      const int t = from + tid + i * THREADS;
      if (t < end) {
        held_acc[i] = acc_in[t];
        held_pos[i] = pos_in[t];
      }
    }
  };
  if (!CL) hold(0, cap);  // a row's only block need not wait for its length to read ahead
  int n = a.c.lens[s];
  if (n < 0 || n > cap) {
    a.c.status[kBadInput] = 1;
    n = n < 0 ? 0 : cap;
  }
  const int per = CL ? (n + cl - 1) / cl : n, b = min(n, rank * per), e = min(n, b + per);
  if (CL) hold(b, e);
  // each slot of the block's range, in strides: f(slot, acc, pos)
  auto each = [&](auto&& f) {
    int t = b + tid;
#pragma unroll
    for (int i = 0; i < kHeld; ++i, t += THREADS)
      if (t < e) f(t, held_acc[i], held_pos[i]);
    // four loads before the first f, which may write where the compiler cannot tell them apart
    for (; t < e; t += 4 * THREADS) {
      float acc[4];
      int pos[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i * THREADS < e) {
          acc[i] = acc_in[t + i * THREADS];
          pos[i] = pos_in[t + i * THREADS];
        }
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (t + i * THREADS < e) f(t + i * THREADS, acc[i], pos[i]);
    }
  };
  if (n <= a.budget) {  // the same for every block of the cluster
    each([&](int t, float acc, int pos) {
      acc_out[t] = acc;
      pos_out[t] = pos;
    });
    if (!a.fused && rank == 0 && tid == 0) a.pairs[row] = 0;
    return;
  }
  uint32_t* keys = use_smem ? smem_keys : a.keys + row * a.stride + b;

  // the newest position
  int newest = INT32_MIN;
  each([&](int, float, int pos) { newest = max(newest, pos); });
  __syncthreads();
  newest = __reduce_max_sync(~0u, newest);
  if (lane == 0) atomicMax(&sh_max, newest);
  sync();
  newest = sh_max;
  if (CL) {
#pragma unroll
    for (int r = 0; r < kEvictMaxCluster; ++r)
      if (r < cl) newest = max(newest, *remote(&sh_max, r));
  }
  each([&](int t, float acc, int pos) {
    const bool held = pos < a.n_sink || (int64_t)pos > (int64_t)newest - a.n_recent;
    const uint32_t key = held ? 0xffffffffu : order_key(acc);
    keys[t - b] = key;
    atomicAdd(&hist[0][key >> 21], 1);
  });

  pdl_launch_dependents();

  // radix select of the budget-th largest key
  uint32_t prefix = 0;
  int need = a.budget;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    sync();
    constexpr int kPer = kBins / THREADS;
    const int bins = pass == 2 ? 1024 : kBins, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const int top = bins - 1 - tid * kPer;  // the highest bins first
    int mine[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) mine[i] = 0;
#pragma unroll
    for (int r = 0; r < (CL ? kEvictMaxCluster : 1); ++r)
      if (r < cl) {
        const int* from = remote(hist[pass], r);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (top - i >= 0) mine[i] += from[top - i];
      }
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum += mine[i];
    uint64_t total;
    int above = (int)block_scan<THREADS>((uint64_t)sum, warp_sum, &total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (above < need && need <= above + mine[i]) {
        sh_bin = top - i;
        sh_need = need - above;
        sh_equal = mine[i];
      }
      above += mine[i];
    }
    __syncthreads();
    prefix |= (uint32_t)sh_bin << shift;
    need = sh_need;
    if (pass < 2) {
      const uint32_t mask = ~0u << shift;
      const int next = pass == 0 ? 10 : 0, width = pass == 0 ? kBins : 1024;
#pragma unroll 4
      for (int i = tid; i < e - b; i += THREADS) {
        const uint32_t key = keys[i];
        if ((key & mask) == prefix) atomicAdd(&hist[pass + 1][(key >> next) & (width - 1)], 1);
      }
    }
  }

  // each thread owns a run of slots (odd length: one bank each)
  const int run = ((e - b + THREADS - 1) / THREADS) | 1;
  const int i0 = min(e - b, tid * run), i1 = min(e - b, i0 + run);
  uint64_t total;
  int eq_at = 0;
  if (need < sh_equal) {  // the first `need` of equal keys stay (the same for every block)
    int eq = 0;
    for (int i = i0; i < i1; ++i) eq += keys[i] == prefix;
    eq_at = (int)block_scan<THREADS>((uint64_t)eq, warp_sum, &total);
    if (tid == 0) sh_eq = (int)total;
    sync();
    for (int r = 0; r < rank; ++r) eq_at += *remote(&sh_eq, r);
  } else {
    need = INT32_MAX;
    __syncthreads();  // the run's keys were written by other threads' strides
  }
  uint64_t counts = 0;  // holes below, movers above 32 bits
  for (int i = i0; i < i1; ++i) {
    const uint32_t key = keys[i];
    bool stay = key > prefix;
    if (key == prefix) stay = eq_at++ < need;
    keys[i] = stay;
    if (b + i < a.budget)
      counts += !stay;
    else
      counts += (uint64_t)stay << 32;
  }
  uint64_t at = block_scan<THREADS>(counts, warp_sum, &total);
  if (CL) {
    if (tid == 0) sh_count = total;
    sync();
    total = 0;
#pragma unroll
    for (int r = 0; r < kEvictMaxCluster; ++r)
      if (r < cl) {
        const uint64_t x = *remote(&sh_count, r);
        if (r < rank) at += x;
        total += x;
      }
  }
  const int pairs = (int)(total & 0xffffffffu);
  int* hole = a.list + row * 4 * a.list_cap + (uint32_t)at;
  int* mover = a.list + row * 4 * a.list_cap + a.list_cap + (at >> 32);
  for (int i = i0; i < i1; ++i) {
    const int t = b + i;
    if (t < a.budget) {
      if (!keys[i]) *hole++ = t;
    } else if (keys[i]) {
      mover[0] = t;
      mover[a.list_cap] = __float_as_int(acc_in[t]);
      mover[2 * a.list_cap] = pos_in[t];
      ++mover;
    }
  }
  __syncthreads();  // acc_out may be acc_in: the movers' values are read above
  each([&](int t, float acc, int pos) {
    if (t >= a.budget) {
      acc_out[t] = 0.f;
      pos_out[t] = -1;
    } else if (keys[t - b]) {
      acc_out[t] = acc;
      pos_out[t] = pos;
    }
  });
  sync();

  if (a.fused) {
    move_pairs<U, 2, 2>(a, row, pairs, rank * (THREADS / 32) + warp, cl * (THREADS / 32));
  } else if (rank == 0 && tid == 0) {
    a.pairs[row] = pairs;
  }
}

// The moves of rows whose lists can be long, over the whole card.
template <typename U>
__global__ void __launch_bounds__(256, 4) k_paged_move(const PagedEvictArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  move_pairs<U, kMoveBatch, 8>(a, blockIdx.x, a.pairs[blockIdx.x], blockIdx.y * 8 + (threadIdx.x >> 5), gridDim.y * 8);
}

// Reordering: block (group, share). Every block works out the group's mapping
// from the parents: the first child of a beam inherits its tail page, the i-th
// later child takes that of the i-th beam without children. The tables and the
// copies of the tail pages' first `fill` slots are shared out over the group's
// blocks, so that they all have the same to do however the parents fall.
// Bound by the copied bytes: 8 groups of 8 beams, 16 layers, 32 slots of 8
// heads of 128 bf16 take 17.6 us, of which 14 are what a plain copy would take;
// one group over 4 layers 2.9, the launch and three dependent loads.
constexpr int kReorderThreads = 256, kReorderUnroll = 8, kReorderChunk = 32 * kReorderUnroll * 2;
template <typename U>
__global__ void __launch_bounds__(kReorderThreads) k_paged_reorder(const PagedReorderArgs a) {
  __shared__ int parent[kBeamMaxBeams], first[kBeamMaxBeams], owner[kBeamMaxBeams], spare[kBeamMaxBeams];
  __shared__ int64_t src[kBeamMaxBeams], dst[kBeamMaxBeams];
  __shared__ int extra_below, spare_below, n_copies;  // of the first 32 beams; of all
  const int tid = threadIdx.x, lane = tid & 31, w = a.n_beams, g = blockIdx.x;
  pdl_wait();
  pdl_launch_dependents();
  const int cap = a.c.width * a.c.page_tokens;
  const int32_t* tables = a.c.tables + (int64_t)g * w * a.c.width;
  int n = a.c.lens[g], p = 0;
  if (tid < w) {
    p = a.parents[(int64_t)g * w + tid];
    if (p < 0 || p >= w) {
      a.c.status[kBadInput] = 1;
      p = tid;
    }
    parent[tid] = p;
    first[tid] = INT32_MAX;
  }
  if (n < 0 || n > cap) {
    a.c.status[kBadInput] = 1;
    n = n < 0 ? 0 : cap;
  }
  __syncthreads();
  if (tid < w) atomicMin(&first[p], tid);
  __syncthreads();
  const int full = n / a.c.page_tokens, fill = n - full * a.c.page_tokens;
  if (tid < kBeamMaxBeams) {  // two warps: the i-th later child, the i-th childless beam
    const bool extra = tid < w && first[p] != tid, childless = tid < w && first[tid] == INT32_MAX;
    const uint32_t e = __ballot_sync(~0u, extra), s = __ballot_sync(~0u, childless), below = (1u << lane) - 1;
    if (tid == 0) {
      extra_below = __popc(e);
      spare_below = __popc(s);
    }
    asm volatile("bar.sync 1, %0;" ::"n"(kBeamMaxBeams) : "memory");
    const int at = __popc(e & below) + (tid >= 32 ? extra_below : 0);
    if (childless) spare[__popc(s & below) + (tid >= 32 ? spare_below : 0)] = tid;
    if (tid == kBeamMaxBeams - 1) n_copies = extra_below + __popc(e);
    asm volatile("bar.sync 1, %0;" ::"n"(kBeamMaxBeams) : "memory");
    if (tid < w) owner[tid] = extra ? spare[at] : p;
    if (extra && fill > 0) {
      const int from = tables[(int64_t)p * a.c.width + full], to = tables[(int64_t)spare[at] * a.c.width + full];
      const bool bad = from < 0 || from >= a.c.n_pages || to < 0 || to >= a.c.n_pages;
      if (bad) a.c.status[kBadInput] = 1;
      src[at] = bad ? -1 : from * a.c.page;
      dst[at] = to * a.c.page;
    }
  }
  __syncthreads();
  for (int x = blockIdx.y * kReorderThreads + tid; x < w * a.c.width; x += gridDim.y * kReorderThreads) {
    const int j = x / a.c.width, i = x - j * a.c.width;
    const int from = i < full ? parent[j] : i == full && fill > 0 ? owner[j] : j;
    a.tables_out[(int64_t)g * w * a.c.width + x] = tables[(int64_t)from * a.c.width + i];
  }
  if (fill == 0) return;
  // the copies' chunks: (copy, layer, K or V, head, chunk of its slots' units), a warp each
  const int units = a.c.d, per_head = units * fill, chunks = (per_head + kReorderChunk - 1) / kReorderChunk;
  const int64_t total = (int64_t)n_copies * a.c.n_layers * 2 * a.c.hkv * chunks;
  const bool packed = a.c.token == units;
  for (int64_t x = (int64_t)blockIdx.y * (kReorderThreads / 32) + (tid >> 5); x < total;
       x += (int64_t)gridDim.y * (kReorderThreads / 32)) {
    const int64_t item = x / chunks;
    const int chunk = (int)(x - item * chunks), pool = (int)(item / a.c.hkv), h = (int)(item - (int64_t)pool * a.c.hkv);
    const int copy = pool / (2 * a.c.n_layers), lp = pool - copy * 2 * a.c.n_layers;
    if (src[copy] < 0) continue;
    U* base = static_cast<U*>(lp & 1 ? a.c.v : a.c.k) + (lp >> 1) * a.c.layer + h * a.c.head;
    const U* from = base + src[copy];
    U* to = base + dst[copy];
    const int end = min(per_head, (chunk + 1) * kReorderChunk);
    for (int z0 = chunk * kReorderChunk + lane; z0 < end; z0 += 32 * kReorderUnroll) {
      U got[kReorderUnroll];
      auto at = [&](int z) -> int64_t {
        if (packed) return z;
        const int t = z / units;
        return t * a.c.token + (z - t * units);
      };
#pragma unroll
      for (int i = 0; i < kReorderUnroll; ++i)
        if (z0 + 32 * i < end) got[i] = from[at(z0 + 32 * i)];
#pragma unroll
      for (int i = 0; i < kReorderUnroll; ++i)
        if (z0 + 32 * i < end) to[at(z0 + 32 * i)] = got[i];
    }
  }
}

// The view with strides and d in units of U.
template <typename U>
PagedView in_units(PagedView c, int esize) {
  const int64_t e = sizeof(U) / esize;
  c.layer /= e;
  c.page /= e;
  c.head /= e;
  c.token /= e;
  c.d = (int32_t)(c.d / e);
  return c;
}

template <typename U>
void launch_move(const PagedEvictArgs& a, int rows, int sms, cudaStream_t s) {
  if (a.fused) return;
  const int64_t most = (a.list_cap + 8 * kMoveBatch - 1) / (8 * kMoveBatch), fill = (4ll * sms + rows - 1) / rows;
  launch_pdl(k_paged_move<U>, dim3((unsigned)rows, (unsigned)std::min<int64_t>(most, fill)), dim3(256), 0, s, a);
}

template <typename U>
void launch_evict(PagedEvictArgs a, int device, int sms, cudaStream_t s) {
  const int64_t cap = std::min<int64_t>((int64_t)a.c.width * a.c.page_tokens, a.stride);
  const int rows = a.n_seqs * a.c.hkv, cl = paged_evict_cluster(cap, rows, sms);
  const bool in_smem = paged_evict_keys_in_smem(cap, cl);
  const size_t smem = in_smem ? (size_t)((cap + cl - 1) / cl) * 4 : 0;
  a.c = in_units<U>(a.c, a.esize);
  a.fused = a.list_cap <= kFusedMoves;
  if (cl == 1) {
    auto one = [&](auto kernel, int threads, SmemOptIn& opt) {
      opt(kernel, kEvictSmemKeys * 4, device);
      launch_pdl(kernel, dim3(rows), dim3(threads), smem, s, a, 1, (int)in_smem);
    };
    static SmemOptIn small, large;
    if (cap <= 2048)
      one(k_paged_evict<U, 256, false>, 256, small);
    else
      one(k_paged_evict<U, 1024, false>, 1024, large);
    LC_CUDA(cudaGetLastError());
    launch_move<U>(a, rows, sms, s);
    return;
  }
  static SmemOptIn opt;
  opt(k_paged_evict<U, 1024, true>, kEvictSmemKeys * 4, device);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cl));
  cfg.blockDim = dim3(1024);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  LC_CUDA(cudaLaunchKernelEx(&cfg, k_paged_evict<U, 1024, true>, a, cl, in_smem ? 1 : 0));
  launch_move<U>(a, rows, sms, s);
}

template <typename U>
void launch_reorder(PagedReorderArgs a, int sms, cudaStream_t s) {
  a.c = in_units<U>(a.c, a.esize);
  // blocks of a group: all groups' as many as run at once, no more than every
  // warp has a chunk where every beam but one is copied
  const int64_t chunks = (a.c.page_tokens * (int64_t)a.c.d + kReorderChunk - 1) / kReorderChunk;
  const int64_t all = 2 * chunks * a.c.n_layers * a.c.hkv * std::max(1, a.n_beams - 1);
  const int64_t y = std::min<int64_t>((all + 7) / 8, (8ll * sms + a.n_groups - 1) / a.n_groups);
  const dim3 grid((unsigned)a.n_groups, (unsigned)std::min<int64_t>(y, 65535));
  launch_pdl(k_paged_reorder<U>, grid, dim3(kReorderThreads), 0, s, a);
}

}  // namespace

// Blocks per row: one up to 12288 slots, more of longer ones while all rows'
// blocks run at once, and as many as hold the row's keys in shared memory. A
// cluster's barriers cost what its blocks bring for shorter rows: with one, two
// and four blocks 32 rows of 12000 slots took 14, 16 and 19 us, 16 of 16384
// 29, 26 and 25, 8 of 32768 51, 40 and 28 (36 with eight).
int paged_evict_cluster(int64_t cap, int rows, int sms) {
  int cl = 1;
  while (cl < kEvictMaxCluster &&
         (!paged_evict_keys_in_smem(cap, cl) || (cap > cl * kEvictBlockSlots && 2 * cl * rows <= sms)))
    cl *= 2;
  return cl;
}

bool paged_evict_keys_in_smem(int64_t cap, int cluster) { return (cap + cluster - 1) / cluster <= kEvictSmemKeys; }

void launch_paged_evict(const PagedEvictArgs& a, int32_t device, int32_t sms, cudaStream_t s) {
  if (vector_rows(a.c, a.esize))
    launch_evict<uint4>(a, device, sms, s);
  else if (a.esize == 4)
    launch_evict<uint32_t>(a, device, sms, s);
  else
    launch_evict<uint16_t>(a, device, sms, s);
}

void launch_paged_reorder(const PagedReorderArgs& a, int32_t sms, cudaStream_t s) {
  if (vector_rows(a.c, a.esize))
    launch_reorder<uint4>(a, sms, s);
  else if (a.esize == 4)
    launch_reorder<uint32_t>(a, sms, s);
  else
    launch_reorder<uint16_t>(a, sms, s);
  LC_CUDA(cudaGetLastError());
}

}  // namespace lc
