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
// A cluster of blocks owns a row: each block a contiguous range of slots,
// keys in its shared memory, a radix select over histograms that the blocks
// read from one another's shared memory, and prefix sums over the blocks for
// the order. Then all warps of the cluster move rows. Bound by latency (a
// chain of block and cluster barriers) for short rows, by the bytes of the
// moved rows for long ones.
#include <cooperative_groups.h>

#include <algorithm>

#include "devutil.cuh"
#include "paged.h"

namespace cg = cooperative_groups;

namespace lc {
namespace {

constexpr int kEvictThreads = 512;
constexpr int kBins = 2048;  // 11 + 11 + 10 bits of the key
constexpr int kEvictMaxCluster = 8;
constexpr int64_t kEvictSmemKeys = 40 * 1024;  // 160 KB of keys a block

// Monotone map to unsigned; NaN below everything, -0 as 0.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Exclusive sum over the block of x; *total gets the block's sum.
__device__ __forceinline__ int block_scan(int x, int* warp_sum, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(~0u, inc, o);
    if (lane >= o) inc += up;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kEvictThreads / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    all += warp_sum[w];
  }
  *total = all;
  return before + inc - x;
}

__device__ __forceinline__ int64_t page_row(const PagedView& c, int s, int t) {
  const int page = c.tables[(int64_t)s * c.width + t / c.page_tokens];
  if (page < 0 || page >= c.n_pages) {
    *c.status = 1;
    return -1;
  }
  return page * c.page + (int64_t)(t % c.page_tokens) * c.token;
}

// U: the unit of a copy (uint4 where rows and strides are 16-byte aligned,
// else the element).
template <typename U>
__global__ void __launch_bounds__(kEvictThreads) k_paged_evict(const PagedEvictArgs a, const int cl, const int use_smem) {
  extern __shared__ uint32_t smem_keys[];
  __shared__ int hist[3][kBins];
  __shared__ int warp_sum[kEvictThreads / 32];
  __shared__ int sh_max, sh_bin, sh_need, sh_eq, sh_hole, sh_move;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x % cl;
  const int row = blockIdx.x / cl, s = row / a.c.hkv, h = row - s * a.c.hkv;
  const int cap = a.c.width * a.c.page_tokens;
  int n = a.c.lens[s];
  if (n < 0 || n > cap || n > a.stride) {
    *a.c.status = 1;
    n = n < 0 ? 0 : (int)min((int64_t)cap, a.stride);
  }
  const float* acc_in = a.acc_in + row * a.stride;
  const int* pos_in = a.pos_in + row * a.stride;
  float* acc_out = a.acc_out + row * a.stride;
  int* pos_out = a.pos_out + row * a.stride;
  const int per = (n + cl - 1) / cl, b = min(n, rank * per), e = min(n, b + per);
  if (n <= a.budget) {  // the same for every block of the cluster
    for (int t = b + tid; t < e; t += kEvictThreads) {
      acc_out[t] = acc_in[t];
      pos_out[t] = pos_in[t];
    }
    return;
  }
  uint32_t* keys = use_smem ? smem_keys : a.keys + row * a.stride + b;

  // the newest position
  int newest = INT32_MIN;
  for (int t = b + tid; t < e; t += kEvictThreads) newest = max(newest, pos_in[t]);
  if (tid == 0) sh_max = INT32_MIN;
  for (int i = tid; i < 3 * kBins; i += kEvictThreads) (&hist[0][0])[i] = 0;
  __syncthreads();
  newest = __reduce_max_sync(~0u, newest);
  if (lane == 0) atomicMax(&sh_max, newest);
  cluster.sync();
  newest = INT32_MIN;
  for (int r = 0; r < cl; ++r) newest = max(newest, *cluster.map_shared_rank(&sh_max, r));

  for (int t = b + tid; t < e; t += kEvictThreads) {
    const int p = pos_in[t];
    const bool held = p < a.n_sink || (int64_t)p > (int64_t)newest - a.n_recent;
    const uint32_t key = held ? 0xffffffffu : order_key(acc_in[t]);
    keys[t - b] = key;
    atomicAdd(&hist[0][key >> 21], 1);
  }

  // radix select of the budget-th largest key
  uint32_t prefix = 0;
  int need = a.budget;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    cluster.sync();
    constexpr int kPer = kBins / kEvictThreads;
    const int bins = pass == 2 ? 1024 : kBins, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    int mine[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int bin = bins - 1 - (tid * kPer + i);
      mine[i] = 0;
      if (bin >= 0)
        for (int r = 0; r < cl; ++r) mine[i] += *cluster.map_shared_rank(&hist[pass][bin], r);
      sum += mine[i];
    }
    int total;
    int above = block_scan(sum, warp_sum, &total);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      if (above < need && need <= above + mine[i]) {
        sh_bin = bins - 1 - (tid * kPer + i);
        sh_need = need - above;
      }
      above += mine[i];
    }
    __syncthreads();
    prefix |= (uint32_t)sh_bin << shift;
    need = sh_need;
    if (pass < 2) {
      const uint32_t mask = ~0u << shift;
      const int next = pass == 0 ? 10 : 0, width = pass == 0 ? kBins : 1024;
      for (int i = tid; i < e - b; i += kEvictThreads) {
        const uint32_t key = keys[i];
        if ((key & mask) == prefix) atomicAdd(&hist[pass + 1][(key >> next) & (width - 1)], 1);
      }
    }
  }

  // each thread owns a run of slots (odd length: one bank each)
  const int run = ((e - b + kEvictThreads - 1) / kEvictThreads) | 1;
  const int i0 = min(e - b, tid * run), i1 = min(e - b, i0 + run);
  int eq = 0, total;
  for (int i = i0; i < i1; ++i) eq += keys[i] == prefix;
  int eq_at = block_scan(eq, warp_sum, &total);
  if (tid == 0) sh_eq = total;
  cluster.sync();
  for (int r = 0; r < rank; ++r) eq_at += *cluster.map_shared_rank(&sh_eq, r);
  int holes = 0, movers = 0;
  for (int i = i0; i < i1; ++i) {
    const uint32_t key = keys[i];
    bool stay = key > prefix;
    if (key == prefix) stay = eq_at++ < need;
    keys[i] = stay;
    holes += b + i < a.budget && !stay;
    movers += b + i >= a.budget && stay;
  }
  int hole_at = block_scan(holes, warp_sum, &total);
  if (tid == 0) sh_hole = total;
  int move_at = block_scan(movers, warp_sum, &total);
  if (tid == 0) sh_move = total;
  cluster.sync();
  int pairs = 0;
  for (int r = 0; r < cl; ++r) {
    const int x = *cluster.map_shared_rank(&sh_hole, r);
    if (r < rank) {
      hole_at += x;
      move_at += *cluster.map_shared_rank(&sh_move, r);
    }
    pairs += x;
  }
  int* hole = a.list + row * 4 * a.list_cap;
  int* mover = hole + a.list_cap;
  for (int i = i0; i < i1; ++i) {
    const int t = b + i;
    if (t < a.budget && !keys[i]) hole[hole_at++] = t;
    if (t >= a.budget && keys[i]) {
      mover[move_at] = t;
      mover[a.list_cap + move_at] = __float_as_int(acc_in[t]);
      mover[2 * a.list_cap + move_at] = pos_in[t];
      ++move_at;
    }
  }
  __syncthreads();  // acc_out may be acc_in: the movers' values are read above
  for (int t = b + tid; t < e; t += kEvictThreads) {
    if (t >= a.budget) {
      acc_out[t] = 0.f;
      pos_out[t] = -1;
    } else if (keys[t - b]) {
      acc_out[t] = acc_in[t];
      pos_out[t] = pos_in[t];
    }
  }
  cluster.sync();

  // the moves: eight pairs a warp at a time
  const int units = a.c.d * a.esize / (int)sizeof(U);
  const int64_t per_u = sizeof(U) / a.esize;
  U* kb = static_cast<U*>(a.c.k) + (a.layer * a.c.layer + h * a.c.head) / per_u;
  U* vb = static_cast<U*>(a.c.v) + (a.layer * a.c.layer + h * a.c.head) / per_u;
  for (int p0 = (rank * (kEvictThreads / 32) + warp) * 8; p0 < pairs; p0 += cl * (kEvictThreads / 32) * 8) {
    int64_t src = -1, dst = -1;
    if (lane < 8 && p0 + lane < pairs) {
      const int to = hole[p0 + lane], from = mover[p0 + lane];
      dst = page_row(a.c, s, to);
      src = page_row(a.c, s, from);
      acc_out[to] = __int_as_float(mover[a.list_cap + p0 + lane]);
      pos_out[to] = mover[2 * a.list_cap + p0 + lane];
      if (src < 0) dst = -1;
    }
    int64_t from[8], to[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      from[i] = __shfl_sync(~0u, src, i) / per_u;
      to[i] = __shfl_sync(~0u, dst, i);
    }
    for (int x = lane; x < 2 * units; x += 32) {
      U* base = x >= units ? vb : kb;
      const int at = x >= units ? x - units : x;
      U got[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (to[i] >= 0) got[i] = base[from[i] + at];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (to[i] >= 0) base[to[i] / per_u + at] = got[i];
    }
  }
}

// Reordering: block (row j, layer, part). The group's mapping (who inherits
// which tail page) is worked out by every block from the parents; blocks of
// layer 0's first part write row j's table, and where row j is a later child
// of its parent, its blocks copy the first `fill` slots of the parent's tail
// page into the spare tail page that it takes.
template <typename U>
__global__ void __launch_bounds__(256) k_paged_reorder(const PagedReorderArgs a) {
  __shared__ int parent[kBeamMaxBeams], first[kBeamMaxBeams];
  __shared__ int owner;
  const int tid = threadIdx.x, w = a.n_beams;
  const int row = blockIdx.x, g = row / w, j = row - g * w;
  if (tid < w) first[tid] = INT32_MAX;
  __syncthreads();
  if (tid < w) {
    int p = a.parents[(int64_t)g * w + tid];
    if (p < 0 || p >= w) {
      *a.c.status = 1;
      p = tid;
    }
    parent[tid] = p;
    atomicMin(&first[p], tid);
  }
  __syncthreads();
  if (tid == 0) {
    int own = parent[j];
    if (first[own] != j) {  // the i-th later child takes the i-th childless beam's tail
      int i = 0;
      for (int x = 0; x < j; ++x) i += first[parent[x]] != x;
      own = -1;
      while (i >= 0) i -= first[++own] == INT32_MAX;
    }
    owner = own;
  }
  __syncthreads();
  const int p = parent[j], own = owner;
  const int cap = a.c.width * a.c.page_tokens;
  int n = a.c.lens[g];
  if (n < 0 || n > cap) {
    *a.c.status = 1;
    n = n < 0 ? 0 : cap;
  }
  const int full = n / a.c.page_tokens, fill = n - full * a.c.page_tokens;
  const int32_t* tables = a.c.tables + (int64_t)g * w * a.c.width;
  if (blockIdx.y == 0 && blockIdx.z == 0)
    for (int i = tid; i < a.c.width; i += 256) {
      const int from = i < full ? p : i == full && fill > 0 ? own : j;
      a.tables_out[(int64_t)row * a.c.width + i] = tables[(int64_t)from * a.c.width + i];
    }
  if (own == p || fill == 0) return;
  const int src = tables[(int64_t)p * a.c.width + full], dst = tables[(int64_t)own * a.c.width + full];
  if (src < 0 || src >= a.c.n_pages || dst < 0 || dst >= a.c.n_pages) {
    if (tid == 0) *a.c.status = 1;
    return;
  }
  const int64_t per_u = sizeof(U) / a.esize;
  const int units = (int)(a.c.d / per_u);
  const int is_v = blockIdx.z & 1, part = blockIdx.z >> 1, parts = gridDim.z >> 1;
  U* base = static_cast<U*>(is_v ? a.c.v : a.c.k) + blockIdx.y * a.c.layer / per_u;
  const int64_t total = (int64_t)a.c.hkv * fill * units;
  for (int64_t x = (int64_t)part * 256 + tid; x < total; x += (int64_t)parts * 256) {
    const int64_t r = x / units;
    const int c = (int)(x - r * units), h = (int)(r / fill), t = (int)(r - (int64_t)h * fill);
    const int64_t at = (h * a.c.head + t * a.c.token) / per_u + c;
    base[dst * a.c.page / per_u + at] = base[src * a.c.page / per_u + at];
  }
}

// Rows and strides of whole 16-byte units.
bool vector_rows(const PagedView& c, int esize) {
  const int64_t e = 16 / esize;
  return c.d % e == 0 && c.layer % e == 0 && c.page % e == 0 && c.head % e == 0 && c.token % e == 0 &&
         (reinterpret_cast<uintptr_t>(c.k) & 15) == 0 && (reinterpret_cast<uintptr_t>(c.v) & 15) == 0;
}

template <typename U>
void launch_evict(const PagedEvictArgs& a, int device, int sms, cudaStream_t s) {
  auto kernel = k_paged_evict<U>;
  static SmemOptIn opt;
  opt(kernel, kEvictSmemKeys * 4, device);
  const int64_t cap = std::min<int64_t>((int64_t)a.c.width * a.c.page_tokens, a.stride);
  const int rows = a.n_seqs * a.c.hkv, cl = paged_evict_cluster(rows, cap, sms);
  const bool in_smem = paged_evict_keys_in_smem(cap, cl);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * cl));
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = in_smem ? (size_t)((cap + cl - 1) / cl) * 4 : 0;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cl;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  LC_CUDA(cudaLaunchKernelEx(&cfg, kernel, a, cl, in_smem ? 1 : 0));
}

}  // namespace

// Blocks per row: enough that the rows fill the card, none with less than
// 1024 slots to itself.
int paged_evict_cluster(int32_t rows, int64_t cap, int32_t sms) {
  int cl = 1;
  while (cl < kEvictMaxCluster && (int64_t)rows * cl < 2 * sms && cap / (2 * cl) >= 1024) cl *= 2;
  while (cl < kEvictMaxCluster && !paged_evict_keys_in_smem(cap, cl)) cl *= 2;
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

void launch_paged_reorder(const PagedReorderArgs& a, cudaStream_t s) {
  const int64_t bytes = (int64_t)a.c.hkv * a.c.page_tokens * a.c.d * a.esize;  // of a whole page
  const unsigned parts = (unsigned)std::max<int64_t>(1, std::min<int64_t>(16, bytes / (32 << 10)));
  const dim3 grid((unsigned)(a.n_groups * a.n_beams), (unsigned)a.c.n_layers, 2 * parts);
  if (vector_rows(a.c, a.esize))
    k_paged_reorder<uint4><<<grid, 256, 0, s>>>(a);
  else if (a.esize == 4)
    k_paged_reorder<uint32_t><<<grid, 256, 0, s>>>(a);
  else
    k_paged_reorder<uint16_t><<<grid, 256, 0, s>>>(a);
  LC_CUDA(cudaGetLastError());
}

}  // namespace lc
