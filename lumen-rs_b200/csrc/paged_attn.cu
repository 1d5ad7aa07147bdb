// Decode attention over the uncompressed paged cache (lc_paged_attn), the
// accumulated attention weights (lc_paged_attn_weights) and the append.
//
//   s_gt = scale q_g . k_t,  p_gt = exp(s_gt - max_t s_gt) / sum_t,
//   out_g = sum_t p_gt v_t          over the slots lo <= t < n of a sequence
//
// One pass over K and V with the running maximum m and sum l of a softmax:
// a tile's scores rescale what was summed before by 2^(m_old - m_new). The
// bytes of K and V bound it: a kv head's `group` query heads are computed
// together so that each row is read once.
//
// Work split: the tiles of all (sequence, kv head, group of query heads)
// items form one list, and every block takes an equal run of it, whatever
// the sequences' lengths are: a long sequence alone fills the card and a
// batch of ragged ones leaves no tail. The lengths are read on the device
// (no host copy, and a captured graph follows them). An item that lies in
// one run is finished by its block; of one that spans several, each block
// leaves (m, l, o) in its slot and the last to arrive joins them, in slot
// order, so results do not depend on the order of arrival. Of one item alone
// (one sequence, one kv head) the parts are joined through one SM: 131072
// slots of 128 bf16 take 30 us, 10 of them the bytes.
#include <algorithm>

#include "devutil.cuh"
#include "paged.h"

namespace lc {
namespace {

constexpr float kNegInf = -INFINITY;
// What an item costs a block beyond its tiles, in tiles (see build_prefix):
// 0, 8, 16 and 32 took 128, 119, 110 and 97 us for 32 sequences of 1 to 8192
// slots on the tensor cores, 37, 30, 30 and 29 for a window of 1024; the FMA
// kernel's tiles cost more each, and 64 sequences of 128 to 512 f32
// slots took 150, 144, 156 and 180.
constexpr int kMmaCost = 32, kFmaCost = 8;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }

__device__ __forceinline__ float load_f32(const void* p, int64_t i, int dtype) {
  if (dtype == LC_F32) return static_cast<const float*>(p)[i];
  if (dtype == LC_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_f32(void* p, int64_t i, int dtype, float x) {
  if (dtype == LC_F32)
    static_cast<float*>(p)[i] = x;
  else if (dtype == LC_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(x);
}

// A sequence's length within what its table can hold.
__device__ __forceinline__ int clamp_len(const PagedView& c, int s) {
  const int cap = c.width * c.page_tokens, n = c.lens[s];
  if (n < 0 || n > cap) {
    c.status[kBadInput] = 1;
    return n < 0 ? 0 : cap;
  }
  return n;
}

__device__ __forceinline__ int first_slot(int n, int window) { return window > 0 && n > window ? n - window : 0; }

// Offset in elements of slot t's row (head 0, this call's layer), or -1 for a
// page id outside the pool.
__device__ __forceinline__ int64_t row_offset(const PagedView& c, int s, int t) {
  const int page = c.tables[(int64_t)s * c.width + t / c.page_tokens];
  if (page < 0 || page >= c.n_pages) {
    c.status[kBadInput] = 1;
    return -1;
  }
  return page * c.page + (int64_t)(t % c.page_tokens) * c.token;
}

// prefix[s] = length in the list of the sequences before s (of one item each);
// prefix[n_seqs] the total. An item of t tiles takes cost + t places: the
// first ones are no tiles but stand for what beginning and ending an item
// costs, so that a block's share holds less of others the more items it has.
// Sequences with nothing to attend to take no place and get their zeros here.
// Every thread of the block calls it.
template <int THREADS>
__device__ void build_prefix(const PagedAttnArgs& a, int tile, int cost, int* prefix) {
  __shared__ int warp_sum[THREADS / 32];
  const int tid = threadIdx.x, per = (a.n_seqs + THREADS - 1) / THREADS;
  const int b = min(a.n_seqs, tid * per), e = min(a.n_seqs, b + per);
  auto places_of = [&](int s) {
    const int n = clamp_len(a.c, s);
    return n == 0 ? 0 : cost + (n - 1) / tile - first_slot(n, a.window) / tile + 1;
  };
  int sum = 0;
  for (int s = b; s < e; ++s) sum += places_of(s);
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(~0u, inc, o);
    if ((tid & 31) >= o) inc += up;
  }
  if ((tid & 31) == 31) warp_sum[tid >> 5] = inc;
  __syncthreads();
  int at = inc - sum;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w)
    if (w < (tid >> 5)) at += warp_sum[w];
  for (int s = b; s < e; ++s) {
    prefix[s] = at;
    at += per == 1 ? sum : places_of(s);
  }
  if (tid == THREADS - 1) prefix[a.n_seqs] = at;
  __syncthreads();
  const int heads = a.c.hkv * a.group, d = a.c.d;
  for (int s = blockIdx.x; s < a.n_seqs; s += gridDim.x) {
    if (prefix[s + 1] != prefix[s]) continue;
    for (int x = tid; x < heads * d; x += THREADS) store_f32(a.out, (int64_t)s * heads * d + x, a.out_dtype, 0.f);
    if (a.stats)
      for (int x = tid; x < 2 * heads; x += THREADS) a.stats[2ll * s * heads + x] = 0.f;
  }
}

// A block's share of one item: tiles [j0, j1) of sequence s, item hh (kv head
// and head group) of it.
struct Segment {
  int s, hh, j0, j1, n, lo;  // j1 <= j0: places only
  int t0;                    // tile 0's first slot: lo, down to whole tiles
  int next;                  // where the block goes on in the list
  // the item's blocks are first .. first + parts - 1; block b's partial is in
  // slot 2 b, or 2 b + 1 where the item does not begin its run (the first only)
  int first, parts, slot0, slot;
};

__device__ __forceinline__ Segment find_segment(const PagedAttnArgs& a, const int* prefix, int tile, int cost, int hh_n,
                                                int per, int u, int u_end) {
  Segment g;
  const int key = u / hh_n;
  int b = 0, e = a.n_seqs;  // the last s with prefix[s] <= key
  while (e - b > 1) {
    const int mid = (b + e) >> 1;
    if (prefix[mid] <= key)
      b = mid;
    else
      e = mid;
  }
  g.s = b;
  const int places = prefix[b + 1] - prefix[b], r = u - prefix[b] * hh_n;
  g.hh = r / places;
  const int start = prefix[b] * hh_n + g.hh * places + cost;  // the item's first tile
  const int end = start + places - cost;
  g.j0 = max(u, start) - start;
  g.j1 = min(end, u_end) - start;
  g.next = min(end, u_end);
  g.n = clamp_len(a.c, b);
  g.lo = first_slot(g.n, a.window);
  g.t0 = g.lo - g.lo % tile;
  g.first = start / per;
  g.parts = (end - 1) / per - g.first + 1;
  // an item begins its first block's run unless other places are before its own
  g.slot0 = 2 * g.first + (g.first * per < start - cost ? 1 : 0);
  g.slot = (int)blockIdx.x == g.first ? g.slot0 : 2 * (int)blockIdx.x;
  return g;
}

// Joins the warps' (m, l, o) of a segment (shared memory: om, ol [warps][GP],
// oo [warps][GP][DP]) and writes the item's rows, its partial, or, as the last
// block of a split item, the join of all its partials. Block-wide; the weights
// of the sums are worked out once a head, in om and (for the partials) in oo.
template <int THREADS, int GP, int DP>
__device__ void finish_segment(const PagedAttnArgs& a, const Segment& g, int hg_n, float* om, const float* ol,
                               float* oo) {
  constexpr int W = THREADS / 32;
  constexpr int64_t kSlot = GP * (DP + 2);
  __shared__ int last;
  __shared__ float scale[GP];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, d = a.c.d;
  const int h = g.hh / hg_n, head0 = (g.hh - h * hg_n) * GP, nh = min(GP, a.group - head0);
  const int64_t row0 = (int64_t)g.s * a.c.hkv * a.group + (int64_t)h * a.group + head0;
  float* part = a.part + g.slot * kSlot;
  auto row_stats = [&](int i, float m, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // no slot with a finite score: zeros
    scale[i] = inv;
    if (a.stats && i < nh) {
      a.stats[2 * (row0 + i)] = m == kNegInf ? 0.f : m;
      a.stats[2 * (row0 + i) + 1] = inv;
    }
  };
  __syncthreads();
  if (tid < GP) {
    float m = kNegInf, l = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) m = fmaxf(m, om[w * GP + tid]);
    const float mg = m == kNegInf ? 0.f : m;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = ex2(om[w * GP + tid] - mg);
      l += f * ol[w * GP + tid];
      om[w * GP + tid] = f;
    }
    if (g.parts == 1) {
      row_stats(tid, m, l);
    } else {
      part[tid] = m;
      part[GP + tid] = l;
    }
  }
  __syncthreads();
  for (int e = tid; e < nh * DP; e += THREADS) {
    const int i = e / DP, x = e % DP;
    if (x >= d) continue;
    float o = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) o = fmaf(om[w * GP + i], oo[(w * GP + i) * DP + x], o);
    if (g.parts == 1)
      store_f32(a.out, (row0 + i) * d + x, a.out_dtype, o * scale[i]);
    else
      part[2 * GP + i * DP + x] = o;
  }
  if (g.parts > 1) {
    int* counter = a.counters + (int64_t)g.s * a.c.hkv * hg_n + g.hh;
    __syncthreads();
    if (tid == THREADS - 1) {  // a thread without loads in flight, which a fence would wait for
      __threadfence();         // the block's writes, which the barrier put before this thread
      last = atomicAdd(counter, 1) == g.parts - 1;
      if (last) {
        *counter = 0;
        __threadfence();
      }
    }
    __syncthreads();
    if (last) {
      // In few instructions rather than unrolled: they are fetched for this one
      // time (74 parts took 20 to 30 us with all loads of a thread unrolled).
      const float* first_part = a.part + g.slot0 * kSlot;
      const float* parts = a.part + 2 * g.first * kSlot;  // + 2 b kSlot: part b > 0
      for (int i = warp; i < nh; i += W) {
        float m = kNegInf, l = 0.f;
#pragma unroll 1
        for (int b = lane; b < g.parts; b += 32) {
          const float* from = (b == 0 ? first_part : parts + 2 * b * kSlot) + i;
          const float pm = __ldcg(from), pl = __ldcg(from + GP);
          const float mn = fmaxf(m, pm), mg = mn == kNegInf ? 0.f : mn;
          l = l * ex2(m - mg) + pl * ex2(pm - mg);
          m = mn;
          oo[b * GP + i] = pm;
        }
        float top = m;
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
        const float mg = top == kNegInf ? 0.f : top;
        l *= ex2(m - mg);
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
        if (lane == 0) {
          row_stats(i, top, l);
          om[i] = mg;
        }
      }
      __syncthreads();
      // four dimensions a thread, the parts shared out where threads are left
      constexpr int kVecs = GP * DP / 4, kShare = THREADS > kVecs ? THREADS / kVecs : 1;
      float4* sums = reinterpret_cast<float4*>(oo + kPagedMaxBlocks * GP);
      const int share = kShare > 1 ? tid / kVecs : 0;
      for (int v = tid - share * kVecs; v < nh * DP / 4 && share < kShare; v += THREADS) {
        const int i = v * 4 / DP, x = v * 4 % DP;
        const float mg = om[i];
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (share == 0) {
          const float f = ex2(oo[i] - mg);
          o = __ldcg(reinterpret_cast<const float4*>(first_part + 2 * GP) + v);
          o.x *= f;
          o.y *= f;
          o.z *= f;
          o.w *= f;
        }
#pragma unroll 8
        for (int b = share == 0 ? kShare : share; b < g.parts; b += kShare) {
          const float4 p = __ldcg(reinterpret_cast<const float4*>(parts + 2 * b * kSlot + 2 * GP) + v);
          const float f = ex2(oo[b * GP + i] - mg);
          o.x = fmaf(f, p.x, o.x);
          o.y = fmaf(f, p.y, o.y);
          o.z = fmaf(f, p.z, o.z);
          o.w = fmaf(f, p.w, o.w);
        }
        if (kShare > 1) {
          sums[share * kVecs + v] = o;
          continue;
        }
        const float r[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (x + c < d) store_f32(a.out, (row0 + i) * d + x + c, a.out_dtype, r[c] * scale[i]);
      }
      if (kShare > 1) {
        __syncthreads();
        for (int e = tid; e < nh * DP; e += THREADS) {
          const int i = e / DP, x = e % DP;
          if (x >= d) continue;
          float o = 0.f;
#pragma unroll
          for (int b = 0; b < kShare; ++b) o += reinterpret_cast<const float*>(sums + b * kVecs)[e];
          store_f32(a.out, (row0 + i) * d + x, a.out_dtype, o * scale[i]);
        }
      }
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

// The FMA kernel: products and sums in f32 for pools of any of the three
// types, head dimension up to DP. A warp owns whole tiles of TT = 32 / LPT
// slots: LPT lanes share a slot's dot product, 16 bytes at a time in turn, and
// for the values the lanes own dimensions. Rows sit in shared memory as f32
// with 4 LPT words of padding, which keeps the eight lanes of a 16-byte read
// phase on different banks.
//
// ST > 1: f32 pools whose rows are whole 16-byte units, through ST stages of
// cp.async a warp. What a warp waits for its own products bounds it, so as many
// warps as shared memory takes with two stages of small tiles: one sequence of
// 65536 slots, 8 heads of 128 under 32 queries takes 92 us, 5.9 TB/s, with 11
// warps, 93 with 10, 96 with 8, and 98 with 4 of three stages of tiles twice
// as long; one of 131072, 4 heads of 256, 167 and 201. Under 8 queries a head
// the reads of q do, eight of 16 bytes for one of K: 4 of 81000 slots, 2 heads
// of 96, 165 us, of which 76 the bytes; shared memory's port is busy 72 % of
// it, the FMA pipes 28 %. One of 19 slots, 2 heads of 80: 5.4, the launch and
// one tile.
// ST = 1: 16-bit pools by 16-byte loads into registers (VEC), or any alignment
// and type, value by value: 32 sequences of 2048 slots, 8 heads of 128 bf16
// under f32 queries take 129 us so and 470 value by value, bound by their
// instructions (the tensor cores take 53 under bf16 queries).
template <typename T, int DP, int GP, int W, int ST, bool VEC>
__global__ void __launch_bounds__(W * 32, ST > 1 ? 1 : 2) k_paged_attn(const PagedAttnArgs a) {
  constexpr int LPT = ST > 1 ? DP / 32 : DP / 64, TT = 32 / LPT, PITCH = DP + 4 * LPT, VL = DP / 32;
  constexpr int kCost = ST > 1 ? 2 * kFmaCost : kFmaCost;
  constexpr int TILE = TT * PITCH, CH = DP / 4;
  extern __shared__ __align__(16) uint8_t smem[];
  float* tiles = reinterpret_cast<float*>(smem);  // [W][ST][K, V][TT][PITCH]
  float* qs = tiles + W * ST * 2 * TILE;          // [GP][DP]
  float* ps = qs + GP * DP;                       // [W][TT][GP]
  float* om = ps + W * TT * GP;                   // [W][GP]
  float* ol = om + W * GP;
  int* prefix = reinterpret_cast<int*>(ol + W * GP);
  float* oo = tiles;  // [W][GP][DP]: the tiles' room, free when a segment ends
  static_assert(GP * DP <= 2 * TILE && kPagedMaxBlocks * GP + W * 128 <= W * ST * 2 * TILE,
                "the warps' outputs, and the joins' weights and sums, fit the tiles");
  static_assert(ST == 1 || sizeof(T) == 4, "cp.async does not convert");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hg_n = (a.group + GP - 1) / GP, hh_n = a.c.hkv * hg_n;
  pdl_wait();
  pdl_launch_dependents();
  build_prefix<W * 32>(a, TT, kCost, prefix);
  const int total = prefix[a.n_seqs] * hh_n;
  const int per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, a.min_tiles);
  const int u_end = min(total, ((int)blockIdx.x + 1) * per);
  float* mine = tiles + warp * ST * 2 * TILE;
  const uint32_t mine_at = (uint32_t)__cvta_generic_to_shared(mine);
  float* pw = ps + warp * TT * GP;
  const int tok = lane / LPT, part = lane % LPT;
  auto dim = [&](int x) { return DP == 64 ? lane * 2 + x : (x >> 2) * 128 + lane * 4 + (x & 3); };
  for (int u = blockIdx.x * per; u < u_end;) {
    const Segment g = find_segment(a, prefix, TT, kCost, hh_n, per, u, u_end);
    u = g.next;
    if (g.j1 <= g.j0) continue;
    const int h = g.hh / hg_n, head0 = (g.hh - h * hg_n) * GP, nh = min(GP, a.group - head0);
    const T* kb = static_cast<const T*>(a.c.k) + a.layer * a.c.layer + h * a.c.head;
    const T* vb = static_cast<const T*>(a.c.v) + a.layer * a.c.layer + h * a.c.head;
    const int32_t* table = a.c.tables + (int64_t)g.s * a.c.width;

    // lane r looks up slot r of a tile
    auto page_of = [&](int j) -> int {
      const int t = g.t0 + j * TT + lane;
      return j < g.j1 && lane < TT && t >= g.lo && t < g.n ? table[t / a.c.page_tokens] : INT32_MIN;
    };
    auto row_of = [&](int j, int page) -> int64_t {
      const int t = g.t0 + j * TT + lane;
      if (page >= 0 && page < a.c.n_pages) return page * a.c.page + (int64_t)(t % a.c.page_tokens) * a.c.token;
      if (page != INT32_MIN) a.c.status[kBadInput] = 1;
      return -1;
    };
    auto issue = [&](int j, int stage, int page) {
      if (j < g.j1) {
        const int64_t off = row_of(j, page);
        const uint32_t to = mine_at + stage * 2 * TILE * 4;
#pragma unroll
        for (int x = 0; x < TT * CH / 32; ++x) {
          const int e = x * 32 + lane, r = e / CH, c = e - r * CH;
          const int64_t o = __shfl_sync(~0u, off, r);
          const bool read = o >= 0 && c * 4 < a.c.d;
          const int64_t from = read ? o + c * 4 : 0;
          cp_async16_or_zero(to + (r * PITCH + c * 4) * 4, kb + from, read);
          cp_async16_or_zero(to + (TILE + r * PITCH + c * 4) * 4, vb + from, read);
        }
      }
      cp_commit();
    };

    // VEC: a tile's 16-byte units in registers, fetched while the one before is worked on
    constexpr int CV = DP * (int)sizeof(T) / 16, E = 16 / (int)sizeof(T), N = VEC ? TT * CV / 32 : 1;
    uint4 kg[N], vg[N];
    auto fetch = [&](int j, int page) {
      if (j >= g.j1) return;
      const int64_t row = row_of(j, page);
#pragma unroll
      for (int x = 0; x < N; ++x) {
        const int e = x * 32 + lane, r = e / CV, c = e - r * CV;
        const int64_t off = __shfl_sync(~0u, row, r);
        kg[x] = vg[x] = make_uint4(0, 0, 0, 0);
        if (off >= 0 && c * E < a.c.d) {
          kg[x] = *reinterpret_cast<const uint4*>(kb + off + c * E);
          vg[x] = *reinterpret_cast<const uint4*>(vb + off + c * E);
        }
      }
    };
    auto spread = [&](float* to, const uint4& u) {
      const T* x = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < E; i += 4)
        *reinterpret_cast<float4*>(to + i) =
            make_float4(to_f32(x[i]), to_f32(x[i + 1]), to_f32(x[i + 2]), to_f32(x[i + 3]));
    };

    const int first = g.j0 + warp;
    int page = page_of(first);
    if constexpr (VEC) {
      fetch(first, page);
      page = page_of(first + W);
    }
    if constexpr (ST > 1) {
#pragma unroll
      for (int i = 0; i < ST - 1; ++i) {
        const int now = page;
        page = page_of(first + (i + 1) * W);
        issue(first + i * W, i, now);
      }
    }
    const int64_t qrow = ((int64_t)g.s * a.c.hkv + h) * a.group + head0;
    for (int e = tid; e < GP * DP; e += W * 32) {
      const int i = e / DP, x = e - i * DP;
      qs[e] = i < nh && x < a.c.d ? load_f32(a.q, (qrow + i) * a.c.d + x, a.q_dtype) * a.scale_log2 : 0.f;
    }
    __syncthreads();
    float m[GP], l[GP], o[GP][VL];
#pragma unroll
    for (int i = 0; i < GP; ++i) {
      m[i] = kNegInf;
      l[i] = 0.f;
#pragma unroll
      for (int x = 0; x < VL; ++x) o[i][x] = 0.f;
    }
    int stage = 0, fill = ST - 1;
    for (int j = first; j < g.j1; j += W) {
      const int t0 = g.t0 + j * TT;
      const bool seen = t0 + tok >= g.lo && t0 + tok < g.n;
      if constexpr (ST > 1) {
        cp_wait<(ST > 1 ? ST - 2 : 0)>();
        __syncwarp();
        issue(j + (ST - 1) * W, fill, page);
        page = page_of(j + ST * W);
      } else if constexpr (VEC) {
#pragma unroll
        for (int x = 0; x < N; ++x) {
          const int e = x * 32 + lane, r = e / CV, c = e - r * CV;
          spread(mine + r * PITCH + c * E, kg[x]);
          spread(mine + TILE + r * PITCH + c * E, vg[x]);
        }
        __syncwarp();
        fetch(j + W, page);
        page = page_of(j + 2 * W);
      } else {
        const int64_t row = row_of(j, page);
        page = page_of(j + W);
#pragma unroll 4
        for (int r = 0; r < TT; ++r) {
          const int64_t off = __shfl_sync(~0u, row, r);
#pragma unroll
          for (int x = 0; x < VL; ++x) {
            const int c = x * 32 + lane;
            const bool in = off >= 0 && c < a.c.d;
            mine[r * PITCH + c] = in ? to_f32(kb[off + c]) : 0.f;
            mine[TILE + r * PITCH + c] = in ? to_f32(vb[off + c]) : 0.f;
          }
        }
        __syncwarp();
      }
      const float* kw = mine + stage * 2 * TILE;
      const float* vw = kw + TILE;
      fill = stage;
      stage = stage + 1 == ST ? 0 : stage + 1;

      float s[GP];
#pragma unroll
      for (int i = 0; i < GP; ++i) s[i] = 0.f;
#pragma unroll 4
      for (int c = 0; c < DP / (4 * LPT); ++c) {
        const int x = 4 * (c * LPT + part);
        const float4 kk = *reinterpret_cast<const float4*>(kw + tok * PITCH + x);
#pragma unroll
        for (int i = 0; i < GP; ++i) {
          const float4 qq = *reinterpret_cast<const float4*>(qs + i * DP + x);
          s[i] = fmaf(kk.x, qq.x, fmaf(kk.y, qq.y, fmaf(kk.z, qq.z, fmaf(kk.w, qq.w, s[i]))));
        }
      }
      bool grow = false;
#pragma unroll
      for (int i = 0; i < GP; ++i) {
#pragma unroll
        for (int b = 1; b < LPT; b <<= 1) s[i] += __shfl_xor_sync(~0u, s[i], b);
        if (!seen) s[i] = kNegInf;
        grow |= s[i] > m[i];
      }
      if (a.scores && part == 0 && seen) {
        float* to = a.scores + (((int64_t)g.s * a.c.hkv + h) * a.score_tokens + t0 + tok) * a.group + head0;
#pragma unroll
        for (int i = 0; i < GP; ++i)
          if (i < nh) to[i] = s[i];
      }
      if (__any_sync(~0u, grow)) {
#pragma unroll
        for (int i = 0; i < GP; ++i) {
          float top = s[i];
#pragma unroll
          for (int b = LPT; b < 32; b <<= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, b));
          top = fmaxf(top, m[i]);
          const float f = ex2(m[i] - (top == kNegInf ? 0.f : top));
          m[i] = top;
          l[i] *= f;
#pragma unroll
          for (int x = 0; x < VL; ++x) o[i][x] *= f;
        }
      }
#pragma unroll
      for (int i = 0; i < GP; ++i) {
        const float p = ex2(s[i] - (m[i] == kNegInf ? 0.f : m[i]));
        if (part == 0) {
          l[i] += p;
          pw[tok * GP + i] = p;
        }
      }
      __syncwarp();
#pragma unroll 4
      for (int r = 0; r < TT; ++r) {
        float v[VL], p[GP];
        if constexpr (DP == 64) {
          *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(vw + r * PITCH + lane * 2);
        } else {
#pragma unroll
          for (int x = 0; x < VL / 4; ++x)
            *reinterpret_cast<float4*>(v + 4 * x) =
                *reinterpret_cast<const float4*>(vw + r * PITCH + x * 128 + lane * 4);
        }
#pragma unroll
        for (int i = 0; i < GP / 4; ++i)
          *reinterpret_cast<float4*>(p + 4 * i) = *reinterpret_cast<const float4*>(pw + r * GP + 4 * i);
#pragma unroll
        for (int i = 0; i < GP; ++i)
#pragma unroll
          for (int x = 0; x < VL; ++x) o[i][x] = fmaf(p[i], v[x], o[i][x]);
      }
      __syncwarp();
    }
    if constexpr (ST > 1) cp_wait<0>();
    __syncthreads();
#pragma unroll
    for (int i = 0; i < GP; ++i) {
      float sum = l[i];
#pragma unroll
      for (int b = 1; b < 32; b <<= 1) sum += __shfl_xor_sync(~0u, sum, b);
      if (lane == 0) {
        om[warp * GP + i] = m[i];
        ol[warp * GP + i] = sum;
      }
#pragma unroll
      for (int x = 0; x < VL; ++x) oo[(warp * GP + i) * DP + dim(x)] = o[i][x];
    }
    finish_segment<W * 32, GP, DP>(a, g, hg_n, om, ol, oo);
  }
}

// ---- 16-bit pools on the tensor cores --------------------------------------
__device__ __forceinline__ void mma_16(float* c, const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  mma16816(c, a[0], a[1], a[2], a[3], b0, b1);
}
__device__ __forceinline__ void mma_16(float* c, const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// (x, y) as a sum of parts of 16 bits, the largest first. Three of bf16 hold all
// 24 bits of an f32; of two, outputs were off by 2^-17 and differed from those of
// f32 weights in 1e-4 of their norm. Two of f16 hold 22 bits, of numbers up to 1
// scaled by 2^15 (f16 ends at 65504) down to 2^-18 of it; below, they are off by
// 2^-40, the half step of f16's least numbers. Unscaled that was 2^-25: a slot of
// a 2^20-th of the largest weight had 5 bits, and those below 2^-25 were lost.
template <typename T>
constexpr int kParts = 2;
template <>
constexpr int kParts<__nv_bfloat16> = 3;
template <typename T>
constexpr float kScale = 32768.f;
template <>
constexpr float kScale<__nv_bfloat16> = 1.f;
__device__ __forceinline__ void split_16(float x, float y, uint32_t (&part)[2], __half) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  part[0] = h2_as_u32(h);
  part[1] = h2_as_u32(__floats2half2_rn(x - f.x, y - f.y));
}
__device__ __forceinline__ void split_16(float x, float y, uint32_t (&part)[3], __nv_bfloat16) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    const float2 f = __bfloat1622float2(h);
    part[i] = *reinterpret_cast<const uint32_t*>(&h);
    x -= f.x;
    y -= f.y;
  }
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// One box of a pool into shared memory, completing on an mbarrier.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int token, int head, int page,
                                         int layer, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
      "%6}], [%7];" ::"r"(dst),
      "l"(map), "r"(x), "r"(token), "r"(head), "r"(page), "r"(layer), "r"(bar)
      : "memory");
}

// The tensor-core kernel: 16-bit pools whose rows are whole 16-byte units,
// queries of the pool's type, head dimension up to DP.
//
// S^T = K Q^T and O^T = V^T P^T by m16n8k16 products: slots (then dimensions)
// are the 16 rows and up to 8 query heads the 8 columns, so a group of 8 heads
// wastes nothing and every K and V byte is read from shared memory once, as a
// fragment of the larger operand. The products take a fifth of what the
// HBM-bound pace leaves room for, which is why these are warp-wide products
// and not tcgen05's: its smallest tile has 64 rows of one operand against the
// 8 here, and no two warps share a tile. P is fed as a sum of 16-bit parts (see
// kParts), which makes the output's own rounding the only one that shows; the
// third of bf16 costs 0.5 us of 94 for one sequence of 131072 and nothing in a
// batch. The products cut what does not fit their f32 sums, so each tile starts
// from zero and its sums are added to O by rounding: run on from tile to tile
// they were 3e-6 off after 8192 slots, and are 3e-7 so (the plain form 1.7e-6).
// That takes 0.4 us of 29 in a window of 1024 with dimension 256 and none in a
// batch; four blocks of dimensions at a time, one after the other 1.3.
//
// Each warp runs its own pipeline over tiles of 16 slots in ST stages, no block
// barrier inside a segment. Slots outside the sequence or its window weigh
// nothing and their V rows are zeros in shared memory, whatever memory holds.
//
// TMA: pages of whole 8 slots, d >= 64. One lane fetches a tile with boxes of
// BR slots x 64 dimensions in the 128-byte swizzle, which puts the eight rows
// of an ldmatrix on different banks. Else: cp.async of 16 bytes a lane into
// rows with 16 bytes of padding. The latter's addresses are half of the
// instructions of a tile, and a warp that has eight to share an SM with must
// not take longer than the SM's share of the HBM does.
//
// 32 sequences of 8192 slots, 8 kv heads of 128 bf16: 174 us, 6.2 TB/s, 0.94 of
// a plain copy; the tensor pipe is busy 21 % and the issue slots 28 %. One of
// 131072: 95 us, 5.7 TB/s. What is left is the first loads' latency (4.5 us),
// items' ends and beginnings (3.7 us each) and SMs that reach the memory at
// different speeds (blocks with equal shares end between 0.75 and 1 of the
// whole time). 16 sequences of up to 4096 under a window of 1024, 8 heads of
// 256 f16: 29.1 us, 3.9 TB/s, where the first two are a third.
template <typename T, int DP, int W, int ST, bool TMA, int PER_SM>
__global__ void __launch_bounds__(W * 32, PER_SM)
    k_paged_attn_mma(const PagedAttnArgs a, const __grid_constant__ CUtensorMap k_map,
                     const __grid_constant__ CUtensorMap v_map) {
  constexpr int GP = 8, TT = 16, CH = DP / 8, PITCH = TMA ? DP * 2 : DP * 2 + 16, TILE = TT * PITCH, kCost = kMmaCost;
  extern __shared__ __align__(1024) uint8_t smem[];
  float* om = reinterpret_cast<float*>(smem + W * ST * 2 * TILE);
  float* ol = om + W * GP;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ol + W * GP);  // [W][ST], TMA
  int* prefix = reinterpret_cast<int*>(bars + W * ST);
  float* oo = reinterpret_cast<float*>(smem);  // [W][GP][DP]: the stages' room, free when a segment ends
  static_assert(GP * DP * 4 <= ST * 2 * TILE && (kPagedMaxBlocks * GP + W * 128) * 4 <= W * ST * 2 * TILE,
                "the warps' outputs, and the joins' weights and sums, fit the stages");
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gr = lane >> 2, tg = lane & 3;
  const int hg_n = (a.group + GP - 1) / GP, hh_n = a.c.hkv * hg_n;
  const uint32_t bar = (uint32_t)__cvta_generic_to_shared(bars + warp * ST);
  if (TMA && lane == 0) {
#pragma unroll
    for (int i = 0; i < ST; ++i) mbar_init(bar + 8 * i, 1);
    mbar_init_fence();
  }
  pdl_wait();
  pdl_launch_dependents();
  build_prefix<W * 32>(a, TT, kCost, prefix);
  const int total = prefix[a.n_seqs] * hh_n;
  const int per = max((total + (int)gridDim.x - 1) / (int)gridDim.x, a.min_tiles);
  const int u_end = min(total, ((int)blockIdx.x + 1) * per);
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem), stages = base + warp * ST * 2 * TILE;
  // this lane's row and 16-byte half in the fragments of K (slots x dimensions)
  // and V (transposed); under the swizzle a row's chunk c is at c ^ (row & 7)
  const int k_row = lane & 15, k_half = lane >> 4, v_row = (lane & 7) + ((lane >> 4) << 3), v_half = (lane >> 3) & 1;
  uint32_t k_at[TMA ? 4 : 1], v_at[TMA ? 4 : 1];
#pragma unroll
  for (int i = 0; i < (TMA ? 4 : 1); ++i) {
    k_at[i] = TMA ? k_row * 128 + (((2 * i + k_half) ^ (k_row & 7)) << 4) : k_row * PITCH + k_half * 16;
    v_at[i] = TMA ? v_row * 128 + (((2 * i + v_half) ^ (v_row & 7)) << 4) : v_row * PITCH + v_half * 16;
  }
  auto k_frag = [&](int i) -> uint32_t { return TMA ? (i >> 2) * 2048 + k_at[i & (TMA ? 3 : 0)] : k_at[0] + i * 32; };
  auto v_frag = [&](int i) -> uint32_t { return TMA ? (i >> 2) * 2048 + v_at[i & (TMA ? 3 : 0)] : v_at[0] + i * 32; };
  uint32_t phases = 0;
  bool lost = false;  // TMA: a copy of this warp's did not come; it loads no more, and its sums are NaN
  for (int u = blockIdx.x * per; u < u_end;) {
    const Segment g = find_segment(a, prefix, TT, kCost, hh_n, per, u, u_end);
    u = g.next;
    if (g.j1 <= g.j0) continue;
    const int h = g.hh / hg_n, head0 = (g.hh - h * hg_n) * GP, nh = min(GP, a.group - head0);
    const T* kb = static_cast<const T*>(a.c.k) + a.layer * a.c.layer + h * a.c.head;
    const T* vb = static_cast<const T*>(a.c.v) + a.layer * a.c.layer + h * a.c.head;
    const int32_t* table = a.c.tables + (int64_t)g.s * a.c.width;

    // cp.async: lane r (and r + 16) looks up slot r of a tile; TMA: lane b that
    // of box row b (those past either end fetch page 0, to be masked)
    auto page_of = [&](int j) -> int {
      if (TMA) {
        const int t = g.t0 + j * TT + lane * a.box;
        return j < g.j1 && lane * a.box < TT && t < g.n && t + a.box > g.lo ? table[t / a.c.page_tokens] : 0;
      }
      const int t = g.t0 + j * TT + (lane & 15);
      return j < g.j1 && t >= g.lo && t < g.n ? table[t / a.c.page_tokens] : INT32_MIN;
    };
    auto issue = [&](int j, int stage, int page) {
      const uint32_t to = stages + stage * 2 * TILE;
      if constexpr (TMA) {
        if (j >= g.j1 || lost) return;
        if (page < 0 || page >= a.c.n_pages) {
          a.c.status[kBadInput] = 1;
          page = 0;
        }
        const int page1 = __shfl_sync(~0u, page, 1);
        if (lane != 0) return;
        const int t = g.t0 + j * TT;
        mbar_expect_tx(bar + 8 * stage, 2 * TILE);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half * a.box >= TT) break;
          const int tok = (t + half * a.box) % a.c.page_tokens, pg = half ? page1 : page;
#pragma unroll
          for (int b = 0; b < DP / 64; ++b) {
            tma_load(to + b * 2048 + half * 1024, &k_map, b * 64, tok, h, pg, a.layer, bar + 8 * stage);
            tma_load(to + TILE + b * 2048 + half * 1024, &v_map, b * 64, tok, h, pg, a.layer, bar + 8 * stage);
          }
        }
      } else {
        if (j < g.j1) {
          const int t = g.t0 + j * TT + (lane & 15);
          int64_t off = -1;
          if (page >= 0 && page < a.c.n_pages)
            off = page * a.c.page + (int64_t)(t % a.c.page_tokens) * a.c.token;
          else if (page != INT32_MIN)
            a.c.status[kBadInput] = 1;
#pragma unroll
          for (int x = 0; x < TT * CH / 32; ++x) {
            const int e = x * 32 + lane, r = e / CH, c = e - r * CH;
            const int64_t o = __shfl_sync(~0u, off, r);
            const bool read = o >= 0 && c * 8 < a.c.d;
            const int64_t from = read ? o + c * 8 : 0;
            cp_async16_or_zero(to + r * PITCH + c * 16, kb + from, read);
            cp_async16_or_zero(to + TILE + r * PITCH + c * 16, vb + from, read);
          }
        }
        cp_commit();
      }
    };

    uint32_t qf[DP / 16][2];
    {
      const T* q = static_cast<const T*>(a.q) + (((int64_t)g.s * a.c.hkv + h) * a.group + head0 + gr) * a.c.d;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const int x = i * 16 + b * 8 + tg * 2;
          qf[i][b] = gr < nh && x < a.c.d ? *reinterpret_cast<const uint32_t*>(q + x) : 0u;
        }
    }
    float m0 = kNegInf, m1 = kNegInf, l0 = 0.f, l1 = 0.f, o[DP / 16][4];
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) o[i][x] = 0.f;

    const int first = g.j0 + warp;
    int page = page_of(first);
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
      const int now = page;
      page = page_of(first + (i + 1) * W);
      issue(first + i * W, i, now);
    }
    int stage = 0, fill = ST - 1;
    for (int j = first; j < g.j1 && !lost; j += W) {
      const uint32_t kt = stages + stage * 2 * TILE, vt = kt + TILE;
      if constexpr (TMA) {
        __syncwarp();  // the stage to fill has been read
        issue(j + (ST - 1) * W, fill, page);
        if (!__all_sync(~0u, mbar_wait(bar + 8 * stage, phases >> stage & 1))) {
          a.c.status[kTimedOut] = 1;
          lost = true;
          for (int i = 1, at = stage; i < ST; ++i) {  // the others in flight, as long again each
            at = at + 1 == ST ? 0 : at + 1;
            if (j + i * W < g.j1) mbar_wait(bar + 8 * at, phases >> at & 1);
          }
          break;
        }
        phases ^= 1u << stage;
        const int t = g.t0 + j * TT;
        if (t < g.lo || t + TT > g.n) {  // rows outside: zeros in place of what memory held
          for (int e = lane; e < TT * CH; e += 32) {
            const int r = e % TT, c = e / TT;
            uint4* v = reinterpret_cast<uint4*>(smem + (vt - base) + (c >> 3) * 2048 + r * 128 + (c & 7) * 16);
            if (t + r < g.lo || t + r >= g.n) *v = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();
          __syncwarp();
        }
      } else {
        cp_wait<ST - 2>();
        __syncwarp();
        issue(j + (ST - 1) * W, fill, page);
      }
      page = page_of(j + ST * W);
      fill = stage;
      stage = stage + 1 == ST ? 0 : stage + 1;

      float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) {
        uint32_t f[4];
        ldsm_x4(kt + k_frag(i), f);
        mma_16(i & 1 ? sb : sa, f, qf[i][0], qf[i][1], T());
      }
      float s[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) s[x] = (sa[x] + sb[x]) * a.scale_log2;
      const int t = g.t0 + j * TT + gr;
      if (t < g.lo || t >= g.n) s[0] = s[1] = kNegInf;
      if (t + 8 < g.lo || t + 8 >= g.n) s[2] = s[3] = kNegInf;
      if (a.scores) {
        float* to = a.scores + (((int64_t)g.s * a.c.hkv + h) * a.score_tokens + t) * a.group + head0 + 2 * tg;
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (t + (x >> 1) * 8 >= g.lo && t + (x >> 1) * 8 < g.n && 2 * tg + (x & 1) < nh)
            to[(x >> 1) * 8 * a.group + (x & 1)] = s[x];
      }
      if (__any_sync(~0u, s[0] > m0 || s[2] > m0 || s[1] > m1 || s[3] > m1)) {
        float t0 = fmaxf(m0, fmaxf(s[0], s[2])), t1 = fmaxf(m1, fmaxf(s[1], s[3]));
#pragma unroll
        for (int b = 4; b < 32; b <<= 1) {
          t0 = fmaxf(t0, __shfl_xor_sync(~0u, t0, b));
          t1 = fmaxf(t1, __shfl_xor_sync(~0u, t1, b));
        }
        const float f0 = ex2(m0 - (t0 == kNegInf ? 0.f : t0)), f1 = ex2(m1 - (t1 == kNegInf ? 0.f : t1));
        m0 = t0;
        m1 = t1;
        l0 *= f0;
        l1 *= f1;
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) {
          o[i][0] *= f0;
          o[i][1] *= f1;
          o[i][2] *= f0;
          o[i][3] *= f1;
        }
      }
      const float g0 = m0 == kNegInf ? 0.f : m0, g1 = m1 == kNegInf ? 0.f : m1;
      const float p0 = ex2(s[0] - g0), p1 = ex2(s[1] - g1), p2 = ex2(s[2] - g0), p3 = ex2(s[3] - g1);
      l0 += p0 + p2;
      l1 += p1 + p3;
      uint32_t w0[kParts<T>], w1[kParts<T>];
      split_16(p0 * kScale<T>, p1 * kScale<T>, w0, T());
      split_16(p2 * kScale<T>, p3 * kScale<T>, w1, T());
#pragma unroll
      for (int x = 0; x < kParts<T>; ++x) {
        w0[x] = transpose_8x8(w0[x]);
        w1[x] = transpose_8x8(w1[x]);
      }
#pragma unroll
      for (int i = 0; i < DP / 16; i += 4) {
        uint32_t f[4][4];
        float sum[4][4] = {};
#pragma unroll
        for (int y = 0; y < 4; ++y) ldsm_x4_t(vt + v_frag(i + y), f[y]);
#pragma unroll
        for (int x = kParts<T> - 1; x >= 0; --x)
#pragma unroll
          for (int y = 0; y < 4; ++y) mma_16(sum[y], f[y], w0[x], w1[x], T());
#pragma unroll
        for (int y = 0; y < 4; ++y)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[i + y][x] += sum[y][x];
      }
    }
    if constexpr (!TMA) cp_wait<0>();
    if (TMA && lost) l0 = l1 = NAN;
#pragma unroll
    for (int b = 4; b < 32; b <<= 1) {
      l0 += __shfl_xor_sync(~0u, l0, b);
      l1 += __shfl_xor_sync(~0u, l1, b);
    }
    __syncthreads();
    if (gr == 0) {
      om[warp * GP + 2 * tg] = m0;
      om[warp * GP + 2 * tg + 1] = m1;
      ol[warp * GP + 2 * tg] = l0;
      ol[warp * GP + 2 * tg + 1] = l1;
    }
#pragma unroll
    for (int i = 0; i < DP / 16; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x)
        oo[(warp * GP + 2 * tg + (x & 1)) * DP + i * 16 + gr + (x >> 1) * 8] = o[i][x] * (1.f / kScale<T>);
    finish_segment<W * 32, GP, DP>(a, g, hg_n, om, ol, oo);
    if (TMA && u < u_end) {  // the sums were written where the next loads go
      fence_proxy_async();
      __syncthreads();
    }
  }
}


// Blocks for the call: as many as run at once, fewer where even the table's
// full width holds less than min_tiles places of the list for each.
int attn_grid(const PagedAttnArgs& a, int gp, int tile, int cost, int most) {
  const int64_t cap = (int64_t)a.c.width * a.c.page_tokens;
  const int64_t seen = a.window > 0 ? std::min<int64_t>(cap, a.window) : cap;
  const int64_t items = (int64_t)a.n_seqs * a.c.hkv * ((a.group + gp - 1) / gp);
  // a window may begin inside a tile, and so reach one more
  const int64_t tiles = items * ((seen + tile - 1) / tile + (a.window > 0 ? 1 : 0) + cost);
  LC_REQUIRE(tiles < (1ll << 31) - (1 << 20), LC_ERR_INVALID, "more slots than one call can split");
  most = std::min(most, kPagedMaxBlocks);
  return (int)std::max<int64_t>(1, std::min<int64_t>(most, (tiles + a.min_tiles - 1) / a.min_tiles));
}

template <typename T, int DP, int GP, int ST, bool VEC>
void launch_fma(PagedAttnArgs& a, int device, int sms, cudaStream_t s) {
  constexpr int LPT = ST > 1 ? DP / 32 : DP / 64, TT = 32 / LPT, PITCH = DP + 4 * LPT, kWarps = ST > 1 ? 11 : 4;
  constexpr size_t fixed = (size_t)(kWarps * ST * 2 * TT * PITCH + GP * DP + kWarps * TT * GP + 2 * kWarps * GP) * 4;
  static_assert(fixed + (kPagedMaxSeqs + 1) * 4 <= 226 * 1024, "fits a block");
  auto kernel = k_paged_attn<T, DP, GP, kWarps, ST, VEC>;
  static SmemOptIn opt;
  opt(kernel, fixed + (kPagedMaxSeqs + 1) * 4, device);
  a.min_tiles = kWarps;
  const int grid = attn_grid(a, GP, TT, ST > 1 ? 2 * kFmaCost : kFmaCost, ST > 1 ? sms : 2 * sms);
  launch_pdl(kernel, dim3(grid), dim3(kWarps * 32), fixed + (size_t)(a.n_seqs + 1) * 4, s, a);
}

// Rows of 16-byte units: the pipeline for f32, for as many heads at a time as
// the group has (up to 8), and 16-byte loads for 16-bit pools whose queries are
// of another type. Anything else: the plain loads.
template <typename T, int DP>
void launch_fma(PagedAttnArgs& a, bool vec, int device, int sms, cudaStream_t s) {
  if constexpr (sizeof(T) == 4) {
    if (vec && a.group <= 4) return launch_fma<T, DP, 4, 2, false>(a, device, sms, s);
    if (vec) return launch_fma<T, DP, 8, 2, false>(a, device, sms, s);
  } else {
    if (vec) return launch_fma<T, DP, 4, 1, true>(a, device, sms, s);
  }
  launch_fma<T, DP, 4, 1, false>(a, device, sms, s);
}

template <typename T>
void launch_fma(PagedAttnArgs& a, bool vec, int device, int sms, cudaStream_t s) {
  if (a.c.d <= 64)
    launch_fma<T, 64>(a, vec, device, sms, s);
  else if (a.c.d <= 128)
    launch_fma<T, 128>(a, vec, device, sms, s);
  else
    launch_fma<T, 256>(a, vec, device, sms, s);
}

// acc_out[s, h, t] = decay acc_in + sum_g exp2(score_gt - m_g) / l_g. A block
// does 1024 slots of a row, four a thread, so that a thread has all its loads
// in flight at once; 4 (group + 2) bytes a slot, the scores still in L2. 24
// sequences of 1000 to 6000 slots, 8 kv heads of 4 query heads: 7 us after the
// attention's 66, of which its blocks' start and first loads are hidden.
template <bool VEC>
__global__ void __launch_bounds__(256) k_paged_weights(const PagedWeightArgs a) {
  extern __shared__ float st[];  // [group][2]
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, s = row / a.hkv, tid = threadIdx.x;
  const int n = min(max(__ldcg(a.lens + s), 0), a.cap), lo = first_slot(n, a.window);
  const int t0 = chunk * 1024 + tid;
  if (chunk * 1024 >= n) {
    if (chunk == 0) pdl_wait();  // this kernel must not end before the attention, whatever the lengths
    return;
  }
  const float* acc_in = a.acc_in + row * a.acc_stride;
  float acc[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (t0 + i * 256 < n) acc[i] = __ldcg(acc_in + t0 + i * 256);
  // The attention has waited for what came before it when it lets this kernel
  // in, so lengths and acc_in (from L2) are final; what follows is its own.
  pdl_wait();
  for (int i = tid; i < 2 * a.group; i += 256) st[i] = a.stats[2ll * row * a.group + i];
  const float* sc = a.scores + (int64_t)row * a.score_tokens * a.group;
  if (VEC) {
    for (int g = 0; g < a.group; g += 4) {
      float4 x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + i * 256;
        if (t >= lo && t < n) x[i] = *reinterpret_cast<const float4*>(sc + (int64_t)t * a.group + g);
      }
      if (g == 0) __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float* e = st + 2 * g;
        sum[i] += ex2(x[i].x - e[0]) * e[1] + ex2(x[i].y - e[2]) * e[3] + ex2(x[i].z - e[4]) * e[5] +
                  ex2(x[i].w - e[6]) * e[7];
      }
    }
  } else {
    __syncthreads();
#pragma unroll 2
    for (int g = 0; g < a.group; ++g) {
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = t0 + i * 256;
        if (t >= lo && t < n) x[i] = sc[(int64_t)t * a.group + g];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] += ex2(x[i] - st[2 * g]) * st[2 * g + 1];
    }
  }
  float* out = a.acc_out + row * a.acc_stride;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = t0 + i * 256;
    if (t < n) out[t] = fmaf(a.decay, acc[i], t >= lo ? sum[i] : 0.f);
  }
}

__device__ __forceinline__ void from_f32(float x, float& y) { y = x; }
__device__ __forceinline__ void from_f32(float x, __nv_bfloat16& y) { y = __float2bfloat16_rn(x); }
__device__ __forceinline__ void from_f32(float x, __half& y) { y = __float2half_rn(x); }

// New tokens' K and V rows into their pages, converted. A warp takes four
// (token, head) rows at a time, V elements of K or V a lane: V fills 16 bytes
// of the pool where rows are whole 16-byte units. Bound by the bytes of both:
// 32 x 2048 tokens of 8 heads of 128 bf16 take 108 us, 5.0 TB/s read and
// written; value by value (head dimension 100) 194 us, 2.2 TB/s.
constexpr int kAppendRows = 4;
template <typename TI, typename TO, int V>
__global__ void __launch_bounds__(256) k_paged_append(const PagedAppendArgs a) {
  struct alignas(V * sizeof(TI) > 16 ? 16 : V * sizeof(TI)) In {
    TI x[V];
  };
  struct alignas(V * sizeof(TO)) Out {
    TO x[V];
  };
  pdl_wait();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31, units = a.c.d / V;
  const int64_t rows = (int64_t)a.n_seqs * a.c.hkv * a.n_tokens, head0 = a.layer * a.c.layer;
  const int64_t step = gridDim.x * 8ll * kAppendRows;
  for (int64_t r0 = (blockIdx.x * 8ll + (threadIdx.x >> 5)) * kAppendRows; r0 < rows; r0 += step) {
    int64_t to = -1;
    if (lane < kAppendRows && r0 + lane < rows) {
      const int64_t r = r0 + lane, sh = r / a.n_tokens;
      const int tok = (int)(r - sh * a.n_tokens), s = (int)(sh / a.c.hkv), h = (int)(sh - (int64_t)s * a.c.hkv);
      const int64_t t = (int64_t)a.c.lens[s] + tok;
      if (t < 0 || t >= (int64_t)a.c.width * a.c.page_tokens) {
        a.c.status[kBadInput] = 1;
      } else {
        to = row_offset(a.c, s, (int)t);
        if (to >= 0) {
          to += head0 + h * a.c.head;
          if (a.pos) a.pos[sh * a.pos_stride + t] = a.pos0[s] + tok;
        }
      }
    }
    for (int x = lane; x < 2 * units + lane; x += 32) {  // the same count for all lanes: they shuffle
      const bool value = x >= units;
      const int64_t e = (int64_t)(value ? x - units : x) * V;
      const TI* from = static_cast<const TI*>(value ? a.values : a.keys) + r0 * a.c.d + e;
      TO* base = static_cast<TO*>(value ? a.c.v : a.c.k) + e;
      In in[kAppendRows];
      int64_t at[kAppendRows];
#pragma unroll
      for (int i = 0; i < kAppendRows; ++i) {
        at[i] = __shfl_sync(~0u, to, i);
        if (at[i] >= 0 && x < 2 * units) in[i] = *reinterpret_cast<const In*>(from + (int64_t)i * a.c.d);
      }
#pragma unroll
      for (int i = 0; i < kAppendRows; ++i) {
        if (at[i] < 0 || x >= 2 * units) continue;
        Out out;
#pragma unroll
        for (int y = 0; y < V; ++y) from_f32(to_f32(in[i].x[y]), out.x[y]);
        *reinterpret_cast<Out*>(base + at[i]) = out;
      }
    }
  }
}

template <typename T, int DP, int W, int ST, bool TMA, int PER_SM = 1>
void launch_mma(PagedAttnArgs& a, const PagedMaps& maps, int device, int sms, cudaStream_t s) {
  auto kernel = k_paged_attn_mma<T, DP, W, ST, TMA, PER_SM>;
  constexpr size_t fixed = (size_t)W * ST * (2 * 16 * (TMA ? DP * 2 : DP * 2 + 16) + 8) + 2 * W * 8 * 4;
  static_assert(PER_SM * (fixed + (kPagedMaxSeqs + 1) * 4 + 2048) <= 228 * 1024, "the blocks fit an SM");
  static SmemOptIn opt;
  opt(kernel, fixed + (kPagedMaxSeqs + 1) * 4, device);
  a.min_tiles = W;
  a.box = maps.box;
  const int grid = attn_grid(a, 8, 16, kMmaCost, PER_SM * sms);
  launch_pdl(kernel, dim3(grid), dim3(W * 32), fixed + (size_t)(a.n_seqs + 1) * 4, s, a, maps.k, maps.v);
}

template <typename T>
void launch_mma(PagedAttnArgs& a, const PagedMaps& maps, int device, int sms, cudaStream_t s) {
  // More short items than SMs: two blocks an SM of half the warps each, whose
  // items' beginnings and ends overlap (64 sequences of 1 to 64 slots: 12 us
  // against 18.5; one 131072-slot sequence 96 against 94).
  const int64_t cap = (int64_t)a.c.width * a.c.page_tokens;
  const int64_t seen = a.window > 0 ? std::min<int64_t>(cap, a.window) : cap;
  const bool halves = seen <= 256 && (int64_t)a.n_seqs * a.c.hkv > sms;
  if (maps.box && halves) {
    if (a.c.d <= 64)
      launch_mma<T, 64, 4, 5, true, 2>(a, maps, device, sms, s);
    else if (a.c.d <= 128)
      launch_mma<T, 128, 4, 3, true, 2>(a, maps, device, sms, s);
    else
      launch_mma<T, 256, 2, 3, true, 2>(a, maps, device, sms, s);
  } else if (maps.box) {
    if (a.c.d <= 64)
      launch_mma<T, 64, 8, 6, true>(a, maps, device, sms, s);
    else if (a.c.d <= 128)
      launch_mma<T, 128, 8, 3, true>(a, maps, device, sms, s);
    else if (a.c.d <= 192)
      launch_mma<T, 192, 4, 4, true>(a, maps, device, sms, s);
    else
      launch_mma<T, 256, 4, 3, true>(a, maps, device, sms, s);
  } else if (a.c.d <= 64) {
    launch_mma<T, 64, 8, 5, false>(a, maps, device, sms, s);
  } else if (a.c.d <= 128) {
    launch_mma<T, 128, 8, 3, false>(a, maps, device, sms, s);
  } else {
    launch_mma<T, 256, 4, 3, false>(a, maps, device, sms, s);
  }
}

}  // namespace

int64_t paged_part_floats(int32_t sms) { return 2ll * (2 * sms) * 8 * (kPagedMaxDim + 2); }

// Tensor maps for the TMA loads: pages of whole boxes of 16 or 8 slots, rows of
// at least the 64 dimensions of a box; box 0 where the pool has no such shape.
PagedMaps make_paged_maps(const PagedView& c, int32_t dtype) {
  PagedMaps m{};
  if (dtype == LC_F32 || !vector_rows(c, 2) || c.page_tokens % 8 != 0 || c.d < 64) return m;
  static void* const fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    LC_CUDA(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found));
    LC_REQUIRE(found == cudaDriverEntryPointSuccess && f, LC_ERR_CUDA, "the driver has no cuTensorMapEncodeTiled");
    return f;
  }();
  const int box = c.page_tokens % 16 == 0 ? 16 : 8;
  const cuuint64_t dims[5] = {(cuuint64_t)c.d, (cuuint64_t)c.page_tokens, (cuuint64_t)c.hkv, (cuuint64_t)c.n_pages,
                              (cuuint64_t)c.n_layers};
  const int64_t strides[4] = {c.token, c.head, c.page, c.layer};
  cuuint64_t bytes[4];
  for (int i = 0; i < 4; ++i) {
    bytes[i] = 2 * (cuuint64_t)(dims[i + 1] == 1 ? (c.d + 7) / 8 * 8 : strides[i]);  // a lone row's stride is never used
    if (bytes[i] >= 1ull << 40) return m;
  }
  const cuuint32_t shape[5] = {64, (cuuint32_t)box, 1, 1, 1}, ones[5] = {1, 1, 1, 1, 1};
  const auto type = dtype == LC_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  auto encode = reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(fn);
  for (int i = 0; i < 2; ++i) {
    const CUresult r = encode(i ? &m.v : &m.k, type, 5, i ? c.v : c.k, dims, bytes, shape, ones,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return PagedMaps{};
  }
  m.box = box;
  return m;
}

void launch_paged_attn(PagedAttnArgs& a, const PagedMaps& maps, int32_t pool_dtype, int32_t device, int32_t sms,
                       cudaStream_t s) {
  const bool vec = vector_rows(a.c, pool_dtype == LC_F32 ? 4 : 2);
  const bool mma =
      pool_dtype != LC_F32 && a.q_dtype == pool_dtype && vec && (reinterpret_cast<uintptr_t>(a.q) & 3) == 0;
  if (mma && pool_dtype == LC_BF16)
    launch_mma<__nv_bfloat16>(a, maps, device, sms, s);
  else if (mma)
    launch_mma<__half>(a, maps, device, sms, s);
  else if (pool_dtype == LC_F32)
    launch_fma<float>(a, vec, device, sms, s);
  else if (pool_dtype == LC_BF16)
    launch_fma<__nv_bfloat16>(a, vec, device, sms, s);
  else
    launch_fma<__half>(a, vec, device, sms, s);
  LC_CUDA(cudaGetLastError());
}

void launch_paged_weights(PagedWeightArgs a, cudaStream_t s) {
  a.chunks = (a.cap + 1023) / 1024;
  const int64_t blocks = (int64_t)a.n_seqs * a.hkv * a.chunks;
  LC_REQUIRE(blocks < (1ll << 31), LC_ERR_INVALID, "more slots than one call can weigh");
  const bool vec = a.group % 4 == 0;  // a slot's scores are whole float4s (the workspace is 256-byte aligned)
  launch_pdl(vec ? k_paged_weights<true> : k_paged_weights<false>, dim3((unsigned)blocks), dim3(256),
             2 * a.group * 4, s, a);
}

template <typename TI, typename TO>
void launch_append(const PagedAppendArgs& a, int sms, cudaStream_t s) {
  constexpr int V = 16 / sizeof(TO);
  const int64_t rows = (int64_t)a.n_seqs * a.c.hkv * a.n_tokens, per = 8 * kAppendRows;
  const int grid = (int)std::min<int64_t>(8ll * sms, (rows + per - 1) / per);
  const uintptr_t in = reinterpret_cast<uintptr_t>(a.keys) | reinterpret_cast<uintptr_t>(a.values);
  if (vector_rows(a.c, sizeof(TO)) && in % std::min<size_t>(16, V * sizeof(TI)) == 0)
    launch_pdl(k_paged_append<TI, TO, V>, dim3(grid), dim3(256), 0, s, a);
  else
    launch_pdl(k_paged_append<TI, TO, 1>, dim3(grid), dim3(256), 0, s, a);
}

template <typename TO>
void launch_append(const PagedAppendArgs& a, int sms, cudaStream_t s) {
  if (a.dtype == LC_F32)
    launch_append<float, TO>(a, sms, s);
  else if (a.dtype == LC_BF16)
    launch_append<__nv_bfloat16, TO>(a, sms, s);
  else
    launch_append<__half, TO>(a, sms, s);
}

void launch_paged_append(const PagedAppendArgs& a, int32_t sms, cudaStream_t s) {
  if (a.pool_dtype == LC_F32)
    launch_append<float>(a, sms, s);
  else if (a.pool_dtype == LC_BF16)
    launch_append<__nv_bfloat16>(a, sms, s);
  else
    launch_append<__half>(a, sms, s);
}

}  // namespace lc
