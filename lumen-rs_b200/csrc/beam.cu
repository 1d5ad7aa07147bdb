// Beam search's selection (lc_beam_select).
//
//   z[b, v] = score_b + ((x_bv - max_v x_b) - log sum_v exp(x_bv - max_v x_b))
//
// and of all b, v of a group the n_out largest z, lower b * V + v first among
// equals. The bytes of the logits bound it: one pass reads each logit once,
// into registers, and takes from it both the softmax sums and the slice's
// n_out best.
//
// A block takes a part of a row (all of it where there are rows enough for the
// card) slice by slice through a ring of shared memory that one warp of its
// own fills with bulk copies: while the memory is busy a copy's issue alone
// takes some 900 cycles. Rows that begin off 16 bytes are put right as they
// are read from the ring, so that a thread's logits, and with them the order
// of the sums, do not depend on the row's address. A thread keeps a running
// maximum and sum of its own.
//
// The largest but n_out of the maxima of 64 (or 128) disjoint sets of the
// logits so far is a lower bound of the largest but n_out logit. It is taken
// after slices 1, 3, 8, 16 ... (only once: 51 us for 33 million logits; after
// 1, 2, 4, 8: 32; so: 31), and the logits that reach it are gathered, to be
// ranked by counting at the end. The last block of a group turns all parts'
// candidates into totals, cuts them by the same bound, ranks them and writes
// the answer. One launch; ranks are by value and index only, so the order of
// arrival changes nothing.
//
// Totals are rounded, so different logits of a row may have equal ones, of
// which the lower token goes first: next to its n_out best logits a part keeps
// the one after them. Only where that has the total of the answer's last place,
// the first such part is read again (see repair).
//
// 256 rows of 131072 bf16 logits take 32.8 us, 2.1 TB/s; 64 groups of 4 rows of
// 1000 f32 13.3; 4 rows of 50021 f32 14.0. So half is the chain of launch, first
// copy, bound, ranking, the counter's round trip and the merge, all of it
// latency; the other half runs at 0.65 of the pace that a copy of the card's
// memory has. Looking for a part to read again is 0.7 of these, reading one to
// its end is 45 us for all of 256 rows of 131072 f32 at once.
#include <algorithm>

#include "devutil.cuh"
#include "paged.h"

namespace lc {
namespace {

constexpr int kThreads = 512;  // that compute; one more warp fetches
constexpr int kWarps = kThreads / 32;
constexpr int kGran = 2;      // 16-byte granules of a slice for each thread
constexpr int kStages = 4;    // slices of the ring
constexpr int kStage = kGran * kThreads + 8;  // granules of a stage: a slice, and one more for rows off 16 bytes
constexpr int kBeamPerSm = 2;
constexpr int kList = kBeamMaxMerge;  // gathered candidates of a part
// More candidates than these are cut by a bound before they are ranked: 512 of
// 4 beams took 18.7 us uncut and 11.1 cut, 208 13.8 and 13.0; 128 15.5 and 16.4.
constexpr int kRankAll = 128;
constexpr float kNegInf = -INFINITY;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint32_t order_f32(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_to_f32(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// larger is better: value first, then the lower index
__device__ __forceinline__ uint64_t make_key(float x, uint32_t index) {
  return (uint64_t)order_f32(x) << 32 | (0xffffffffu - index);
}
__device__ __forceinline__ uint32_t key_index(uint64_t k) { return 0xffffffffu - (uint32_t)k; }
__device__ __forceinline__ float key_value(uint64_t k) { return order_to_f32((uint32_t)(k >> 32)); }

template <typename T>
__device__ __forceinline__ float elem(const uint4& r, int i);
template <>
__device__ __forceinline__ float elem<float>(const uint4& r, int i) {
  return __uint_as_float(i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w);
}
template <>
__device__ __forceinline__ float elem<__nv_bfloat16>(const uint4& r, int i) {
  const uint32_t w = (i >> 1) == 0 ? r.x : (i >> 1) == 1 ? r.y : (i >> 1) == 2 ? r.z : r.w;
  return __uint_as_float(i & 1 ? w & 0xffff0000u : w << 16);
}
template <>
__device__ __forceinline__ float elem<__half>(const uint4& r, int i) {
  const uint32_t w = (i >> 1) == 0 ? r.x : (i >> 1) == 1 ? r.y : (i >> 1) == 2 ? r.z : r.w;
  return __half2float(__ushort_as_half((unsigned short)(i & 1 ? w >> 16 : w & 0xffffu)));
}

// The 16 bytes that begin `off` bytes into (lo, hi).
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, int off) {
  uint32_t w0, w1, w2, w3, w4;
  switch (off >> 2) {
    case 0: w0 = lo.x, w1 = lo.y, w2 = lo.z, w3 = lo.w, w4 = hi.x; break;
    case 1: w0 = lo.y, w1 = lo.z, w2 = lo.w, w3 = hi.x, w4 = hi.y; break;
    case 2: w0 = lo.z, w1 = lo.w, w2 = hi.x, w3 = hi.y, w4 = hi.z; break;
    default: w0 = lo.w, w1 = hi.x, w2 = hi.y, w3 = hi.z, w4 = hi.w; break;
  }
  const int bits = (off & 3) * 8;
  return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                    __funnelshift_r(w3, w4, bits));
}

// The largest of a granule's values; NaN only where all are.
template <typename T>
__device__ __forceinline__ float granule_max(const uint4& r);
template <>
__device__ __forceinline__ float granule_max<float>(const uint4& r) {
  return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
}
template <typename T2>
__device__ __forceinline__ T2 max_2x4(const uint4& r) {
  const T2* h = reinterpret_cast<const T2*>(&r);
  return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
}
template <>
__device__ __forceinline__ float granule_max<__nv_bfloat16>(const uint4& r) {
  const float2 f = __bfloat1622float2(max_2x4<__nv_bfloat162>(r));
  return fmaxf(f.x, f.y);
}
template <>
__device__ __forceinline__ float granule_max<__half>(const uint4& r) {
  const float2 f = __half22float2(max_2x4<__half2>(r));
  return fmaxf(f.x, f.y);
}

// two f32 at a time
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t x;
  asm("mov.b64 %0, {%1, %2};" : "=l"(x) : "f"(lo), "f"(hi));
  return x;
}
__device__ __forceinline__ float2 unpack2(uint64_t x) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(x));
  return f;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t x;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(a), "l"(b));
  return x;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t x;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(x) : "l"(a), "l"(b));
  return x;
}

// a barrier of the computing threads
__device__ __forceinline__ void sync_threads() { asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory"); }

// of which x holds for so many
__device__ __forceinline__ int count_threads(bool x) {
  int n;
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.popc.aligned.u32 %0, 1, %2, p;\n}\n"
      : "=r"(n)
      : "r"((uint32_t)x), "n"(kThreads)
      : "memory");
  return n;
}

// The next larger value; not of NaN.
__device__ __forceinline__ float next_up(float x) {
  if (x == 0.f) return __uint_as_float(1u);
  const uint32_t u = __float_as_uint(x);
  return x > 0.f ? (x < INFINITY ? __uint_as_float(u + 1) : NAN) : __uint_as_float(u - 1);
}

// The next larger (or smaller) value of type T to x, itself one and finite.
template <typename T>
__device__ __forceinline__ float neighbour(float x, bool larger) {
  if constexpr (sizeof(T) == 4) {
    return larger ? next_up(x) : -next_up(-x);
  } else {
    const T t = T(x);
    unsigned short u = *reinterpret_cast<const unsigned short*>(&t);
    if ((u & 0x7fff) == 0)
      u = larger ? 1 : 0x8001;
    else
      u += larger == !(u & 0x8000) ? 1 : -1;
    return (float)*reinterpret_cast<const T*>(&u);
  }
}

struct BeamShared {
  uint64_t list[kBeamMaxMerge];  // a part's candidates, then the group's
  uint64_t few[kThreads], best[kBeamMaxOut + 1], warp_key[kWarps], key_sets[128], key_bound;
  __align__(16) float sets[128];
  float m[kWarps], l[kWarps], row_top[kBeamMaxBeams], row_log[kBeamMaxBeams], row_next[kBeamMaxBeams];
  float bound;
  int n, n_few, last, again;
};

__device__ __forceinline__ uint64_t block_max_key(uint64_t k, uint64_t* warp_key) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t x = __shfl_xor_sync(~0u, k, o);
    k = x > k ? x : k;
  }
  sync_threads();
  if ((threadIdx.x & 31) == 0) warp_key[threadIdx.x >> 5] = k;
  sync_threads();
  k = warp_key[0];
#pragma unroll
  for (int w = 1; w < kWarps; ++w) k = warp_key[w] > k ? warp_key[w] : k;
  return k;
}

// max and sum of (m, l) over a warp
__device__ __forceinline__ void warp_softmax(float& m, float& l) {
  float top = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  l *= ex2((m - (top == kNegInf ? 0.f : top)) * kLog2e);
#pragma unroll
  for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
  m = top;
}

// A lower bound of the keep-th largest of the values whose maximum over this
// thread's is x: the keep-th largest of the maxima of 64 or 128 sets of threads.
__device__ __forceinline__ float set_bound(BeamShared& sh, float x, int keep) {
  const int tid = threadIdx.x, size = keep <= 17 ? kThreads / 64 : kThreads / 128, n_sets = kThreads / size;
  for (int o = 1; o < size; o <<= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, o));
  const int set = tid / size, sub = tid & (size - 1), span = n_sets / size;
  if (sub == 0) sh.sets[set] = x;
  sync_threads();
  int r = 0;  // this thread counts over `span` of the sets
#pragma unroll 2
  for (int i = sub * span; i < (sub + 1) * span; i += 4) {
    const float4 y = *reinterpret_cast<const float4*>(sh.sets + i);
    r += y.x > x || (y.x == x && i < set);
    r += y.y > x || (y.y == x && i + 1 < set);
    r += y.z > x || (y.z == x && i + 2 < set);
    r += y.w > x || (y.w == x && i + 3 < set);
  }
  for (int o = 1; o < size; o <<= 1) r += __shfl_xor_sync(~0u, r, o);
  if (sub == 0 && r == keep - 1) sh.bound = x;
  sync_threads();
  return sh.bound;
}

// Of a slice's marked logits (bit r * e + i: value i of granule r) those that
// are not among the first `keep` of all threads' in the order of tokens.
__device__ __noinline__ uint32_t past_first(BeamShared& sh, uint32_t marked, int e, int keep) {
  static_assert(kGran == 2, "two counts in a word");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t low = marked & ((1u << e) - 1), high = marked >> e;
  const uint32_t own = __popc(low) | __popc(high) << 16;
  uint32_t inc = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t up = __shfl_up_sync(~0u, inc, o);
    if (lane >= o) inc += up;
  }
  if (lane == 31) sh.warp_key[warp] = inc;
  sync_threads();
  uint32_t before = inc - own, all = 0;
  for (int w = 0; w < kWarps; ++w) {
    const uint32_t x = (uint32_t)sh.warp_key[w];
    if (w < warp) before += x;
    all += x;
  }
  sync_threads();
  int at[2] = {(int)(before & 0xffff), (int)((all & 0xffff) + (before >> 16))};
  uint32_t past = 0;
  for (uint32_t rest = marked; rest; rest &= rest - 1) {
    const int bit = __ffs(rest) - 1;
    if (at[bit >= e]++ >= keep) past |= 1u << bit;
  }
  return past;
}

// The same of keys, which are all different; 0 where the sets with one are fewer.
__device__ __forceinline__ uint64_t set_bound_key(BeamShared& sh, uint64_t x, int keep) {
  const int tid = threadIdx.x, size = keep <= 17 ? kThreads / 64 : kThreads / 128, n_sets = kThreads / size;
  for (int o = 1; o < size; o <<= 1) {
    const uint64_t y = __shfl_xor_sync(~0u, x, o);
    x = y > x ? y : x;
  }
  const int set = tid / size, sub = tid & (size - 1), span = n_sets / size;
  if (sub == 0) sh.key_sets[set] = x;
  if (tid == 0) sh.key_bound = sh.n_few = 0;
  sync_threads();
  int r = 0;
#pragma unroll 4
  for (int i = sub * span; i < (sub + 1) * span; ++i) r += sh.key_sets[i] > x;
  for (int o = 1; o < size; o <<= 1) r += __shfl_xor_sync(~0u, r, o);
  if (sub == 0 && x && r == keep - 1) sh.key_bound = x;
  sync_threads();
  return sh.key_bound;
}

// emit(key, rank) for the `keep` largest of sh.list[0 .. n), all different, 0
// for none: cut by a bound where they are many, then P threads count the
// larger ones of an entry. The bound is of values, which takes half a
// microsecond less than one of keys; that one follows where too many values
// are equal. A merge's list is sorted by parts, so for the bound neighbours go
// to sets far from each other (37 * 429 = 1 mod 512): taken in order, the best
// of 64 rows fell into 8 sets, too many reached the bound, and 4 groups of 64
// beams to 64 took 580 us; they take 27.
template <typename F>
__device__ __forceinline__ void rank_list(BeamShared& sh, int n, int keep, F&& emit) {
  const uint64_t* list = sh.list;
  if (n > kRankAll) {
    auto best_of_mine = [&] {
      uint64_t top = 0;
      for (int c0 = 0; c0 < n; c0 += kThreads) {
        const int c = c0 + ((429 * threadIdx.x + c0 / 64) & (kThreads - 1));
        if (c < n && list[c] > top) top = list[c];
      }
      return top;
    };
    auto cut = [&](auto&& reaches) {
      for (int c = threadIdx.x; c < n; c += kThreads) {
        const uint64_t k = list[c];
        if (k && reaches(k)) {
          const int at = atomicAdd(&sh.n_few, 1);
          if (at < kThreads) sh.few[at] = k;
        }
      }
      sync_threads();
    };
    if (threadIdx.x == 0) sh.n_few = 0;
    const uint64_t top = best_of_mine();
    const float bound = set_bound(sh, top ? key_value(top) : kNegInf, keep);
    cut([&](uint64_t k) { return key_value(k) >= bound; });
    const int reached = sh.n_few;
    sync_threads();  // read by all before it is set anew
    if (reached > kThreads) {
      const uint64_t key_bound = set_bound_key(sh, best_of_mine(), keep);
      cut([&](uint64_t k) { return k >= key_bound; });
    }
    if (sh.n_few <= kThreads) {
      list = sh.few;
      n = sh.n_few;
    }
  }
  int p = 1;
  while (p < 32 && 2 * p * n <= kThreads) p *= 2;
  const int sub = threadIdx.x & (p - 1), step = kThreads / p;
  for (int c0 = 0; c0 < n; c0 += step) {
    const int c = c0 + threadIdx.x / p;
    const uint64_t key = c < n ? list[c] : 0;
    int r = 0;
#pragma unroll 4
    for (int o = sub; o < n; o += p) r += list[o] > key;
    for (int o = 1; o < p; o <<= 1) r += __shfl_xor_sync(~0u, r, o);
    if (sub == 0 && key && r < keep) emit(key, r);
  }
}

// The answer's places of total z, its lowest, where a part may have missed a
// token of that total. All that such a part listed have z or more, so that the
// first of them has enough for the places after those of earlier parts: its
// first tokens of total z, in order.
template <typename T>
__device__ __noinline__ void repair(const BeamArgs& a, BeamShared& sh, int64_t row0, int64_t slot0, int parts, float z) {
  constexpr int kLoads = 16;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) sh.again = INT32_MAX;
  sync_threads();
  for (int c = tid; c < a.n_beams * parts; c += kThreads) {
    const float next = __ldcg(a.slice_next + 2 * (slot0 + c)), least = __ldcg(a.slice_next + 2 * (slot0 + c) + 1);
    const int b = c / parts;
    auto total = [&](float x) { return a.scores[row0 + b] + ((x - sh.row_top[b]) - sh.row_log[b]); };
    // Logits equal to the least listed have higher tokens than it: none is missed
    // where no other value has their total.
    if (next > kNegInf && total(next) >= z &&
        (next < least || total(neighbour<T>(least, false)) >= z || total(neighbour<T>(least, true)) <= z))
      atomicMin(&sh.again, c);
  }
  sync_threads();
  if (sh.again == INT32_MAX) return;
  const int b = sh.again / parts;
  const int64_t i0 = (int64_t)(sh.again - b * parts) * a.per * a.slice;
  const int64_t i1 = min((int64_t)a.vocab, i0 + (int64_t)a.per * a.slice);
  const uint32_t base = (uint32_t)(b * (int64_t)a.vocab);
  const T* x0 = static_cast<const T*>(a.logits) + (row0 + b) * a.row_stride;
  const float score = a.scores[row0 + b], top = sh.row_top[b], log = sh.row_log[b];
  const uint64_t mine = tid < a.n_out ? sh.best[tid] : 0;
  int have = count_threads(mine && (key_value(mine) > z || key_index(mine) < base + (uint32_t)i0));
  for (int64_t i = i0; i < i1 && have < a.n_out; i += kLoads * kThreads) {
    T x[kLoads];
#pragma unroll
    for (int r = 0; r < kLoads; ++r)
      if (i + r * kThreads + tid < i1) x[r] = x0[i + r * kThreads + tid];
    uint32_t hits = 0;
#pragma unroll
    for (int r = 0; r < kLoads; ++r)
      if (i + r * kThreads + tid < i1 && score + (((float)x[r] - top) - log) == z) hits |= 1u << r;
    if (!count_threads(hits != 0)) continue;
    for (int r = 0; r < kLoads && have < a.n_out; ++r) {
      const uint32_t found = __ballot_sync(~0u, hits >> r & 1);
      if (lane == 0) sh.warp_key[warp] = __popc(found);
      sync_threads();
      int at = have + __popc(found & ((1u << lane) - 1));
      for (int w = 0; w < kWarps; ++w) {
        if (w < warp) at += (int)sh.warp_key[w];
        have += (int)sh.warp_key[w];
      }
      if ((hits >> r & 1) && at < a.n_out) sh.best[at] = make_key(z, base + (uint32_t)(i + r * kThreads + tid));
      sync_threads();
    }
  }
  sync_threads();
}

// Ends a part, elements [i0, i1) of a row: its maximum, sum and best
// candidates; then, in the last block of the group, the answer.
template <typename T>
__device__ __noinline__ void finish(const BeamArgs& a, BeamShared& sh, int row, int64_t i0, int64_t i1, bool done,
                                    bool dead, float m, float l, float tau) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int group = row / a.n_beams, parts = gridDim.x;
  const int64_t slot = (int64_t)row * parts + blockIdx.x;
  uint64_t* keys = a.slice_key + slot * a.n_out;
  if (dead) {
    // a finished row's only total is its score: of one logit, 0, of a sum of 1
    const bool one = done && blockIdx.x == 0;
    for (int c = tid; c < a.n_out; c += kThreads) keys[c] = one && c == 0 ? make_key(0.f, a.pad) : 0;
    if (tid == 0) {
      a.slice_stats[2 * slot] = one ? 0.f : kNegInf;
      a.slice_stats[2 * slot + 1] = one ? 1.f : 0.f;
      a.slice_next[2 * slot] = kNegInf;
    }
  } else {
    warp_softmax(m, l);
    if (lane == 0) {
      sh.m[warp] = m;
      sh.l[warp] = l;
    }
    for (int c = tid; c <= a.n_out; c += kThreads) sh.best[c] = 0;
    sync_threads();
    if (warp == kWarps - 1) {
      m = lane < kWarps ? sh.m[lane] : kNegInf;
      l = lane < kWarps ? sh.l[lane] : 0.f;
      warp_softmax(m, l);
      if (lane == 0) {
        a.slice_stats[2 * slot] = m;
        a.slice_stats[2 * slot + 1] = l;
      }
    }
    const int found = sh.n;
    if (found <= kList) {
      rank_list(sh, found, a.n_out + 1, [&](uint64_t k, int r) { sh.best[r] = k; });
    } else {
      // many logits reach the bound: one best after the other, read again
      const T* x0 = static_cast<const T*>(a.logits) + row * a.row_stride;
      uint64_t before = ~0ull;
      for (int o = 0; o <= a.n_out; ++o) {
        uint64_t best = 0;
#pragma unroll 4
        for (int64_t i = i0 + tid; i < i1; i += kThreads) {
          const float x = (float)x0[i];
          const uint64_t k = make_key(x, (uint32_t)i);
          if (x >= tau && k < before && k > best) best = k;
        }
        before = block_max_key(best, sh.warp_key);
        if (tid == 0) sh.best[o] = before;
      }
    }
    sync_threads();
    for (int c = tid; c < a.n_out; c += kThreads) keys[c] = sh.best[c];
    if (tid == 0) {
      a.slice_next[2 * slot] = sh.best[a.n_out] ? key_value(sh.best[a.n_out]) : kNegInf;
      a.slice_next[2 * slot + 1] = sh.best[a.n_out] ? key_value(sh.best[a.n_out - 1]) : kNegInf;
    }
  }

  // the last block of the group goes on
  const int64_t row0 = (int64_t)group * a.n_beams, slot0 = row0 * parts, out0 = (int64_t)group * a.n_out;
  sync_threads();
  if (tid == 0) {
    const int of = a.n_beams * parts;
    __threadfence();  // the block's writes, which the barrier put before this thread
    sh.last = atomicAdd(a.counters + group, 1) == of - 1;
    if (sh.last) {
      __threadfence();
      a.counters[group] = 0;
    }
  }
  sync_threads();
  if (!sh.last) return;
  const int per_row = parts * a.n_out, all = a.n_beams * per_row;
  for (int c = tid; c < all; c += kThreads) sh.list[c] = __ldcg(a.slice_key + slot0 * a.n_out + c);
  for (int c = tid; c < a.n_out; c += kThreads) sh.best[c] = 0;
  for (int b = warp; b < a.n_beams; b += kWarps) {  // the rows' maxima and sums
    m = kNegInf;
    l = 0.f;
    const float score = a.scores[row0 + b];
    float next = kNegInf;
    for (int i = lane; i < parts; i += 32) {
      const int64_t part = slot0 + (int64_t)b * parts + i;
      const float* st = a.slice_stats + 2 * part;
      const float mi = __ldcg(st), li = __ldcg(st + 1);
      next = fmaxf(next, __ldcg(a.slice_next + 2 * part));
      const float mn = fmaxf(m, mi), mg = mn == kNegInf ? 0.f : mn;
      l = l * ex2((m - mg) * kLog2e) + li * ex2((mi - mg) * kLog2e);
      m = mn;
    }
    warp_softmax(m, l);
#pragma unroll
    for (int o = 16; o; o >>= 1) next = fmaxf(next, __shfl_xor_sync(~0u, next, o));
    if (lane == 0) {
      const float log = logf(l);
      sh.row_top[b] = m;
      sh.row_log[b] = log;
      sh.row_next[b] = next > kNegInf ? score + ((next - m) - log) : kNegInf;
    }
  }
  sync_threads();
  for (int c = tid; c < all; c += kThreads) {
    uint64_t k = sh.list[c];
    if (k) {
      const int b = c / per_row;
      const float z = a.scores[row0 + b] + ((key_value(k) - sh.row_top[b]) - sh.row_log[b]);
      k = z > kNegInf ? make_key(z, (uint32_t)(b * (int64_t)a.vocab + key_index(k))) : 0;
    }
    sh.list[c] = k;
  }
  sync_threads();
  rank_list(sh, all, a.n_out, [&](uint64_t k, int r) { sh.best[r] = k; });
  sync_threads();
  if (sh.best[a.n_out - 1]) {  // else every candidate has a place
    const float z = key_value(sh.best[a.n_out - 1]);
    bool tied = false;
    for (int b = lane; b < a.n_beams; b += 32) tied |= sh.row_next[b] >= z;
    if (__any_sync(~0u, tied)) repair<T>(a, sh, row0, slot0, parts, z);
  }
  for (int r = tid; r < a.n_out; r += kThreads) {
    const uint64_t k = sh.best[r];
    const uint32_t index = key_index(k);
    // a place with no candidate keeps a beam
    const int p = k ? (int)(index / (uint32_t)a.vocab) : r % a.n_beams;
    const int tok = k ? (int)(index - (uint32_t)p * (uint32_t)a.vocab) : a.pad;
    a.scores_out[out0 + r] = k ? key_value(k) : kNegInf;
    a.parents[out0 + r] = p;
    a.tokens[out0 + r] = tok;
    a.finished_out[out0 + r] = !k || tok == a.eos || (a.finished && a.finished[row0 + p]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads + 32, kBeamPerSm) k_beam_select(const __grid_constant__ BeamArgs a) {
  constexpr int E = 16 / sizeof(T);
  extern __shared__ __align__(16) uint4 ring[];  // [kStages][kStage]
  __shared__ BeamShared sh;
  __shared__ uint64_t bars[2 * kStages];  // full, then empty
  const int tid = threadIdx.x, row = blockIdx.y;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring), full = (uint32_t)__cvta_generic_to_shared(bars);
  const uint32_t empty = full + 8 * kStages;
  const int slice0 = blockIdx.x * a.per, slices = min(a.slices, slice0 + a.per) - slice0;
  // the row's first element sits at base[mis]: base is 16-byte aligned
  const T* x0 = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int mis = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T)), off = mis * (int)sizeof(T);
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, kWarps);
    }
    mbar_init_fence();
    sh.n = 0;
  }
  __syncthreads();
  pdl_wait();
  pdl_launch_dependents();
  const float score = a.scores[row];
  const uint8_t done = a.finished ? a.finished[row] : 0;

  if (tid >= kThreads) {
    // The fetching warp: a slice's whole granules by one bulk copy; those at the
    // row's ends by hand, -inf where there is no logit.
    const int lane = tid & 31;
    const T* base = x0 - mis;
    const int64_t i_end = mis + (int64_t)a.vocab;
    int it = 0;
    for (; it < slices; ++it) {
      const int stage = it % kStages;
      // the ring's first slices are asked for before it is known whether they matter
      if (it >= kStages && (done || !(score > kNegInf) || !mbar_wait(empty + 8 * stage, (it / kStages - 1) & 1))) break;
      const int64_t at0 = (int64_t)(slice0 + it) * a.slice;
      const int n = kGran * kThreads + (mis ? 1 : 0);
      const int lo = mis && slice0 + it == 0 ? 1 : 0, hi = (int)min((int64_t)n, (i_end - at0) / E);
      if (lo > 0 || hi < n) {
        for (int v = lane; v < n; v += 32) {
          if (v >= lo && v < hi) {
            v += (hi - v) / 32 * 32;  // the copy's
            if (v < hi) continue;
          }
          if (v >= n) break;
          const int64_t at = at0 + v * E;
          alignas(16) T part[E];
#pragma unroll
          for (int i = 0; i < E; ++i) part[i] = T(kNegInf);
          if (at < i_end)
            for (int i = 0; i < E; ++i)
              if (at + i >= mis && at + i < i_end) part[i] = base[at + i];
          ring[stage * kStage + v] = *reinterpret_cast<uint4*>(part);
        }
        fence_proxy_async();  // a later slice's bulk copy may write there
        __syncwarp();
      }
      if (lane == 0) {
        const int bytes = hi > lo ? (hi - lo) * 16 : 0;
        mbar_expect_tx(full + 8 * stage, bytes);
        if (bytes) bulk_g2s(ring_at + (stage * kStage + lo) * 16, base + at0 + lo * E, bytes, full + 8 * stage);
      }
      __syncwarp();
    }
    // the copies in flight, which no one may be waiting for
    for (int i = max(0, it - kStages); i < it; ++i) mbar_wait(full + 8 * (i % kStages), i / kStages & 1);
    return;
  }

  // a finished row's logits, or those of a beam that is out, do not matter
  const bool dead = done || !(score > kNegInf);
  float m = kNegInf, tau = kNegInf, least = next_up(kNegInf);  // least: of the logits to gather
  uint64_t l = pack2(0.f, 0.f);  // the sum in two halves
  bool lost = false;
  const uint64_t log2e = pack2(kLog2e, kLog2e);
#pragma unroll 1
  for (int it = 0; it < slices && !dead; ++it) {
    const int stage = it % kStages;
    if (!lost && !mbar_wait(full + 8 * stage, it / kStages & 1)) {  // a copy that did not come: no candidates
      lost = true;
      a.status[kTimedOut] = 1;
    }
    const uint4* x = ring + stage * kStage + tid;
    uint4 g[kGran];
#pragma unroll
    for (int r = 0; r < kGran; ++r) g[r] = x[r * kThreads];
    if (off) {
#pragma unroll
      for (int r = 0; r < kGran; ++r) g[r] = shifted(g[r], x[r * kThreads + 1], off);
    }
    float top = kNegInf;
#pragma unroll
    for (int r = 0; r < kGran; ++r) top = fmaxf(top, granule_max<T>(g[r]));
    if (top > m) {
      const float f = ex2((m - top) * kLog2e);
      l = mul2(l, pack2(f, f));
      m = top;
    }
    const float mg = m == kNegInf ? 0.f : m;
    const uint64_t less = pack2(-mg, -mg);
#pragma unroll
    for (int r = 0; r < kGran; ++r) {
      uint64_t sum = 0;  // two zeros; products by twos: 31.1 us against 31.7 one by one
#pragma unroll
      for (int i = 0; i < E; i += 2) {
        const float2 y = unpack2(mul2(add2(pack2(elem<T>(g[r], i), elem<T>(g[r], i + 1)), less), log2e));
        sum = add2(sum, pack2(ex2(y.x), ex2(y.y)));
      }
      l = add2(l, sum);
    }
    bool rose = false;
    if (it == 0 || it == 2 || (it & 7) == 7 || tau == kNegInf) {
      const float before = tau;
      tau = set_bound(sh, m, a.n_out + 1);
      rose = tau > before;
      if (rose) least = tau;
    }
    uint32_t hits = 0;
    if (top >= least) {
#pragma unroll
      for (int r = 0; r < kGran; ++r)
#pragma unroll
        for (int i = 0; i < E; ++i) hits |= (elem<T>(g[r], i) >= least ? 1u : 0u) << (r * E + i);
    }
    if (rose) {
      // Logits equal to the bound matter in the slice that raised it alone (n_out + 1
      // others with lower tokens reach it for later ones), and of these the first
      // n_out + 1: of 256 rows masked with the lowest value all were gathered, and
      // then read again and again, in 689 us.
      if (count_threads(hits != 0) > kThreads / 4) {
        uint32_t equal = 0;
        for (uint32_t rest = hits; rest; rest &= rest - 1) {
          const int b = __ffs(rest) - 1, e = (b / E * kThreads + tid) * E + b % E;
          const float v = (float)(reinterpret_cast<const T*>(ring + stage * kStage))[e + mis];
          if (v == tau) equal |= 1u << b;
        }
        hits &= ~past_first(sh, equal, E, a.n_out + 1);
      }
      least = next_up(tau);
    }
    for (; hits; hits &= hits - 1) {
      const int b = __ffs(hits) - 1, e = (b / E * kThreads + tid) * E + b % E;  // of the slice
      const float v = (float)(reinterpret_cast<const T*>(ring + stage * kStage))[e + mis];
      const int at = atomicAdd(&sh.n, 1);
      if (at < kList) sh.list[at] = make_key(v, (uint32_t)((int64_t)(slice0 + it) * a.slice + e));
    }
    __syncwarp();
    if ((tid & 31) == 0) mbar_arrive(empty + 8 * stage);
  }
  const float2 halves = unpack2(l);
  finish<T>(a, sh, row, (int64_t)slice0 * a.slice, min((int64_t)a.vocab, (int64_t)(slice0 + slices) * a.slice), done, dead,
            m, lost ? NAN : halves.x + halves.y, tau);
}

}  // namespace

int beam_slice(int32_t dtype) { return kThreads * kGran * (dtype == LC_F32 ? 4 : 8); }

void launch_beam(BeamArgs a, int device, int sms, cudaStream_t s) {
  // as many parts a row as fill the card, of whole slices, their candidates at
  // most two for each thread of the block that ranks a group's
  const int rows = a.n_groups * a.n_beams, fill = std::max(1, kBeamPerSm * sms / rows);
  const int most = std::max(1, 2 * kThreads / (a.n_beams * a.n_out));
  a.per = (a.slices + std::min(fill, most) - 1) / std::min(fill, most);
  const dim3 grid((unsigned)((a.slices + a.per - 1) / a.per), (unsigned)rows);
  constexpr int kRing = kStages * kStage * 16;
  static_assert(kBeamPerSm * (kRing + (int)sizeof(BeamShared) + 1024) <= 228 * 1024, "the blocks fit an SM");
  auto launch = [&](auto kernel, SmemOptIn& opt) {
    opt(kernel, kRing, device);
    launch_pdl(kernel, grid, dim3(kThreads + 32), kRing, s, a);
  };
  static SmemOptIn f32, bf16, f16;
  if (a.dtype == LC_F32)
    launch(k_beam_select<float>, f32);
  else if (a.dtype == LC_BF16)
    launch(k_beam_select<__nv_bfloat16>, bf16);
  else
    launch(k_beam_select<__half>, f16);
}

}  // namespace lc
