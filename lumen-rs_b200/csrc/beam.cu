// Beam search's selection (lc_beam_select).
//
//   z[b, v] = score_b + ((x_bv - max_v x_b) - log sum_v exp(x_bv - max_v x_b))
//
// and of all b, v of a group the n_out largest z, lower b * V + v first among
// equals. The bytes of the logits bound it: one pass reads each logit once,
// into registers, and takes from it both the softmax sums and the slice's
// n_out best.
//
// A block takes a slice of one row. The n_out-th largest of the maxima of 64
// (or 256) disjoint sets of its logits is a lower bound of the slice's n_out-th
// largest logit, and few logits besides the best reach it; they are gathered
// and ranked by counting. The last slice of a row to finish has the row's sum,
// turns the slices' candidates into totals and ranks them; the last row of a
// group ranks the rows' candidates and writes the answer. One launch; ranks
// are by value and index only, so the order of arrival changes nothing.
#include <algorithm>

#include "devutil.cuh"
#include "paged.h"

namespace lc {
namespace {

constexpr int kThreads = 256;
constexpr int kGran = 8;      // 16-byte granules a thread holds
constexpr int kList = 1024;   // gathered candidates of a slice
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

__device__ __forceinline__ uint64_t block_max_key(uint64_t k, uint64_t* warp_key) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const uint64_t x = __shfl_xor_sync(~0u, k, o);
    k = x > k ? x : k;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warp_key[threadIdx.x >> 5] = k;
  __syncthreads();
  k = warp_key[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) k = warp_key[w] > k ? warp_key[w] : k;
  return k;
}

// Entries of the descending list[0 .. n) above key.
__device__ __forceinline__ int count_above(const uint64_t* list, int n, uint64_t key) {
  int b = 0, e = n;
  while (b < e) {
    const int m = (b + e) >> 1;
    if (list[m] > key)
      b = m + 1;
    else
      e = m;
  }
  return b;
}

// true in every thread of the block that arrives last of `of`
__device__ __forceinline__ bool arrive_last(int* counter, int of) {
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicAdd(counter, 1) == of - 1;
    if (last) *counter = 0;
  }
  __syncthreads();
  if (last) __threadfence();
  return last;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 4) k_beam_select(const BeamArgs a) {
  constexpr int E = 16 / sizeof(T);
  __shared__ __align__(16) uint64_t list[kBeamMaxMerge];  // the slice's list, then the merges' candidates
  __shared__ uint64_t warp_key[kThreads / 32];
  __shared__ __align__(16) float sets[kThreads];
  __shared__ float red_m[kThreads / 32], red_s[kThreads / 32];
  __shared__ float sh_tau, sh_shift;
  __shared__ int sh_n, sh_at[kThreads + 1];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y, slice = blockIdx.x, group = row / a.n_beams, beam = row - group * a.n_beams;
  const float score = a.scores[row];
  const bool done = a.finished && a.finished[row];
  const bool dead = done || !(score > kNegInf);  // its logits do not matter
  const int64_t srow = (int64_t)row * a.slices + slice;

  if (!dead) {
    const T* x0 = static_cast<const T*>(a.logits) + row * a.row_stride;
    const int mis = (int)((reinterpret_cast<uintptr_t>(x0) & 15) / sizeof(T));
    const T* base = x0 - mis;  // index i of the row sits at base[i + mis]
    const int i_end = mis + a.vocab;
    uint4 raw[kGran];
    const int64_t at0 = (int64_t)slice * a.slice + tid * E;
    if (at0 - tid * E >= mis && at0 - tid * E + a.slice <= i_end) {  // the whole slice is inside the row
#pragma unroll
      for (int r = 0; r < kGran; ++r) raw[r] = __ldcs(reinterpret_cast<const uint4*>(base + at0 + r * kThreads * E));
    } else {
#pragma unroll
      for (int r = 0; r < kGran; ++r) {
        const int64_t at = at0 + r * kThreads * E;
        if (at >= mis && at + E <= i_end) {
          raw[r] = __ldcs(reinterpret_cast<const uint4*>(base + at));
        } else {
          alignas(16) T part[E];
#pragma unroll
          for (int i = 0; i < E; ++i) part[i] = at + i >= mis && at + i < i_end ? base[at + i] : T(kNegInf);
          raw[r] = *reinterpret_cast<uint4*>(part);
        }
      }
    }
    float top = kNegInf;
#pragma unroll
    for (int r = 0; r < kGran; ++r) top = fmaxf(top, granule_max<T>(raw[r]));
    const float tg = top == kNegInf ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < kGran; ++r) {
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < E; ++i) part += ex2((elem<T>(raw[r], i) - tg) * kLog2e);
      sum += part;
    }
    // maxima of 64 sets of four threads, or of 256
    const bool few = a.n_out <= 16;
    float set = top;
    if (few) {
      set = fmaxf(set, __shfl_xor_sync(~0u, set, 1));
      set = fmaxf(set, __shfl_xor_sync(~0u, set, 2));
    }
    const int n_sets = few ? kThreads / 4 : kThreads;
    if (!few || (tid & 3) == 0) sets[few ? tid >> 2 : tid] = set;
    // the slice's max and sum
    float m = top, l = sum;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const float mo = __shfl_xor_sync(~0u, m, o), lo = __shfl_xor_sync(~0u, l, o);
      const float mn = fmaxf(m, mo), mg = mn == kNegInf ? 0.f : mn;
      l = l * ex2((m - mg) * kLog2e) + lo * ex2((mo - mg) * kLog2e);
      m = mn;
    }
    if (lane == 0) {
      red_m[warp] = m;
      red_s[warp] = l;
    }
    if (tid == 0) sh_n = 0;
    __syncthreads();
    if (tid < n_sets) {
      int r = 0;
      const float v = sets[tid];
#pragma unroll 4
      for (int i = 0; i < n_sets; i += 4) {
        const float4 x = *reinterpret_cast<const float4*>(sets + i);
        r += x.x > v || (x.x == v && i < tid);
        r += x.y > v || (x.y == v && i + 1 < tid);
        r += x.z > v || (x.z == v && i + 2 < tid);
        r += x.w > v || (x.w == v && i + 3 < tid);
      }
      if (r == a.n_out - 1) sh_tau = v;
    }
    if (tid == kThreads - 1) {  // a warp that has no set to rank where there are 64
      float mm = kNegInf, ll = 0.f;
      for (int w = 0; w < kThreads / 32; ++w) {
        const float mn = fmaxf(mm, red_m[w]), mg = mn == kNegInf ? 0.f : mn;
        ll = ll * ex2((mm - mg) * kLog2e) + red_s[w] * ex2((red_m[w] - mg) * kLog2e);
        mm = mn;
      }
      a.slice_stats[2 * srow] = mm;
      a.slice_stats[2 * srow + 1] = ll;
    }
    __syncthreads();
    const float tau = sh_tau;
#pragma unroll
    for (int r = 0; r < kGran; ++r) {
      if (!(granule_max<T>(raw[r]) >= tau)) continue;
      const int64_t index = at0 + r * kThreads * E - mis;
      for (int i = 0; i < E; ++i) {
        const float x = elem<T>(raw[r], i);
        if (x >= tau && x > kNegInf) {
          const int at = atomicAdd(&sh_n, 1);
          if (at < kList) list[at] = make_key(x, (uint32_t)(index + i));
        }
      }
    }
    __syncthreads();
    const int found = sh_n;
    uint64_t* keys = a.slice_key + srow * a.n_out;
    if (found <= kList) {
      for (int i = tid; i < found; i += kThreads) {
        const uint64_t k = list[i];
        int r = 0;
        for (int o = 0; o < found; ++o) r += list[o] > k;
        if (r < a.n_out) keys[r] = k;
      }
    } else {
      // many logits equal to the bound: one best after the other, from shared memory
      uint4* held = reinterpret_cast<uint4*>(list);
      static_assert(sizeof(list) >= kGran * kThreads * 16, "the slice fits the list");
#pragma unroll
      for (int r = 0; r < kGran; ++r) held[r * kThreads + tid] = raw[r];
      uint64_t before = ~0ull;
      for (int o = 0; o < a.n_out; ++o) {
        uint64_t best = 0;
#pragma unroll 1
        for (int r = 0; r < kGran; ++r) {
          const uint4 x4 = held[r * kThreads + tid];
#pragma unroll 1
          for (int i = 0; i < E; ++i) {
            const float x = elem<T>(x4, i);
            const uint64_t k = make_key(x, (uint32_t)(at0 + r * kThreads * E + i - mis));
            if (x >= tau && k < before && k > best) best = k;
          }
        }
        before = block_max_key(best, warp_key);
        if (tid == 0) keys[o] = before;
      }
    }
    if (tid == 0) a.slice_count[srow] = min(found, a.n_out);
  }

  // the row
  if (!arrive_last(a.counters + row, a.slices)) return;
  uint64_t* row_key = a.row_key + (int64_t)row * a.n_out;
  if (dead) {
    if (tid == 0) {
      const bool one = done && score > kNegInf;
      if (one) row_key[0] = make_key(score, (uint32_t)(beam * (int64_t)a.vocab + a.pad));
      a.row_count[row] = one;
    }
  } else {
    if (warp == 0) {  // max and sum over the slices, and where each slice's candidates start
      float m = kNegInf;
      for (int i = lane; i < a.slices; i += 32) m = fmaxf(m, __ldcg(a.slice_stats + 2 * ((int64_t)row * a.slices + i)));
#pragma unroll
      for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
      const float mg = m == kNegInf ? 0.f : m;
      float l = 0.f;
      for (int i = lane; i < a.slices; i += 32) {
        const float* st = a.slice_stats + 2 * ((int64_t)row * a.slices + i);
        l += __ldcg(st + 1) * ex2((__ldcg(st) - mg) * kLog2e);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(~0u, l, o);
      if (lane == 0) {
        red_m[0] = m;
        sh_shift = logf(l);
      }
    }
    for (int i = tid; i < a.slices; i += kThreads) sh_at[i] = __ldcg(a.slice_count + (int64_t)row * a.slices + i);
    if (tid == 0) sh_n = 0;
    __syncthreads();
    const float m = red_m[0], log_sum = sh_shift;
    // totals; a slice's list stays sorted but for totals that round to the same value
    for (int c = tid; c < a.slices * a.n_out; c += kThreads) {
      const int i = c / a.n_out, o = c - i * a.n_out;
      uint64_t k = 0;
      if (o < sh_at[i]) {
        const uint64_t x = __ldcg(a.slice_key + ((int64_t)row * a.slices + i) * a.n_out + o);
        const float z = score + ((key_value(x) - m) - log_sum);
        if (z > kNegInf) k = make_key(z, (uint32_t)(beam * (int64_t)a.vocab + key_index(x)));
      }
      list[c] = k;
      if (k) atomicAdd(&sh_n, 1);
    }
    __syncthreads();
    for (int c = tid; c < a.slices * a.n_out; c += kThreads) {
      const uint64_t k = list[c];
      if (!k) continue;
      int r = 0;
      for (int o = 0; o < a.slices * a.n_out; ++o) r += list[o] > k;
      if (r < a.n_out) row_key[r] = k;
    }
    if (tid == 0) a.row_count[row] = min(sh_n, a.n_out);
  }

  // the group
  if (!arrive_last(a.counters + a.n_groups * a.n_beams + group, a.n_beams)) return;
  const int64_t row0 = (int64_t)group * a.n_beams;
  for (int i = tid; i < a.n_beams; i += kThreads) sh_at[i] = __ldcg(a.row_count + row0 + i);
  if (tid == 0) sh_n = 0;
  __syncthreads();
  for (int c = tid; c < a.n_beams * a.n_out; c += kThreads) {
    const int i = c / a.n_out, o = c - i * a.n_out;
    if (o < sh_at[i]) list[c] = __ldcg(a.row_key + row0 * a.n_out + c);
  }
  __syncthreads();
  for (int c = tid; c < a.n_beams * a.n_out; c += kThreads) {
    const int i = c / a.n_out, o = c - i * a.n_out;
    if (o >= sh_at[i]) continue;
    const uint64_t k = list[c];
    int r = o;
    for (int b = 0; b < a.n_beams && r < a.n_out; ++b)
      if (b != i) r += count_above(list + b * a.n_out, sh_at[b], k);
    if (r >= a.n_out) continue;
    const uint32_t index = key_index(k), p = index / (uint32_t)a.vocab, tok = index - p * (uint32_t)a.vocab;
    const int64_t to = (int64_t)group * a.n_out + r;
    a.scores_out[to] = key_value(k);
    a.parents[to] = (int32_t)p;
    a.tokens[to] = (int32_t)tok;
    a.finished_out[to] = (a.finished && a.finished[row0 + p]) || (int32_t)tok == a.eos;
    atomicAdd(&sh_n, 1);
  }
  __syncthreads();
  for (int r = sh_n + tid; r < a.n_out; r += kThreads) {  // places with no candidate
    const int64_t to = (int64_t)group * a.n_out + r;
    a.scores_out[to] = kNegInf;
    a.parents[to] = r % a.n_beams;
    a.tokens[to] = a.pad;
    a.finished_out[to] = 1;
  }
}

}  // namespace

int beam_slice(int32_t dtype) { return kThreads * kGran * (dtype == LC_F32 ? 4 : 8); }

void launch_beam(const BeamArgs& a, cudaStream_t s) {
  const dim3 grid((unsigned)a.slices, (unsigned)(a.n_groups * a.n_beams));
  if (a.dtype == LC_F32)
    k_beam_select<float><<<grid, kThreads, 0, s>>>(a);
  else if (a.dtype == LC_BF16)
    k_beam_select<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
  else
    k_beam_select<__half><<<grid, kThreads, 0, s>>>(a);
  LC_CUDA(cudaGetLastError());
}

}  // namespace lc
