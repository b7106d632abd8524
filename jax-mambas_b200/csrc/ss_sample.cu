// Tokens from logits by temperature, top-k, top-p and min-p with given uniform
// numbers, for sm_100a.
//
//   s_i = logit_i / T;  w_i = round(2^31 exp(s_i - max s))
//   order: s descending, then index ascending
//   top-k keeps the first k; top-p of those the ones whose predecessors hold
//   less than p of their mass; min-p the ones with w_i >= p_min 2^31
//   token: the first i, by index, with sum of kept w_0..w_i > floor(u sum w)
//
// The weights are whole numbers, so every sum is exact and no result depends on
// the order in which threads add. (A token less likely than 2^-32 of the
// likeliest has weight 0 and is never drawn.) No sort of the row: what the
// filters need is one cutoff in the order, a 64-bit key of (s, index).
//
// A row is shared by a cluster of CTAs, each keeping its slice in shared memory
// as it comes, so logits are read from HBM once; later passes run on chip.
//  * top-k up to a few hundred: every thread's own maximum is known after the load. Each
//    warp gives the largest of its 32, somewhat more than its share of k; the
//    k-th largest of those (k elements are at least that large), found bit by bit,
//    bounds the row's k-th largest from below and leaves little more than k
//    candidates. They go to rank 0; all filters and the draw work on that list.
//  * otherwise a histogram of 1024 bins of s below the maximum (count, and mass in
//    two 16-bit halves so that 32-bit shared-memory atomics suffice), then a sort
//    of the one bin where the cutoff falls; a bin that is too full (rows with very many equal
//    logits) takes a binary search over the key instead. The draw needs the kept
//    mass by units of 512 elements: the pass that gathers the bin sums it as well.
// Bound by the latency of its passes and barriers for few rows, by the passes'
// instructions (an exponential, and a division where T is not 1, per element) for
// many. Measured at 50280 logits, 32 rows fp32 / 512 rows bf16: greedy 7 / 31 us, no
// filter 9 / 44, top-k 50 10 / 40, top-k 200 with top-p 0.9 13 / 61, top-k 500 19 /
// 109, top-p 0.9 alone 21 / 114, at T = 0.8 23 / 130; a mixture of all 25 / 67 us.
#include "ss_ops.h"
#include "ss_tcgen05.cuh"

#include <cstddef>

namespace mss {

constexpr int kSampleThreads = 512;
constexpr int kWarps = kSampleThreads / 32;
constexpr int kBins = 1024;
constexpr float kBinsPerNat = 46.f;  // 1024 / 46 = 22.26 > 32 ln 2: covers every weight > 0
constexpr int kSortCap = 2048;
constexpr int kUnit = 512;  // elements whose kept mass is summed as one
constexpr float kOne = 2147483648.f;
constexpr int kBoundLow = 14;  // bits of the candidates' bound that are not searched

// Rows up to which the costly ones are taken first, and the top_k above which a row is
// one (512 rows of 5000 in a mixture, 200 among its top_k: 24 us, 29 at 512).
constexpr int kOrderRows = 2048;
constexpr int kCheapK = 128;
// top_k up to which a list serves top-k alone. 512 rows of 50280 bf16 logits / 32 rows
// fp32, list against histogram: 300 99 / 18.4 against 107 / 19.0 us, 400 120 / 21.5
// against 108 / 19.2. With top-p as well, a second cutoff of the histogram: 400 114 / 20.7
// against 152 / 27.3.
constexpr int kListK = 320;

struct __align__(16) SampleShared {
  unsigned long long red[2][2][kWarps];  // per-warp values of a reduction
  unsigned long long sum[2][2];          // this CTA's value, read by the cluster
  float maxv[kWarps];
  float cta_max;
  uint32_t lead[kWarps * 32];            // each warp's leading lane maxima, ordered
  unsigned int count;                    // of this CTA's list (rank 0: of the joint one)
  int bin;                               // where the cutoff falls, and what is ahead of it
  unsigned long long before_count, before_mass;
  unsigned long long cut, kept_mass;     // rank 0's copy is the cluster's
  int costly[kOrderRows / kSampleThreads][kWarps];  // rows' order (row_of)
  int row;
  // block scan of the bins
  unsigned long long scan[2][kWarps];
  unsigned long long total[2];           // this CTA's bins
  // the histogram is read for the last time before the sort begins
  union {
    struct {
      unsigned int cnt[kBins], lo[kBins], hi[kBins];
    };
    __align__(16) unsigned long long sort[kSortCap];  // read by 16 bytes as well
  };
};
static_assert(offsetof(SampleShared, sort) % 16 == 0 && sizeof(SampleShared) % 16 == 0,
              "16-byte accesses of the list and of what follows the struct");

// A slice of logits in shared memory as they came, read as s = x / div, filled up
// with -inf to whole units. NaN needs no care: its weight converts to 0 and every
// comparison with it is false.
template <typename T>
struct Slice {
  const T* x;
  int n;
  float div;
  __device__ __forceinline__ float operator[](int i) const {
    const float v = to_f32(x[i]);
    return div != 1.f ? v / div : v;
  }
  // Elements i .. i + 3, i a multiple of 4.
  __device__ __forceinline__ float4 four(int i) const {
    float4 v;
    if constexpr (sizeof(T) == 4)
      v = *reinterpret_cast<const float4*>(x + i);
    else
      v = bf16x4_to_f32(*reinterpret_cast<const uint2*>(x + i));
    if (div != 1.f) v = make_float4(v.x / div, v.y / div, v.z / div, v.w / div);
    return v;
  }
  // f(s, index) for every element of the slice, four at a time per thread.
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 2
    for (int i = threadIdx.x * 4; i < n; i += kSampleThreads * 4) {
      const float4 v = four(i);
      f(v.x, i);
      f(v.y, i + 1);
      f(v.z, i + 2);
      f(v.w, i + 3);
    }
  }
};

__device__ __forceinline__ unsigned long long cluster_ld64(uint32_t addr) {
  unsigned long long v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t cluster_ld32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_st64(uint32_t addr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}

// A shared-memory word of every CTA of the row, zero past the last; the loads are
// all under way before the first is used.
__device__ __forceinline__ void cluster_gather32(const void* at, int ctas, uint32_t (&v)[8]) {
#pragma unroll
  for (int r = 0; r < 8; ++r) v[r] = r < ctas ? cluster_ld32(cluster_map(smem_u32(at), r)) : 0u;
}
__device__ __forceinline__ void cluster_gather64(const void* at, int ctas,
                                                 unsigned long long (&v)[8]) {
#pragma unroll
  for (int r = 0; r < 8; ++r) v[r] = r < ctas ? cluster_ld64(cluster_map(smem_u32(at), r)) : 0ull;
}

// Every thread of the cluster.
__device__ __forceinline__ void sync_row(int ctas) {
  if (ctas == 1)
    __syncthreads();
  else
    cluster_sync_all();
}

// Position in the order as a whole number, larger first: s as an ordered
// integer, then the complement of the index.
__device__ __forceinline__ unsigned long long order_key(float s, int i) {
  uint32_t b = __float_as_uint(s + 0.f);  // -0 counts as 0
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return (static_cast<unsigned long long>(b) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ float key_value(unsigned long long key) {
  const uint32_t b = static_cast<uint32_t>(key >> 32);
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

// top is finite here (see the kernel).
__device__ __forceinline__ uint32_t weight_of(float s, float top) {
  return __float2uint_rn(expf(s - top) * kOne);
}
__device__ __forceinline__ int bin_of(float s, float top) {
  return min(kBins - 1, static_cast<int>((top - s) * kBinsPerNat));
}

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums of (a, b) over the cluster, in every thread. `slot` alternates, so a
// slot is written again only after the barrier of the call in between.
__device__ void row_sums(SampleShared& sh, int ctas, int& slot, unsigned long long& a,
                         unsigned long long& b) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  a = warp_sum64(a);
  b = warp_sum64(b);
  if (lane == 0) {
    sh.red[slot][0][warp] = a;
    sh.red[slot][1][warp] = b;
  }
  __syncthreads();
  a = b = 0;
  for (int w = 0; w < kWarps; ++w) {
    a += sh.red[slot][0][w];
    b += sh.red[slot][1][w];
  }
  if (ctas > 1) {
    if (threadIdx.x == 0) {
      sh.sum[slot][0] = a;
      sh.sum[slot][1] = b;
    }
    cluster_sync_all();
    unsigned long long va[8], vb[8];
    cluster_gather64(&sh.sum[slot][0], ctas, va);
    cluster_gather64(&sh.sum[slot][1], ctas, vb);
    a = b = 0;
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      a += va[r];
      b += vb[r];
    }
  }
  slot ^= 1;
}

// The smallest key t for which the elements above t hold less than the limit:
// fewer than `limit` of them (by_mass false), or mass below `limit`. Those at
// or above t are the kept ones. One pass over the slice per key bit.
template <typename T>
__device__ unsigned long long search_cut(SampleShared& sh, const Slice<T>& s, int base, float top,
                                         int ctas, int& slot, bool by_mass, double limit) {
  unsigned long long t = 0;
  for (int bit = 63; bit >= 0; --bit) {
    // is some t' < 2^bit above t's prefix enough? test the largest such
    const unsigned long long probe = t | ((1ull << bit) - 1);
    unsigned long long c = 0, m = 0;
    s.each([&](float v, int i) {
      const uint32_t w = weight_of(v, top);
      if (w != 0 && order_key(v, base + i) > probe) {
        ++c;
        m += w;
      }
    });
    row_sums(sh, ctas, slot, c, m);
    if (!(static_cast<double>(by_mass ? m : c) < limit)) t |= 1ull << bit;
  }
  return t;
}

// Sorts the different numbers sh.sort[0..m) by the whole CTA, m <= kSortCap,
// descending; the result's place is returned. Up to 512 by counting what is larger (each number's place), one to
// eight neighbouring lanes per number: a sorting network's 45 steps and barriers
// take longer. Above that a bitonic network.
__device__ const unsigned long long* sort_desc(SampleShared& sh, int m) {
  if (m <= kSampleThreads) {
    unsigned long long* out = sh.sort + kSampleThreads;
    const int parts = m <= 64 ? 8 : m <= 128 ? 4 : m <= 256 ? 2 : 1;
    const int t = threadIdx.x / parts, part = threadIdx.x % parts;
    const unsigned long long own = t < m ? sh.sort[t] : 0;
    int ahead = (m & 1) && part == 0 ? sh.sort[m - 1] > own : 0;
    const ulonglong2* pairs = reinterpret_cast<const ulonglong2*>(sh.sort);
#pragma unroll 4
    for (int j = part; j < m / 2; j += parts) {
      const ulonglong2 two = pairs[j];
      ahead += (two.x > own) + (two.y > own);
    }
    for (int o = 1; o < parts; o *= 2) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    if (t < m && part == 0) out[ahead] = own;
    __syncthreads();
    return out;
  }
  int size = 1024;
  while (size < m) size *= 2;
  for (int i = m + threadIdx.x; i < size; i += kSampleThreads) sh.sort[i] = 0;
  __syncthreads();
  for (int k = 2; k <= size; k *= 2) {
    for (int j = k / 2; j > 0; j /= 2) {
      for (int p = threadIdx.x; p < size / 2; p += kSampleThreads) {
        const int i = 2 * p - (p & (j - 1));
        const unsigned long long x = sh.sort[i], y = sh.sort[i + j];
        if ((x < y) == ((i & k) == 0)) {
          sh.sort[i] = y;
          sh.sort[i + j] = x;
        }
      }
      // pairs up to 32 apart stay within one warp's 64 places
      if (j > 32 || (j == 1 && k > 32))
        __syncthreads();
      else
        __syncwarp();
    }
  }
  __syncthreads();
  return sh.sort;
}

// Inclusive sum over the warp's lanes up to this one.
__device__ __forceinline__ unsigned long long warp_scan64(unsigned long long v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o *= 2) {
    const unsigned long long up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}

// Appends an element to this CTA's list (dropped, but counted, past its end).
__device__ __forceinline__ void push(SampleShared& sh, unsigned long long key) {
  const unsigned int at = atomicAdd(&sh.count, 1u);
  if (at < kSortCap) sh.sort[at] = key;
}

// After the CTAs' lists are complete: their joint length in every thread (more
// than kSortCap: not joined), and rank 0's list is all of them. Ends with a
// barrier after the last access to another CTA's memory; a row's only CTA has none after
// its read of sh.count, so who sets that anew waits for its threads first.
__device__ int join_lists(SampleShared& sh, int rank, int ctas) {
  sync_row(ctas);
  if (ctas == 1) return static_cast<int>(sh.count);
  uint32_t n[8];
  cluster_gather32(&sh.count, ctas, n);
  int total = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) total += static_cast<int>(n[r]);
  if (rank == 0 && total <= kSortCap) {
    // place i of the joint list: rank r's place i - start
    for (int i = static_cast<int>(n[0] + threadIdx.x); i < total; i += kSampleThreads) {
      int start = 0, from = 0;
      int end = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (i >= end && i < end + static_cast<int>(n[r])) {
          start = end;
          from = r;
        }
        end += static_cast<int>(n[r]);
      }
      sh.sort[i] = cluster_ld64(cluster_map(smem_u32(&sh.sort[0]), from) + 8 * (i - start));
    }
  }
  sync_row(ctas);
  return total;
}

__device__ __forceinline__ unsigned long long target_of(float uniform, unsigned long long total) {
  const double u = fmin(fmax(static_cast<double>(uniform), 0.0), 1.0);
  return min(static_cast<unsigned long long>(u * static_cast<double>(total)), total - 1);
}

// Gathers the elements of one bin in rank 0, which sorts them, finds the cutoff and
// publishes it (sh.cut, sh.kept_mass: the mass of all kept). False if there are
// too many. With unit_mass (the last cutoff) the pass also sums the mass of w >= w_min by
// units: all that is ahead of the bin, then the list's kept ones.
template <typename T>
__device__ bool sort_cut(SampleShared& sh, const Slice<T>& s, int base, float top, int rank,
                         int ctas, int bin, bool by_mass, unsigned long long before_count,
                         unsigned long long before_mass, double limit,
                         unsigned long long* unit_mass, int units, uint32_t w_min) {
  // bin_of(v) == bin, without the conversion
  const float from = static_cast<float>(bin), to = bin + 1 == kBins ? INFINITY : from + 1.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int u = warp; u < units; u += kWarps) {
    unsigned long long sum = 0;
#pragma unroll
    for (int e = 0; e < kUnit / 128; ++e) {
      const int i = u * kUnit + e * 128 + lane * 4;
      const float4 v = s.four(i);
      const float most = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w));
      if (__any_sync(0xffffffffu, (top - most) * kBinsPerNat < to)) {
        const float each[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const float f = (top - each[c]) * kBinsPerNat;
          const uint32_t w = weight_of(each[c], top);
          if (f >= from && f < to && w != 0) push(sh, order_key(each[c], base + i + c));
          sum += (f < from) & (w >= w_min) ? w : 0u;
        }
      }
    }
    if (unit_mass != nullptr) {
      sum = warp_sum64(sum);
      if (lane == 0) unit_mass[u] = sum;
    }
  }
  const int m = join_lists(sh, rank, ctas);
  const int own = rank == 0 ? m : static_cast<int>(sh.count);  // entries of this CTA's list
  if (m > kSortCap) {
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;  // counted in again after another barrier
    return false;
  }
  if (rank == 0) {
    const unsigned long long* sorted = sort_desc(sh, m);
    // one warp walks the sorted bin, 32 elements at a time
    if (threadIdx.x < 32) {
      unsigned long long count = before_count, mass = before_mass, cut = 0, kept = before_mass;
      for (int p = 0; p < m; p += 32) {
        const int i = p + threadIdx.x;
        const unsigned long long key = i < m ? sorted[i] : 0;
        const unsigned long long w = i < m ? weight_of(key_value(key), top) : 0;
        const unsigned long long run = warp_scan64(w);
        const double ahead = by_mass ? static_cast<double>(mass + run - w)
                                     : static_cast<double>(count + threadIdx.x);
        const unsigned keep = __ballot_sync(0xffffffffu, i < m && ahead < limit);
        if (keep != 0) {  // a prefix of the lanes: the order's first ones
          const int last = 31 - __clz(keep);
          cut = __shfl_sync(0xffffffffu, key, last);
          kept = mass + __shfl_sync(0xffffffffu, run, last);
        }
        if (keep != 0xffffffffu) break;
        count += 32;
        mass += __shfl_sync(0xffffffffu, run, 31);
      }
      if (threadIdx.x == 0) {
        sh.cut = cut;
        sh.kept_mass = kept;
      }
    }
  }
  sync_row(ctas);
  if (threadIdx.x == 0) sh.count = 0;  // likewise
  if (unit_mass != nullptr) {
    // rank 0's list is all ranks', in some order; the others still hold their own
    const unsigned long long cut = cluster_ld64(cluster_map(smem_u32(&sh.cut), 0));
    for (int j = threadIdx.x; j < own; j += kSampleThreads) {
      const unsigned long long key = sh.sort[j];
      const int64_t i = static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(key)) - base;
      const uint32_t w = weight_of(key_value(key), top);
      if (key >= cut && w >= w_min && i < s.n)
        atomicAdd(&unit_mass[i / kUnit], static_cast<unsigned long long>(w));
    }
  }
  return true;
}

// Sum over the CTA, in every thread; buf is one of the scan buffers.
__device__ __forceinline__ unsigned long long cta_sum64(unsigned long long v,
                                                        unsigned long long* buf) {
  v = warp_sum64(v);
  if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int q = 0; q < kWarps; ++q) v += buf[q];
  return v;
}

// Number and mass (mass[j]: weight of sh.sort[j]) of the m elements ahead of key.
__device__ __forceinline__ void count_ahead(const SampleShared& sh, const unsigned long long* mass,
                                            int m, unsigned long long key, int part, int parts,
                                            int& ahead, unsigned long long& before) {
  ahead = 0;
  before = 0;
#pragma unroll 4
  for (int j = part; j < m; j += parts) {
    const bool first = sh.sort[j] > key;
    ahead += first;
    before += first ? mass[j] : 0ull;
  }
  for (int o = 1; o < parts; o *= 2) {
    ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
    before += __shfl_xor_sync(0xffffffffu, before, o);
  }
}

// Rank 0, with m <= kCountCap candidates in sh.sort (all elements down to some key,
// the first top_k among them): applies the filters and draws. No sort: for each
// candidate, shared by kCountParts neighbouring lanes, the list is walked, adding up
// what is ahead of it in the order, then what is kept at lower indices.
// (512 bf16 rows of 50280 with top-k 50, m about 55: 40 us against 43 by sorting; with
// top-k 100, m about 110, 48 against 47.)
constexpr int kCountCap = 64, kCountParts = kSampleThreads / kCountCap;
__device__ void draw_by_counting(SampleShared& sh, int m, float top, int top_k, float top_p,
                                 uint32_t w_min, float uniform, int64_t* token) {
  unsigned long long* mass = sh.sort + kSampleThreads;  // weights, then kept weights
  constexpr int parts = kCountParts;
  const int t = threadIdx.x / parts, part = threadIdx.x % parts;
  const unsigned long long key = t < m ? sh.sort[t] : 0;
  const uint32_t w = t < m ? weight_of(key_value(key), top) : 0;
  if (part == 0) mass[t] = w;
  __syncthreads();
  int ahead;
  unsigned long long before;
  count_ahead(sh, mass, m, key, part, parts, ahead, before);
  const bool in_k = w != 0 && ahead < top_k;
  const unsigned long long row_mass = cta_sum64(in_k && part == 0 ? w : 0u, sh.scan[0]);
  const double limit = static_cast<double>(top_p) * static_cast<double>(row_mass);
  const bool keep =
      in_k && (!(top_p < 1.f) || static_cast<double>(before) < limit) && (w >= w_min);
  // (the weights were last read before the sum's barrier)
  if (part == 0) mass[t] = keep ? w : 0u;
  const unsigned long long total = cta_sum64(keep && part == 0 ? w : 0u, sh.scan[1]);
  const unsigned long long target = target_of(uniform, total);
  const uint32_t rev = static_cast<uint32_t>(key);  // complement of the index
  unsigned long long run = 0;
#pragma unroll 4
  for (int j = part; j < m; j += parts)
    run += static_cast<uint32_t>(sh.sort[j]) > rev ? mass[j] : 0ull;
  for (int o = 1; o < parts; o *= 2) run += __shfl_xor_sync(0xffffffffu, run, o);
  if (keep && part == 0 && run <= target && target < run + w)
    *token = static_cast<int64_t>(0xffffffffu - rev);
}

// The same for up to kSortCap candidates: sorted by the order, of which the first top_k
// (at most one per thread) pass the filters, and the kept ones put in the indices'
// order by counting as in sort_desc.
__device__ void draw_by_sorting(SampleShared& sh, int m, float top, int top_k, float top_p,
                                uint32_t w_min, float uniform, int64_t* token) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, t = threadIdx.x;
  const unsigned long long* sorted = sort_desc(sh, m);
  m = min(m, top_k);
  const unsigned long long key = t < m ? sorted[t] : 0;
  const uint32_t w = t < m ? weight_of(key_value(key), top) : 0;
  unsigned long long run = warp_scan64(w);
  if (lane == 31) sh.scan[0][warp] = run;
  __syncthreads();
  unsigned long long total = 0;
  for (int q = 0; q < kWarps; ++q) {
    if (q < warp) run += sh.scan[0][q];
    total += sh.scan[0][q];
  }
  const double limit = static_cast<double>(top_p) * static_cast<double>(total);
  // weights fall along the order, so what is kept is its beginning
  const bool keep =
      w != 0 && (!(top_p < 1.f) || static_cast<double>(run - w) < limit) && w >= w_min;
  uint32_t* revs = reinterpret_cast<uint32_t*>(sh.sort);  // complements of the indices
  uint32_t* mass = revs + kSampleThreads;
  unsigned long long* placed = sh.sort + kSampleThreads;
  const int kept = __syncthreads_count(keep);
  revs[t] = keep ? static_cast<uint32_t>(key) : 0u;  // 0: after every index
  mass[t] = w;
  placed[t] = 0;
  __syncthreads();
  const int parts = kept <= 64 ? 8 : kept <= 128 ? 4 : kept <= 256 ? 2 : 1;
  const int at = t / parts, part = t % parts;
  const uint32_t own = revs[at];
  int ahead = 0;
#pragma unroll 4
  for (int j = part * 4; j < kept; j += parts * 4) {
    const uint4 four = *reinterpret_cast<const uint4*>(revs + j);
    ahead += (four.x > own) + (four.y > own) + (four.z > own) + (four.w > own);
  }
  for (int o = 1; o < parts; o *= 2) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
  if (at < kept && part == 0)
    placed[ahead] = (static_cast<unsigned long long>(own) << 32) | mass[at];
  __syncthreads();
  const unsigned long long mine = placed[t];
  const uint32_t weight = static_cast<uint32_t>(mine);
  run = warp_scan64(weight);
  if (lane == 31) sh.scan[1][warp] = run;
  __syncthreads();
  total = 0;
  for (int q = 0; q < kWarps; ++q) {
    if (q < warp) run += sh.scan[1][q];
    total += sh.scan[1][q];
  }
  const unsigned long long target = target_of(uniform, total);
  if (run - weight <= target && target < run)
    *token = static_cast<int64_t>(0xffffffffu - static_cast<uint32_t>(mine >> 32));
}

// A float's bits as a whole number of the same order, and back.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t b) {
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}

// The row of cluster n. Rows that need a histogram or a long list take several times
// as long as others; where the clusters come in a few rounds (by_cost) they are taken
// first, so that none of them starts last.
__device__ int row_of(const SampleParams& p, SampleShared& sh, int n, int by_cost) {
  if (!by_cost) return n;
  constexpr int kEach = kOrderRows / kSampleThreads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned mine[kEach];
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int r = q * kSampleThreads + threadIdx.x;
    bool costly = false;
    if (r < p.rows) {
      const float t = p.temperature ? p.temperature[r] : p.temperature_all;
      const int k = p.top_k ? p.top_k[r] : p.top_k_all;
      const float f = p.top_p ? p.top_p[r] : p.top_p_all;
      costly = t > 0.f && f > 0.f && (k > kCheapK || (k <= 0 && f < 1.f));
    }
    mine[q] = __ballot_sync(0xffffffffu, costly);
    if (lane == 0) sh.costly[q][warp] = __popc(mine[q]);
  }
  __syncthreads();
  int all = 0, before[kEach];
#pragma unroll
  for (int q = 0; q < kEach; ++q)
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) before[q] = all;
      all += sh.costly[q][w];
    }
#pragma unroll
  for (int q = 0; q < kEach; ++q) {
    const int r = q * kSampleThreads + threadIdx.x;
    const int ahead = before[q] + __popc(mine[q] & ((1u << lane) - 1u));  // costly rows before r
    const int place = (mine[q] >> lane) & 1u ? ahead : all + r - ahead;
    if (r < p.rows && place == n) sh.row = r;
  }
  __syncthreads();
  return sh.row;
}

template <typename T, int kCtasPerSm>
__global__ void __launch_bounds__(kSampleThreads, kCtasPerSm)
    ss_sample_kernel(const SampleParams p, int chunk, int vec, int by_cost) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem_raw);
  const int units = (chunk + kUnit - 1) / kUnit;
  unsigned long long* unit_mass =
      reinterpret_cast<unsigned long long*>(smem_raw + sizeof(SampleShared));
  T* cache = reinterpret_cast<T*>(unit_mass + (units + 1) / 2 * 2);
  const int ctas = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_rank());
  const int row = row_of(p, sh, blockIdx.x / ctas, by_cost);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int base = rank * chunk;
  const int n = max(0, min(chunk, p.vocab - base));  // this CTA's elements
  int slot = 0;

  const float temp = p.temperature ? p.temperature[row] : p.temperature_all;
  int top_k = p.top_k ? p.top_k[row] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[row] : p.top_p_all;
  const float min_p = p.min_p ? p.min_p[row] : p.min_p_all;
  // one kept token: the first in the order
  const bool greedy = !(temp > 0.f) || top_k == 1 || !(top_p > 0.f) || !(min_p <= 1.f);
  const Slice<T> s{cache, n, temp > 0.f ? temp : 1.f};
  if (top_k >= p.vocab) top_k = 0;
  const bool by_p = top_p < 1.f;
  // top-k up to kListK, with top-p up to kSampleThreads: a list of the row's largest
  // elements. per_warp: lane maxima that a warp gives, its share of top_k and about one
  // and a half deviations.
  const bool list = !greedy && top_k > 0 && top_k <= (by_p ? kSampleThreads : kListK);
  const float lead_share = static_cast<float>(top_k) / static_cast<float>(kWarps * ctas);
  const int per_warp = min(32, static_cast<int>(lead_share + 1.5f * sqrtf(lead_share)) + 1);

  // ---- the slice and its maximum (of x: x / div is monotone)
  const T* x = static_cast<const T*>(p.logits) + row * p.stride + base;
  constexpr int kPer = 16 / sizeof(T);
  float mx = -INFINITY;
  if (vec) {
    const int whole = n / kPer;
#pragma unroll 4
    for (int i = threadIdx.x; i < whole; i += kSampleThreads) {
      const uint4 w = __ldg(reinterpret_cast<const uint4*>(x) + i);
      *reinterpret_cast<uint4*>(cache + i * kPer) = w;
      if constexpr (sizeof(T) == 4) {
        mx = fmaxf(mx, fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)),
                             fmaxf(__uint_as_float(w.z), __uint_as_float(w.w))));
      } else {
        const float4 a = bf16x4_to_f32(make_uint2(w.x, w.y));
        const float4 b = bf16x4_to_f32(make_uint2(w.z, w.w));
        mx = fmaxf(mx, fmaxf(fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)),
                             fmaxf(fmaxf(b.x, b.y), fmaxf(b.z, b.w))));
      }
    }
    for (int i = whole * kPer + threadIdx.x; i < n; i += kSampleThreads) {
      cache[i] = x[i];
      mx = fmaxf(mx, to_f32(x[i]));
    }
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += kSampleThreads) {
      cache[i] = x[i];
      mx = fmaxf(mx, to_f32(x[i]));
    }
  }
  for (int i = n + threadIdx.x; i < units * kUnit; i += kSampleThreads)
    Elem<T>::st(cache + i, -INFINITY);
  if (threadIdx.x == 0) sh.count = 0;
  {
    uint32_t left = ordered(mx);
    const uint32_t most = __reduce_max_sync(0xffffffffu, left);
    if (list) {
      uint32_t next = most;
      for (int q = 0; q < per_warp; ++q) {
        if (lane == 0) sh.lead[warp * per_warp + q] = next;
        if (lane == __ffs(__ballot_sync(0xffffffffu, left == next)) - 1) left = 0;
        next = __reduce_max_sync(0xffffffffu, left);
      }
    }
    if (lane == 0) sh.maxv[warp] = unordered(most);
  }
  __syncthreads();
  mx = sh.maxv[0];
  for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, sh.maxv[w]);
  if (ctas > 1) {
    if (threadIdx.x == 0) sh.cta_max = mx;
    cluster_sync_all();
    uint32_t v[8];
    cluster_gather32(&sh.cta_max, ctas, v);
#pragma unroll
    for (int r = 0; r < 8; ++r)
      if (r < ctas) mx = fmaxf(mx, __uint_as_float(v[r]));
  }
  float top = mx == -INFINITY ? mx : mx / s.div;
  // Rare: an infinity, or a quotient that is not finite. Against the largest logit any
  // other then has no weight (floats that far out differ by many powers of e), so the
  // largest are the only tokens, all equal.
  const bool flat = mx > -INFINITY && !(fabsf(top) < INFINITY);
  if (flat) {
    for (int i = threadIdx.x; i < n; i += kSampleThreads)
      Elem<T>::st(cache + i, to_f32(cache[i]) == mx ? 0.f : -INFINITY);
    top = 0.f;
    __syncthreads();
  }

  if (greedy || top == -INFINITY) {
    int first = 0x7fffffff;
    if (top > -INFINITY)
      for (int i = threadIdx.x; i < n; i += kSampleThreads)
        if (s[i] == top) {
          first = base + i;
          break;
        }
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) sh.red[0][0][warp] = static_cast<unsigned long long>(first);
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 0; w < kWarps; ++w) first = min(first, static_cast<int>(sh.red[0][0][w]));
      sh.sum[0][0] = static_cast<unsigned long long>(first);
    }
    sync_row(ctas);
    if (rank == 0 && threadIdx.x == 0) {
      for (int r = 1; r < ctas; ++r)
        first = min(first, static_cast<int>(cluster_ld64(cluster_map(smem_u32(&sh.sum[0][0]), r))));
      p.tokens[row] = top > -INFINITY ? first : -1;
    }
    if (ctas > 1) cluster_sync_all();  // no CTA leaves while another reads its memory
    return;
  }
  // w >= min_p 2^31 in whole numbers
  const uint32_t w_min =
      static_cast<uint32_t>(ceil(fmax(static_cast<double>(min_p), 0.0) * kOne));

  // ---- few candidates
  if (list) {
    // The top_k-th largest of the warps' leading maxima, rounded down (kBoundLow bits
    // left out: a few candidates more, fewer steps), bit by bit by the whole CTA; in all
    // of the row's CTAs alike. Fewer than that many: no bound.
    const int lead_n = kWarps * per_warp, all_n = lead_n * ctas;
    uint32_t own[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = e * kSampleThreads + threadIdx.x;
      own[e] = i < all_n ? cluster_ld32(cluster_map(smem_u32(&sh.lead[i % lead_n]), i / lead_n)) : 0u;
    }
    uint32_t bound = 0;
    if (all_n >= top_k) {
      for (int bit = 31; bit >= kBoundLow; --bit) {
        const uint32_t t = bound | (1u << bit);
        int above = __syncthreads_count(own[0] >= t);
        if (all_n > kSampleThreads) above += __syncthreads_count(own[1] >= t);
        if (above >= top_k) bound = t;
      }
    }
    const bool bounded = bound > ordered(-INFINITY);
    float lowest = bounded ? unordered(bound) / s.div : -INFINITY;
    if (flat) lowest = 0.f;
    s.each([&](float v, int i) {
      if (v >= lowest && v > -INFINITY) push(sh, order_key(v, base + i));
    });
    const int m = join_lists(sh, rank, ctas);
    if (m <= kSortCap) {
      if (rank == 0) {
        if (m <= kCountCap)
          draw_by_counting(sh, m, top, top_k, top_p, w_min, p.uniform[row], p.tokens + row);
        else
          draw_by_sorting(sh, m, top, top_k, top_p, w_min, p.uniform[row], p.tokens + row);
      }
      return;
    }
    // too many equal logits: the general way
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;  // counted in again after another barrier
  }

  // ---- cutoff of top-k and top-p
  unsigned long long cut = 0;
  bool summed = false;  // unit_mass is ready
  if (top_k > 0 || by_p) {
    for (int i = threadIdx.x; i < kBins; i += kSampleThreads) sh.cnt[i] = sh.lo[i] = sh.hi[i] = 0;
    __syncthreads();
    s.each([&](float v, int) {
      const uint32_t w = weight_of(v, top);
      if (w != 0) {
        const int b = bin_of(v, top);
        if (top_k > 0) atomicAdd(&sh.cnt[b], 1u);
        atomicAdd(&sh.lo[b], w & 0xffffu);
        atomicAdd(&sh.hi[b], w >> 16);
      }
    });
    sync_row(ctas);
    // this CTA's share of the bins, `per` consecutive ones per thread
    const int share = kBins / ctas;
    const int per = max(1, share / kSampleThreads);
    const bool owner = static_cast<int>(threadIdx.x) * per < share;
    const int bin0 = rank * share + threadIdx.x * per;
    constexpr int kMost = kBins / kSampleThreads;
    unsigned long long bc[kMost], bm[kMost];
    unsigned long long c = 0, m = 0;
#pragma unroll
    for (int e = 0; e < kMost; ++e) {
      bc[e] = bm[e] = 0;
      if (owner && e < per) {
        uint32_t lo[8], hi[8];
        cluster_gather32(&sh.lo[bin0 + e], ctas, lo);
        cluster_gather32(&sh.hi[bin0 + e], ctas, hi);
#pragma unroll
        for (int r = 0; r < 8; ++r)
          bm[e] += lo[r] + (static_cast<unsigned long long>(hi[r]) << 16);
        if (top_k > 0) {
          cluster_gather32(&sh.cnt[bin0 + e], ctas, lo);
#pragma unroll
          for (int r = 0; r < 8; ++r) bc[e] += lo[r];
        }
      }
      c += bc[e];
      m += bm[e];
    }
    // exclusive prefix over the cluster's bins
    const unsigned long long rc = warp_scan64(c), rm = warp_scan64(m);
    if (lane == 31) {
      sh.scan[0][warp] = rc;
      sh.scan[1][warp] = rm;
    }
    __syncthreads();
    unsigned long long pc = rc - c, pm = rm - m, all_c = 0, all_m = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) {
        pc += sh.scan[0][w];
        pm += sh.scan[1][w];
      }
      all_c += sh.scan[0][w];
      all_m += sh.scan[1][w];
    }
    if (ctas > 1) {
      if (threadIdx.x == 0) {
        sh.total[0] = all_c;
        sh.total[1] = all_m;
      }
      cluster_sync_all();
      all_c = all_m = 0;
      unsigned long long tc[8], tm[8];
      cluster_gather64(&sh.total[0], ctas, tc);
      cluster_gather64(&sh.total[1], ctas, tm);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        if (r < rank) {
          pc += tc[r];
          pm += tm[r];
        }
        all_c += tc[r];
        all_m += tm[r];
      }
    }
    // the bin where the order passes `limit`, told to every CTA
    auto find_bin = [&](bool by_mass, double limit) {
      unsigned long long qc = pc, qm = pm;
#pragma unroll
      for (int e = 0; e < kMost; ++e) {
        if (owner && e < per && bm[e] != 0) {
          const double before = static_cast<double>(by_mass ? qm : qc);
          const double after = static_cast<double>(by_mass ? qm + bm[e] : qc + bc[e]);
          if (before < limit && !(after < limit)) {
            for (int r = 0; r < ctas; ++r) {
              cluster_st32(cluster_map(smem_u32(&sh.bin), r), bin0 + e);
              cluster_st64(cluster_map(smem_u32(&sh.before_count), r), qc);
              cluster_st64(cluster_map(smem_u32(&sh.before_mass), r), qm);
            }
          }
        }
        qc += bc[e];
        qm += bm[e];
      }
      sync_row(ctas);
    };
    auto shared64 = [&](const void* at) { return cluster_ld64(cluster_map(smem_u32(at), 0)); };
    // cutoff for `limit`; `mass` becomes the mass of what is kept
    auto find_cut = [&](bool by_mass, double limit, unsigned long long& mass, bool last) {
      find_bin(by_mass, limit);
      const int bin = sh.bin;
      const unsigned long long before_count = sh.before_count, before_mass = sh.before_mass;
      unsigned long long found;
      if (sort_cut(sh, s, base, top, rank, ctas, bin, by_mass, before_count, before_mass, limit,
                   last ? unit_mass : nullptr, units, w_min)) {
        summed = last;
        found = shared64(&sh.cut);
        mass = shared64(&sh.kept_mass);
      } else {
        found = search_cut(sh, s, base, top, ctas, slot, by_mass, limit);
        unsigned long long kc = 0, km = 0;
        s.each([&](float v, int i) {
          const uint32_t w = weight_of(v, top);
          if (w != 0 && order_key(v, base + i) >= found) km += w;
        });
        row_sums(sh, ctas, slot, kc, km);
        mass = km;
      }
      cut = max(cut, found);
    };
    unsigned long long mass = all_m;
    if (top_k > 0 && static_cast<unsigned long long>(top_k) < all_c)
      find_cut(false, static_cast<double>(top_k), mass, !by_p);
    if (by_p) {
      const double limit = static_cast<double>(top_p) * static_cast<double>(mass);
      sync_row(ctas);  // rank 0's results are read before they are written again
      find_cut(true, limit, mass, true);
    }
  }

  // ---- kept mass by units of consecutive elements, then the draw
  const float s_cut = cut != 0 ? key_value(cut) : -INFINITY;
  const int i_cut = cut != 0 ? static_cast<int>(0xffffffffu - static_cast<uint32_t>(cut)) - base
                             : 0x7fffffff;
  auto weight_kept = [&](float v, int i) -> uint32_t {
    const uint32_t w = weight_of(v, top);
    const bool in = (v > s_cut) | ((v == s_cut) & (i <= i_cut));
    return in & (w >= w_min) ? w : 0u;
  };
  // of four consecutive elements; zeros at once where none of the warp's is kept
  auto four_kept = [&](int i, uint32_t (&w)[4]) {
    const float4 v = s.four(i);
    const bool any = fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= s_cut;
    w[0] = w[1] = w[2] = w[3] = 0u;
    if (__any_sync(0xffffffffu, any)) {
      w[0] = weight_kept(v.x, i);
      w[1] = weight_kept(v.y, i + 1);
      w[2] = weight_kept(v.z, i + 2);
      w[3] = weight_kept(v.w, i + 3);
    }
  };
  if (!summed) {
    for (int u = warp; u < units; u += kWarps) {
      unsigned long long m = 0;
#pragma unroll
      for (int e = 0; e < kUnit / 128; ++e) {
        uint32_t w[4];
        four_kept(u * kUnit + e * 128 + lane * 4, w);
        m += static_cast<unsigned long long>(w[0]) + w[1];
        m += static_cast<unsigned long long>(w[2]) + w[3];
      }
      m = warp_sum64(m);
      if (lane == 0) unit_mass[u] = m;
    }
  }
  __syncthreads();
  if (warp == 0) {
    unsigned long long mine = 0;
    for (int u = lane; u < units; u += 32) mine += unit_mass[u];
    mine = warp_sum64(mine);
    if (lane == 0) sh.sum[slot][0] = mine;
  }
  sync_row(ctas);
  if (warp == 0) {
    unsigned long long before = 0, total = 0, sums[8];
    cluster_gather64(&sh.sum[slot][0], ctas, sums);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r < rank) before += sums[r];
      total += sums[r];
    }
    const unsigned long long own_mass = sh.sum[slot][0];
    const unsigned long long target = target_of(p.uniform[row], total);
    if (target >= before && target < before + own_mass) {  // the token is in this slice
      for (int u0 = 0; u0 < units; u0 += 32) {
        const unsigned long long m = u0 + lane < units ? unit_mass[u0 + lane] : 0;
        unsigned long long run = warp_scan64(m);
        const unsigned past = __ballot_sync(0xffffffffu, before + run > target);
        if (past == 0) {
          before += __shfl_sync(0xffffffffu, run, 31);
          continue;
        }
        const int at = __ffs(past) - 1;
        before += __shfl_sync(0xffffffffu, run - m, at);
        // the unit's elements in order, 128 at a time, four per lane
        for (int e = 0; e < kUnit / 128; ++e) {
          const int i0 = (u0 + at) * kUnit + e * 128 + lane * 4;
          uint32_t w[4];
          four_kept(i0, w);
          const unsigned long long mine4 =
              static_cast<unsigned long long>(w[0]) + w[1] + (static_cast<unsigned long long>(w[2]) + w[3]);
          run = warp_scan64(mine4);
          const unsigned here = __ballot_sync(0xffffffffu, before + run > target);
          if (here == 0) {
            before += __shfl_sync(0xffffffffu, run, 31);
            continue;
          }
          if (lane == __ffs(here) - 1) {
            unsigned long long acc = before + run - mine4;
            int c = 0;
            while (c < 3 && acc + w[c] <= target) acc += w[c++];
            p.tokens[row] = base + i0 + c;
          }
          break;
        }
        break;
      }
    }
  }
  if (ctas > 1) cluster_sync_all();  // no CTA leaves while another reads its memory
}

template <typename T>
static cudaError_t sample_go(const SampleParams& p, cudaStream_t stream) {
  // CTAs per row: until three fit an SM by their shared memory (one's passes then
  // run under the others' barriers), and more while there are fewer CTAs than SMs and
  // slices of at least 2048 remain
  auto slice = [&](int c) { return ((p.vocab + c - 1) / c + 7) / 8 * 8; };
  auto bytes_of = [](size_t elems) {
    const size_t units = (elems + kUnit - 1) / kUnit;
    return sizeof(SampleShared) + (units + 1) / 2 * 16 + units * kUnit * sizeof(T);
  };
  auto need = [&](int c) { return bytes_of(slice(c)); };
  int ctas = 1;
  constexpr size_t kThirdOfSm = 75 * 1024;
  while (ctas < 8 && need(ctas) > kThirdOfSm) ctas *= 2;
  while (ctas < 8 && static_cast<int64_t>(p.rows) * ctas * 2 <= sm_count() &&
         p.vocab / (ctas * 2) >= 2048)
    ctas *= 2;
  const int chunk = slice(ctas);
  const size_t bytes = need(ctas);
  const int vec = (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0 &&
                  (p.stride * static_cast<int64_t>(sizeof(T))) % 16 == 0;
  // Three CTAs per SM (40 registers, some spilled) where their shared memory fits and
  // they need fewer rounds of the SMs than two do: 512 rows of 50280 bf16 logits take
  // 67 us against 73 (mixed filters), 44.5 against 51.6 (top-k 50); at 256 rows, two
  // rounds either way, 49 against 44 and 28.1 against 28.0; 512 rows of 131072 fp32, of
  // which three do not fit, 257 against 241.
  const int64_t all = static_cast<int64_t>(p.rows) * ctas;
  auto rounds = [&](int per_sm) {
    const int64_t at_once = static_cast<int64_t>(per_sm) * sm_count();
    return (all + at_once - 1) / at_once;
  };
  const int per_sm = bytes <= kThirdOfSm && rounds(3) < rounds(2) ? 3 : 2;
  auto fn = per_sm == 3 ? ss_sample_kernel<T, 3> : ss_sample_kernel<T, 2>;
  // The limit is the function's, shared by all host threads: the same in every call, the
  // most that any call of this form takes.
  const size_t most = per_sm == 3 ? kThirdOfSm : bytes_of(kSampleMaxSlice);
  const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(most));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.rows) * ctas, 1, 1);
  cfg.blockDim = dim3(kSampleThreads, 1, 1);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  // Over many rounds costly rows run better among cheap ones: mixed filters on 50280
  // bf16 logits, 256 rows (two rounds) 44 us in order of cost against 54, 1024 (five)
  // 125 against 137; fp32, 400 rows (four) 83 against 87, 1024 (ten) 198 against 189.
  const int by_cost = rounds(per_sm) > 1 && rounds(per_sm) <= 5 && p.rows <= kOrderRows &&
                      (p.temperature || p.top_k || p.top_p);
  return cudaLaunchKernelEx(&cfg, fn, p, chunk, vec, by_cost);
}

cudaError_t launch_sample(const SampleParams& p, int dtype, cudaStream_t stream) {
  return dtype == MSS_BF16 ? sample_go<__nv_bfloat16>(p, stream) : sample_go<float>(p, stream);
}

}  // namespace mss
