// dash_sample.cu -- the next token of a row of logits from a given random number, with
// temperature, top-k, top-p and min-p, or the distribution that it is drawn from.
//
// A cluster of CTAs takes a row; each CTA owns a contiguous slice of the vocabulary
// and each warp a contiguous part of the slice, so running sums follow the
// vocabulary's order.  The slice is kept in shared memory where it fits.
//
// The tokens in descending order, lowest index first among equals, are cut off at one
// place by all three filters.  It is found as a key (the logit as an ordered 32-bit
// number) and a number of tokens of that key, by a radix descent in three
// digits (11, 11 and 10 bits): histograms of counts (top-k) or of weights (top-p) in
// shared memory, added over the cluster, then a search for the digit in which the
// count or the share is reached.
//
// Weights exp((z - max) / t) are whole numbers of 2^-43 of the largest: sums do not
// depend on the order of adding, so atomics and any split give the same token.  They
// are made in 64-bit floating point: with 10^5 tokens of shares around 10^-5, errors of a 32-bit
// exponential alone would move the borders between tokens by a share of 10^-8 or more, which
// picks another token in one row of a thousand.
//
// The radix descent is what always works; most rows do not need it.  A small top_k is cut
// out of the tokens that reach the top_k-th largest of the groups' largest logits; a large
// one, and a share of all tokens, out of those in one of 2,048 linear bins.  Such a list
// (up to 2,048 tokens) lies in every CTA, is sorted there and decides alone; up to 128
// kept tokens are drawn from it, too.
//
// Measured (vocabulary 129,280, CUDA graph): one row 9 us greedy, 14 with top-k 50 and top-p,
// 15 unfiltered, 28 with top-k 1,000 or top-p 0.9 alone.  One row's time is that of code
// that runs once (half of the stalls are for instructions) and of four to seven cluster
// barriers of 0.8 us.  64 rows (fp32): 25 greedy, 40 unfiltered (the weights: 25 instructions
// each, 8 of them in 64 bits), 89 with top-p 0.9 (two atomics per token besides); memory
// takes 5.  In bf16, with four CTAs per row: 14, 37 and 87, and 16 with top-k 20.
#include <cooperative_groups.h>

#include "dash_common.cuh"
#include "dash_internal.h"

namespace cg = cooperative_groups;

namespace dash {

namespace {

constexpr int kMaxWarps = 16;
constexpr int kMaxCluster = 8;
constexpr int kBins = 2048;
constexpr int kList = 2048;                      // tokens that one CTA sorts out by itself
constexpr int kDraw = 128;                       // of which it draws one by itself
constexpr int kTable = 256;                      // 2^(j / 256)
// (the slice lies behind Shared, whose size is a multiple of its alignment)
constexpr int kSliceMost = 128 * 1024;           // bytes of a slice kept in shared memory
constexpr int kSliceTwo = 68 * 1024;             // the same with two CTAs on an SM
// With four, which Shared leaves 12 KB each: at 15 KB only three ran at once, and rows cut for four in two waves
// (70 rows of 60,000, bf16: greedy 18.8 us, top-p 0.9 74; left in global memory, 13.4 and 55; 72 of 32,000, fp32,
// where clusters of 8 do not fill every SM: 17.5 and 51, 19.5 and 55).
constexpr int kSliceMany = 12 * 1024;
// Up to so many rows a CTA has 512 threads (two on an SM, slices in shared memory), above it 256
// (four).  64 rows of 129,280 (fp32) with settings of their own 59 us, with 256 threads 78; with
// top-k 20 alone 37 and 30.  Distributions of 128 rows (bf16), top-k 50: 88 and 52.
constexpr int kFewRows = 64;

struct alignas(16) Shared {
  uint32_t lo[kBins], hi[kBins];                 // this CTA's histogram: counts (lo), or 64-bit weights
  union {
    uint64_t tot[kBins];                         // the cluster's
    uint64_t list[kList];                        // ~key << 32 | index: what may be kept
  };
  uint32_t bucket[kBins + 1];                    // of the list's sorting
  uint32_t n_own;
  uint32_t floor_key;
  double table[kTable];
  uint64_t warp_sum[kMaxWarps];
  uint32_t warp_cnt[2 * kMaxWarps];              // (512 threads: two groups per warp, 256: four)
  alignas(16) uint32_t top[kMaxCluster * 2 * kMaxWarps];     // the largest key of each group of lanes
  uint64_t cta_sum[kMaxCluster];
  uint32_t cta_cnt[kMaxCluster];
  uint64_t scan[kMaxWarps];
  uint64_t found_before, found_here;             // of the digit that was looked for
  uint32_t found;
  int32_t last;                                  // cutoff index, exchanged
};
static_assert(4 * (sizeof(Shared) + kSliceMany + 1024) <= 228 * 1024 && 2 * (sizeof(Shared) + kSliceTwo + 1024) <= 228 * 1024,
              "as many CTAs on an SM as their names say");

// -inf and NaN: 0 (out); otherwise in the order of the values, -0 as 0
__device__ __forceinline__ uint32_t key_of(float z) {
  z += 0.0f;
  if (!(z > -INFINITY)) return 0u;
  const uint32_t b = __float_as_uint(z);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// exp((z - top) / t) in units of 2^-43, relative error below 3e-12: with y = (z - top) / (t ln 2) * 256
// = 256 k + j + r, |r| <= 1, it is 2^k * 2^(j/256) * exp(r ln2 / 256), the last factor by its series
// (the term behind the cubic one is 2.2e-12).  `add` is rounded, too: 1.1e-16 * |top| / t, which passes that where
// |top| / t is above 3e4 (bf16 and fp16 logits are 7 t apart there or more, fp32 ones 0.0009 t, and above 1e9 nothing
// but the largest has a weight).  Eight 64-bit operations per weight; the largest logit has 1 exactly, an
// infinite one, too.
struct Weight {
  float top;                                     // largest logit
  double mul, add;                               // y = z * mul + add
  const double* table;                           // 2^(j/256) * 2^43
  static constexpr double kOne = 8796093022208.0;                                        // 2^43
  static constexpr double kShift = 6755399441055744.0;                                   // 1.5 * 2^52

  __device__ __forceinline__ Weight(float t, float temperature, const double* tab) : top(t), table(tab) {
    mul = 369.32993046757462271 / (double)temperature;                                   // 256 / ln 2
    add = -(double)t * mul;
  }
  // a 32-bit number as a 64-bit one, without the conversion unit (0 becomes 2^-127)
  static __device__ __forceinline__ double wide(float z) {
    const uint32_t b = __float_as_uint(z);
    return __hiloint2double((int)((((b & 0x7fffffffu) >> 3) + 0x38000000u) | (b & 0x80000000u)), (int)(b << 29));
  }
  // (without branches, so that the chains of several weights run side by side)
  __device__ __forceinline__ double e(float z) const {
    const double w = wide(z), t = fma(w, mul, add + kShift);
    const int n = __double2loint(t);
    const double r = fma(w, mul, add - (t - kShift));
    double p = fma(r, 3.3083026805413711e-9, 3.6655755969101061e-6);                     // (ln2/256)^3 / 6, ^2 / 2
    p = fma(p, r, 2.7076061740622863e-3);                                                // ln 2 / 256
    p = fma(p, r, 1.0);
    const double s = table[n & (kTable - 1)];
    p *= __hiloint2double(__double2hiint(s) + (n >> 8) * (1 << 20), __double2loint(s));
    // below 2^-44 nothing; further down the whole part does not fit
    return z == top ? kOne : (z - top) * (float)mul > -44.0f * 256.0f ? p : 0.0;
  }
  // rounded to whole units
  static __device__ __forceinline__ uint64_t whole(double e) {
    return (uint64_t)__double_as_longlong(e + 4503599627370496.0) & 0xfffffffffffffull;  // 2^52
  }
  __device__ __forceinline__ uint64_t units(float z) const { return whole(e(z)); }
};

// a row's slice: in shared memory, or in global memory where it is too long
template <typename T, int E>
struct Slice {
  const T* kept;                                 // shared memory or null
  const T* row;                                  // the slice's first element in global memory
  int have;                                      // elements of the row in the slice (may be <= 0)
  bool vec;
  // elements at .. at + E - 1 of the slice as they are; behind its end -inf
  __device__ __forceinline__ uint4 raw(int at) const { return kept ? *reinterpret_cast<const uint4*>(kept + at) : global(at); }
  __device__ __forceinline__ uint4 global(int at) const {
    if (vec && at + E <= have) return *reinterpret_cast<const uint4*>(row + at);
    union {
      uint4 v;
      T t[E];
    } u;
#pragma unroll
    for (int e = 0; e < E; ++e) u.t[e] = at + e < have ? row[at + e] : (T)-INFINITY;
    return u.v;
  }
  // half of them
  static constexpr int H = E / 2;
  static __device__ __forceinline__ void half(uint32_t x, uint32_t y, float (&z)[H]) {
    if constexpr (E == 4) {
      z[0] = __uint_as_float(x), z[1] = __uint_as_float(y);
    } else {
      const float2 a = unpack2(x, (T*)nullptr), b = unpack2(y, (T*)nullptr);
      z[0] = a.x, z[1] = a.y, z[2] = b.x, z[3] = b.y;
    }
  }
  __device__ __forceinline__ void read(int at, float (&z)[E]) const {
    const uint4 v = raw(at);
    float a[H], b[H];
    half(v.x, v.y, a);
    half(v.z, v.w, b);
#pragma unroll
    for (int e = 0; e < H; ++e) z[e] = a[e], z[H + e] = b[e];
  }
};

// adds w to the 64-bit number in (lo, hi)
__device__ __forceinline__ void add64(uint32_t* lo, uint32_t* hi, uint64_t w) {
  const uint32_t l = (uint32_t)w;
  const uint32_t old = atomicAdd(lo, l);
  const uint32_t h = (uint32_t)(w >> 32) + (old + l < old ? 1u : 0u);
  if (h) atomicAdd(hi, h);
}

// the cluster's histogram into everybody's `tot`
template <int kThreads>
__device__ void total_of(Shared& S, cg::cluster_group& cl, int C, int rank, bool counts) {
  const int tid = threadIdx.x;
  cl.sync();
  const int per = kBins / C;
  for (int i = tid; i < per; i += kThreads) {
    const int b = rank * per + i;
    uint64_t s = 0;
    for (int c = 0; c < C; ++c) {
      const Shared* o = cl.map_shared_rank(&S, c);
      s += counts ? (uint64_t)o->lo[b] : ((uint64_t)o->hi[b] << 32) + o->lo[b];
    }
    for (int c = 0; c < C; ++c) cl.map_shared_rank(&S, c)->tot[b] = s;
  }
  cl.sync();
}

// The largest digit d whose bins above it hold less than `want` in sum, and those down to d
// at least `want`: S.found, with the sum above it and its own.
template <int kThreads>
__device__ void digit_of(Shared& S, uint64_t want) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int PER = kBins / kThreads;
  // thread t: PER bins from PER * t down, counted from the top
  uint64_t v[PER], own = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    v[i] = S.tot[kBins - 1 - (tid * PER + i)];
    own += v[i];
  }
  uint64_t incl = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) S.scan[warp] = incl;
  __syncthreads();
  uint64_t before = incl - own;
  for (int w = 0; w < warp; ++w) before += S.scan[w];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (before < want && before + v[i] >= want) {
      S.found = kBins - 1 - (tid * PER + i);
      S.found_before = before;
      S.found_here = v[i];
    }
    before += v[i];
  }
  __syncthreads();
}

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) sample_kernel(const DashSampleArgs a, int chunk, int keep_slice) {
  constexpr int E = 16 / sizeof(T), kWarps = kThreads / 32;
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& S = *reinterpret_cast<Shared*>(raw);
  T* kept = reinterpret_cast<T*>(raw + sizeof(Shared));
  cg::cluster_group cl = cg::this_cluster();
  const int C = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  auto started = cl.barrier_arrive();            // no CTA is written into before it has started
  const int row = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int slice = chunk * kWarps, first = rank * slice;

  const float temp = a.temperature ? a.temperature[row] : a.temperature_all;
  const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_all, 
              min_p = fminf(a.min_p ? a.min_p[row] : a.min_p_all, 1.0f);

  Slice<T, E> sl;
  sl.row = static_cast<const T*>(a.logits) + (int64_t)row * a.logits_stride + first;
  sl.have = a.vocab - first;
  sl.kept = nullptr;
  sl.vec = (reinterpret_cast<uintptr_t>(sl.row) & 15) == 0;

  if (tid < kTable) S.table[tid] = exp2(43.0 + (double)tid / kTable);

  // ---- the largest logit; the slice into shared memory ----
  const int w0 = warp * chunk + lane * E, w1 = (warp + 1) * chunk;
  if (keep_slice) {
    for (int at = w0; at < w1; at += 32 * E) {   // all on their way at once
      if (sl.vec && at + E <= sl.have) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(kept + at)), "l"(sl.row + at) : "memory");
      } else {
        *reinterpret_cast<uint4*>(kept + at) = sl.global(at);
      }
    }
    asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
    sl.kept = kept;                              // (a thread reads what it has written)
  }
  constexpr int GROUP = kThreads / 32;           // lanes: 32 groups in a CTA
  float most = -INFINITY;                        // (fmaxf leaves NaN out)
#pragma unroll 4
  for (int at = w0; at < w1; at += 32 * E) {
    float z[E];
    sl.read(at, z);
#pragma unroll
    for (int e = 0; e < E; ++e) most = fmaxf(most, z[e]);
  }
  uint32_t top = key_of(most);
#pragma unroll
  for (int o = GROUP / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane % GROUP == 0) S.warp_cnt[tid / GROUP] = top;
  cl.barrier_wait(std::move(started));
  __syncthreads();
  constexpr int OWN = kThreads / GROUP;
  const int parts = C * OWN;
  for (int i = tid; i < parts; i += kThreads) cl.map_shared_rank(&S, i / OWN)->top[rank * OWN + i % OWN] = S.warp_cnt[i % OWN];
  cl.sync();
  top = 0;
  for (int i = lane; i < parts; i += 32) top = max(top, S.top[i]);
  top = __reduce_max_sync(0xffffffffu, top);

  const Weight wt(value_of(top), temp, S.table);

  bool counted = false;                          // the histogram has been used
  // kept: key > cut, or key == cut and one of the first `ties` tokens of that key
  uint32_t cut = 1u, ties = 0xffffffffu, equals = 0;
  // The slice's elements, as f(index in the slice, H logits): two words of four at a time,
  // as with few rows most of the time goes into fetching instructions, which a loop saves
  constexpr int H = Slice<T, E>::H;
  const auto halves = [&](auto&& f) {
#pragma unroll 1
    for (int at = w0; at < w1; at += 32 * E) {
      uint4 v = sl.raw(at);
#pragma unroll 1
      for (int h = 0; h < E; h += H) {
        float z[H];
        Slice<T, E>::half(v.x, v.y, z);
        f(at + h, z);
        v.x = v.z, v.y = v.w;
      }
    }
  };
  const auto each = [&](auto&& f) {
    halves([&](int at, const float (&z)[H]) {
#pragma unroll
      for (int e = 0; e < H; ++e) f(at + e, z[e]);
    });
  };
  const auto clear = [&] {
    for (int i = tid; i < kBins; i += kThreads) S.lo[i] = S.hi[i] = 0;
    counted = true;
    __syncthreads();
  };

  // Tokens that `in` holds for into every CTA's list, in any order; their number
  const auto gather = [&](auto&& in) {
    if (counted) cl.sync();                      // nobody reads `tot` any more
    // this CTA's own first (on the histogram), then every CTA's behind those of the CTAs before it
    uint64_t* own = reinterpret_cast<uint64_t*>(S.lo);
    if (tid == 0) S.n_own = 0;
    __syncthreads();
    each([&](int i, float z) {
      if (z > -INFINITY && in(z)) {
        const uint32_t place = atomicAdd(&S.n_own, 1u);
        if (place < kList) own[place] = (uint64_t)~key_of(z) << 32 | (uint32_t)(first + i);
      }
    });
    __syncthreads();
    if (tid < C) cl.map_shared_rank(&S, tid)->cta_cnt[rank] = S.n_own;
    cl.sync();
    uint32_t start = 0, total = 0;
    for (int c = 0; c < C; ++c) {
      if (c < rank) start += S.cta_cnt[c];
      total += S.cta_cnt[c];
    }
    if (total <= kList)
      for (int c = 0; c < C; ++c) {
        uint64_t* to = cl.map_shared_rank(&S, c)->list + start;
        for (uint32_t i = tid; i < S.n_own; i += kThreads) to[i] = own[i];
      }
    cl.sync();
    return total;
  };
  // The list's n tokens in descending order (lowest index first among equals), and the weights'
  // running sums in `cums` (on the histogram)
  uint64_t* sorted = S.list;
  uint64_t* cums = reinterpret_cast<uint64_t*>(S.lo);
  const auto sort = [&](int n) {
    constexpr int PER = kList / kThreads;
    if (n <= 128) {
      // each one's place is the number before it
      const uint64_t v = tid < n ? S.list[tid] : ~0ull;
      int place = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) place += S.list[j] < v;
      __syncthreads();
      if (tid < n) sorted[place] = v;
    } else {
      // By buckets between the largest logit and the list's least (monotone), then by place
      // within the bucket.  (1,100 tokens: comparing all with all takes 20 us, a bitonic
      // network 17; it is what remains for many equal ones.)
      uint64_t* dealt = reinterpret_cast<uint64_t*>(S.lo);
      uint32_t far = 0;                          // ~key
      for (int i = tid; i < n; i += kThreads) far = max(far, (uint32_t)(S.list[i] >> 32));
      far = __reduce_max_sync(0xffffffffu, far);
      if (lane == 0) S.warp_cnt[warp] = far;
      for (int i = tid; i <= kBins; i += kThreads) S.bucket[i] = 0;
      __syncthreads();
      for (int w = 0; w < kWarps; ++w) far = max(far, S.warp_cnt[w]);
      const float t = value_of(top), step = (float)(kBins - 1) / (t - value_of(~far));
      const auto of = [&](uint64_t v) { return min(kBins - 1, (int)((t - value_of(~(uint32_t)(v >> 32))) * step)); };
      for (int i = tid; i < n; i += kThreads) atomicAdd(&S.bucket[of(S.list[i])], 1u);
      __syncthreads();
      constexpr int EACH = kBins / kThreads;
      uint32_t c[EACH], own = 0, crowd = 0;
#pragma unroll
      for (int i = 0; i < EACH; ++i) c[i] = S.bucket[tid * EACH + i], own += c[i], crowd = max(crowd, c[i]);
      uint32_t incl = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
      }
      if (lane == 31) S.warp_cnt[warp] = incl;
      const bool crowded = __syncthreads_or(crowd > 64);
      uint32_t run = incl - own;
      for (int w = 0; w < warp; ++w) run += S.warp_cnt[w];
#pragma unroll
      for (int i = 0; i < EACH; ++i) S.bucket[tid * EACH + i] = run, run += c[i];
      __syncthreads();
      if (!crowded) {
        // (a bucket's entry becomes its end, which is the next one's start)
        for (int i = tid; i < n; i += kThreads) {
          const uint64_t v = S.list[i];
          dealt[atomicAdd(&S.bucket[of(v)], 1u)] = v;
        }
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
          const uint64_t v = dealt[i];
          const int b = of(v), from = b ? (int)S.bucket[b - 1] : 0, to = (int)S.bucket[b];
          int place = from;
          for (int j = from; j < to; ++j) place += dealt[j] < v;
          sorted[place] = v;
        }
      } else {
        int m = 256;
        while (m < n) m *= 2;
        for (int i = n + tid; i < m; i += kThreads) sorted[i] = ~0ull;
#pragma unroll 1
        for (int size = 2; size <= m; size *= 2)
#pragma unroll 1
          for (int d = size / 2; d; d /= 2) {
            __syncthreads();
            for (int x = tid; x < m / 2; x += kThreads) {
              const int i = 2 * x - (x & (d - 1)), j = i + d;
              const uint64_t p = sorted[i], q = sorted[j];
              if ((p > q) == ((i & size) == 0)) sorted[i] = q, sorted[j] = p;
            }
          }
      }
    }
    __syncthreads();
    uint64_t w[PER], own = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int x = tid * PER + i;
      w[i] = x < n ? wt.units(value_of(~(uint32_t)(sorted[x] >> 32))) : 0;
      own += w[i];
    }
    uint64_t incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint64_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) S.scan[warp] = incl;
    __syncthreads();
    uint64_t run = incl - own;
    for (int x = 0; x < warp; ++x) run += S.scan[x];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      run += w[i];
      if (tid * PER + i < n) cums[tid * PER + i] = run;
    }
    __syncthreads();
  };
  // how many of the first n places have a sum before them that is below `want`
  const auto count_below = [&](int n, uint64_t want) {
    int mine = 0;
    for (int i = tid; i < n; i += kThreads) mine += (i ? cums[i - 1] : 0) < want;
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) S.warp_cnt[warp] = (uint32_t)mine;
    __syncthreads();
    int s = 0;
    for (int w = 0; w < kWarps; ++w) s += (int)S.warp_cnt[w];
    __syncthreads();
    return s;
  };

  const bool greedy = !(temp > 0.0f), k_on = top_k > 0 && top_k < a.vocab;
  int last = 0x7fffffff;                         // the row's index behind which equals of the cutoff are left out
  bool done = false;                             // cut and last are final
  int n_kept = -1;                               // of the sorted list, if it holds all kept ones
  const auto keep_first = [&](int k) {
    cut = ~(uint32_t)(sorted[k - 1] >> 32);
    ties = 1;
    last = (int)(uint32_t)sorted[k - 1];
    done = true;
  };
  // all that is kept is among the tokens that `in` holds for
  const auto by_list = [&](auto&& in) {
    const uint32_t n = gather(in);
    if (n > kList) return;
    sort((int)n);
    int k = k_on ? min((int)n, top_k) : (int)n;
    if (top_p < 1.0f) k = count_below(k, max((uint64_t)1, (uint64_t)ceil((double)fmaxf(top_p, 0.0f) * (double)cums[k - 1])));
    keep_first(k);
    if (k <= kDraw) n_kept = k;
  };
  // A bin per 1/50 of an exponent below the largest logit's (bins of the key's digits hold a
  // tenth of the vocabulary each: atomics on few addresses); monotone, like each of its steps
  const float top_f = value_of(top), scale = 50.0f / temp;
  const auto bin = [&](float z) { return kBins - 1 - min(kBins - 1, (int)((top_f - z) * scale)); };
  // the weights' total in `tot`
  const auto total_weight = [&] {
    uint64_t s = 0;
    for (int i = tid; i < kBins; i += kThreads) s += S.tot[i];
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) S.warp_sum[warp] = s;
    __syncthreads();
    s = 0;
    for (int w = 0; w < kWarps; ++w) s += S.warp_sum[w];
    return s;
  };
  const auto share_of = [&](uint64_t s) { return max((uint64_t)1, (uint64_t)ceil((double)fmaxf(top_p, 0.0f) * (double)s)); };

  if (top == 0) {
    cut = 0xffffffffu, ties = 0, done = true;    // nothing is left of the row
  } else if (greedy || top_k == 1) {
    const float best = value_of(top);
    const uint32_t n = gather([=](float z) { return z == best; });
    if (n <= kList) {
      sort((int)n);
      keep_first(1);
      n_kept = 1;
    } else {
      cut = top, ties = 1;
    }
  } else if (a.vocab <= kList) {
    by_list([](float) { return true; });
  } else {
    if (k_on && top_k <= parts / 4 * 3) {
      // At least top_k tokens are as large as the top_k-th largest of the groups' largest,
      // and not many more (1.4 times top_k at half their number).
      for (int i = tid; i < parts; i += kThreads) {
        const uint32_t mine = S.top[i];
        int before = 0;
#pragma unroll 4
        for (int j = 0; j < parts; j += 4) {
          const uint4 o = *reinterpret_cast<const uint4*>(S.top + j);
          before += (o.x > mine || (o.x == mine && j < i)) + (o.y > mine || (o.y == mine && j + 1 < i)) +
                    (o.z > mine || (o.z == mine && j + 2 < i)) + (o.w > mine || (o.w == mine && j + 3 < i));
        }
        if (before == top_k - 1) S.floor_key = mine;
      }
      __syncthreads();
      // (none, where a mask leaves most of them nothing)
      const float from = value_of(S.floor_key);
      if (S.floor_key) by_list([=](float z) { return z >= from; });
    }
    if (!done && k_on) {
      clear();
      each([&](int, float z) {
        if (z > -INFINITY) atomicAdd(&S.lo[bin(z)], 1u);
      });
      if (tid == 0) S.found = 0u, S.found_before = S.found_here = 0;      // fewer tokens than top_k: all
      total_of<kThreads>(S, cl, C, rank, true);
      digit_of<kThreads>(S, (uint64_t)top_k);
      const int from = (int)S.found;
      if (S.found_before + S.found_here <= kList) by_list([&](float z) { return bin(z) >= from; });
    } else if (!done && top_p < 1.0f) {
      clear();
      halves([&](int, const float (&z)[H]) {
        bool any = false;
#pragma unroll
        for (int e = 0; e < H; ++e) any |= z[e] > -INFINITY;
        if (!__any_sync(0xffffffffu, any)) return;
        uint64_t w[H];
#pragma unroll
        for (int e = 0; e < H; ++e) w[e] = wt.units(z[e]);
#pragma unroll
        for (int e = 0; e < H; ++e)
          if (z[e] > -INFINITY && w[e]) {
            const int b = bin(z[e]);
            add64(&S.lo[b], &S.hi[b], w[e]);
          }
      });
      total_of<kThreads>(S, cl, C, rank, false);
      const uint64_t want = share_of(total_weight());
      digit_of<kThreads>(S, want);
      const int at = (int)S.found;
      const uint64_t left = want - S.found_before;
      const uint32_t n = gather([&](float z) { return bin(z) == at; });
      if (n <= kList) {
        sort((int)n);
        keep_first(max(1, count_below((int)n, left)));
      }
    }
    // what no list could hold: by the key's digits
    if (!done && k_on) {
      uint64_t want = (uint64_t)top_k;
      uint32_t prefix = 0;
      bool all = false;
#pragma unroll 1
      for (int level = 0; level < 3 && !all; ++level) {
        const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
        clear();
        each([&](int, float z) {
          const uint32_t k = key_of(z);
          if (k && (level == 0 || k >> (shift + bits) == prefix)) atomicAdd(&S.lo[(k >> shift) & ((1u << bits) - 1)], 1u);
        });
        if (tid == 0) S.found = 0xffffffffu;
        total_of<kThreads>(S, cl, C, rank, true);
        digit_of<kThreads>(S, want);
        if (S.found == 0xffffffffu) {            // fewer tokens than top_k
          all = true;
        } else {
          want -= S.found_before;
          prefix = (prefix << bits) | S.found;
          equals = (uint32_t)S.found_here;
        }
      }
      if (!all && !done) cut = prefix, ties = (uint32_t)want;
    }
    if (!done && top_p < 1.0f) {
      // the weights' total over what top-k left, and the share of it
      uint64_t want = 0;
      uint32_t prefix = 0;
      const uint32_t floor_key = cut;
#pragma unroll 1
      for (int level = 0; level < 3; ++level) {
        const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, bits = level == 2 ? 10 : 11;
        clear();
        each([&](int, float z) {
          const uint32_t k = key_of(z);
          if (k >= floor_key && (level == 0 || k >> (shift + bits) == prefix)) {
            const uint64_t w = wt.units(z);
            const uint32_t b = (k >> shift) & ((1u << bits) - 1);
            if (w) add64(&S.lo[b], &S.hi[b], w);
          }
        });
        total_of<kThreads>(S, cl, C, rank, false);
        if (level == 0) {
          uint64_t s = total_weight();
          if (ties < equals) s -= (uint64_t)(equals - ties) * wt.units(value_of(cut));
          want = share_of(s);
        }
        digit_of<kThreads>(S, want);
        want -= S.found_before;
        prefix = (prefix << bits) | S.found;
      }
      const uint64_t w = wt.units(value_of(prefix));
      const uint64_t n = w ? (want + w - 1) / w : 1;
      const uint32_t had = prefix == cut ? ties : 0xffffffffu;
      cut = prefix;
      ties = n < had ? (uint32_t)n : had;
    }
  }

  // ---- the index behind which tokens of the cutoff's key are left out ----
  if (!done && ties != 0xffffffffu) {
    uint32_t n = 0;
    const float cut_z = value_of(cut);
    each([&](int, float z) { n += z == cut_z; });
    n = __reduce_add_sync(0xffffffffu, n);
    if (lane == 0) S.warp_cnt[warp] = n;
    __syncthreads();
    if (tid < C) {
      uint32_t s = 0;
      for (int w = 0; w < kWarps; ++w) s += S.warp_cnt[w];
      cl.map_shared_rank(&S, tid)->cta_cnt[rank] = s;
    }
    cl.sync();
    uint32_t before = 0, total = 0;
    for (int c = 0; c < C; ++c) {
      if (c < rank) before += S.cta_cnt[c];
      total += S.cta_cnt[c];
    }
    if (total > ties) {
      for (int w = 0; w < warp; ++w) before += S.warp_cnt[w];
      if (before < ties && before + S.warp_cnt[warp] >= ties) {
        // this warp holds the last one: by its 32 * E elements at a time
        for (int at = warp * chunk + lane * E; at - lane * E < (warp + 1) * chunk; at += 32 * E) {
          float z[E];
          sl.read(at, z);
          uint32_t own = 0;
#pragma unroll
          for (int e = 0; e < E; ++e) own += key_of(z[e]) == cut;
          uint32_t incl = own;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
          }
          uint32_t b = before + incl - own;
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (key_of(z[e]) == cut && ++b == ties)
              for (int c = 0; c < C; ++c) cl.map_shared_rank(&S, c)->last = first + at + e;
          before += __shfl_sync(0xffffffffu, incl, 31);
        }
      }
      cl.sync();
      last = S.last;
    }
  }
  // by the values: above the cutoff, or equal to it and not behind `last` (without a cutoff above -inf)
  const float cut_at = cut == 0xffffffffu ? INFINITY : cut == 1u ? -INFINITY : value_of(cut);
  const int cut_last = ties && cut != 1u && cut != 0xffffffffu ? (last == 0x7fffffff ? last : last - first) : -1;
  const auto is_kept = [&](int i, float z) { return z > cut_at || (z == cut_at && i <= cut_last); };
  // a greedy row has one token, of weight 1
  const double least = (double)min_p * Weight::kOne;
  const auto weight = [&](float z) -> double {
    const double e = wt.e(z);
    return greedy ? Weight::kOne : e >= least ? e : 0.0;
  };
  const auto put_probs = [&](uint64_t total) {
    const double inv = total ? 1.0 / (double)total : 0.0;
    float* out = a.probs + (int64_t)row * a.probs_stride + first;
    const bool ov = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    for (int at = warp * chunk + lane * E; at < (warp + 1) * chunk; at += 32 * E) {
      float z[E], p[E];
      sl.read(at, z);
      bool any = false;
#pragma unroll
      for (int e = 0; e < E; ++e) any |= is_kept(at + e, z[e]), p[e] = 0.0f;
      if (__any_sync(0xffffffffu, any)) {
#pragma unroll
        for (int e = 0; e < E; ++e) p[e] = is_kept(at + e, z[e]) ? (float)(weight(z[e]) * inv) : 0.0f;
      }
      if (ov && at + E <= sl.have) {
#pragma unroll
        for (int e = 0; e < E; e += 4)
          *reinterpret_cast<float4*>(out + at + e) = make_float4(p[e], p[e + 1], p[e + 2], p[e + 3]);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (at + e < sl.have) out[at + e] = p[e];
      }
    }
  };

  if (n_kept >= 0) {
    // the list has all: its weights again, without those that min_p leaves out, and their sum
    uint64_t sum = 0;
    for (int i = tid; i < n_kept; i += kThreads) {
      const uint64_t w = Weight::whole(weight(value_of(~(uint32_t)(sorted[i] >> 32))));
      cums[i] = w;
      sum += w;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) S.warp_sum[warp] = sum;
    __syncthreads();
    uint64_t total = 0;
    for (int w = 0; w < kWarps; ++w) total += S.warp_sum[w];
    if (a.probs) put_probs(total);
    if (a.tokens && rank == 0) {
      uint64_t at_sum = (uint64_t)((double)a.u[row] * (double)total);
      if (at_sum >= total) at_sum = total - 1;
      for (int i = tid; i < n_kept; i += kThreads) {
        const uint32_t mine = (uint32_t)sorted[i];
        uint64_t before = 0;
        for (int j = 0; j < n_kept; ++j)
          if ((uint32_t)sorted[j] < mine) before += cums[j];
        if (before <= at_sum && before + cums[i] > at_sum) a.tokens[row] = mine;
      }
    }
    return;
  }

  // ---- the kept sum ----
  uint64_t sum = 0;
  halves([&](int at, const float (&z)[H]) {
    bool any = false;
#pragma unroll
    for (int e = 0; e < H; ++e) any |= is_kept(at + e, z[e]);
    if (!__any_sync(0xffffffffu, any)) return;
    uint64_t w[H];
#pragma unroll
    for (int e = 0; e < H; ++e) w[e] = Weight::whole(weight(z[e]));
#pragma unroll
    for (int e = 0; e < H; ++e) sum += is_kept(at + e, z[e]) ? w[e] : 0;
  });
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) S.warp_sum[warp] = sum;
  __syncthreads();
  if (tid < C) {
    uint64_t s = 0;
    for (int w = 0; w < kWarps; ++w) s += S.warp_sum[w];
    cl.map_shared_rank(&S, tid)->cta_sum[rank] = s;
  }
  cl.sync();
  uint64_t before = 0, total = 0;
  for (int c = 0; c < C; ++c) {
    if (c < rank) before += S.cta_sum[c];
    total += S.cta_sum[c];
  }

  if (a.probs) put_probs(total);
  if (a.tokens) {
    if (total == 0) {
      if (rank == 0 && tid == 0) a.tokens[row] = -1;
      return;
    }
    // the first token whose running sum exceeds u * total
    uint64_t at_sum = (uint64_t)((double)a.u[row] * (double)total);
    if (at_sum >= total) at_sum = total - 1;
    for (int w = 0; w < warp; ++w) before += S.warp_sum[w];
    if (before <= at_sum && before + S.warp_sum[warp] > at_sum) {
      for (int at = warp * chunk + lane * E; at - lane * E < (warp + 1) * chunk; at += 32 * E) {
        float z[E];
        sl.read(at, z);
        uint64_t w[E], own = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          w[e] = is_kept(at + e, z[e]) ? Weight::whole(weight(z[e])) : 0;
          own += w[e];
        }
        uint64_t incl = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint64_t y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        uint64_t b = before + incl - own;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          if (b <= at_sum && b + w[e] > at_sum) a.tokens[row] = first + at + e;
          b += w[e];
        }
        before += __shfl_sync(0xffffffffu, incl, 31);
      }
    }
  }
}

template <typename T, int THREADS>
int launch_sample_t(const DashSampleArgs& a, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T), WARPS = THREADS / 32;
  // Eight CTAs per row, as far as that leaves each warp some work and, with many rows, all of
  // them run at once (of 512 threads: while two slices fit an SM.  64 rows, bf16, top-k 20: 34
  // us with 8 CTAs, 16 with 4; in fp32, where the slices of 4 do not fit, rows of several
  // settings 59 with 8, 79 with 4).
  int C = kMaxCluster;
  while (C > 1 && (int64_t)a.rows * C > (THREADS == 256 ? 4 : 2) * 148 &&
         (THREADS == 256 || (int64_t)a.vocab * sizeof(T) <= (int64_t)(C / 2) * kSliceTwo))
    C >>= 1;
  while (C > 1 && a.vocab <= (C / 2) * WARPS * 32 * E) C >>= 1;
  const int parts = C * WARPS;
  const int chunk = ((a.vocab + parts - 1) / parts + 32 * E - 1) / (32 * E) * (32 * E);
  const int64_t bytes = (int64_t)chunk * WARPS * sizeof(T);
  const int keep = bytes <= (THREADS == 512 ? kSliceMost : kSliceMany);
  static std::atomic<uint64_t> done{0};
  const cudaError_t set = once_per_device(done, [] {
    return cudaFuncSetAttribute(sample_kernel<T, THREADS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)sizeof(Shared) + kSliceMost);
  });
  if (set != cudaSuccess) return set_error(DASH_ERR_CUDA, "sample_kernel: %s", cudaGetErrorString(set));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * C);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = sizeof(Shared) + (keep ? (size_t)bytes : 0);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T, THREADS>, a, chunk, keep);
  if (e != cudaSuccess) return set_error(DASH_ERR_CUDA, "sample_kernel launch failed: %s", cudaGetErrorString(e));
  count_launch();
  return check_launch("sample_kernel");
}

template <typename T>
int launch_sample_rows(const DashSampleArgs& a, cudaStream_t st) {
  return a.rows <= kFewRows ? launch_sample_t<T, 512>(a, st) : launch_sample_t<T, 256>(a, st);
}

}  // namespace

int launch_sample(const DashSampleArgs& a, cudaStream_t st) {
  if (a.dtype == DASH_DTYPE_F32) return launch_sample_rows<float>(a, st);
  if (a.dtype == DASH_DTYPE_BF16) return launch_sample_rows<__nv_bfloat16>(a, st);
  return launch_sample_rows<__half>(a, st);
}

}  // namespace dash
