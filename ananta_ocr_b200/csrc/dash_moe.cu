// dash_moe.cu -- a whole mixture-of-experts layer for a few tokens.
//
// Bound by memory: the weights of the experts that the tokens picked cross the bus
// once, 3 * ffn * hidden numbers each, for a handful of tokens each.  So the weights
// are the M side of the products (128 rows of an expert's matrix per tile, straight from
// TMA into shared memory and from there into tcgen05.mma) and the tokens the N side (16 to
// 64 columns, gathered by row).
//
//   moe_route_kernel    scores to 64 bits, the picks and their weights
//   moe_ffn_kernel      gate_up: act = silu(g) * u of every pick and of the shared expert
//   moe_ffn_kernel      down: down * act, by tile of 128 rows and by part of the ffn
//   moe_combine_kernel  the weighted sum of the parts in a fixed order, and the residual
//
// Each kernel is launched while the one before it runs and waits for its results on the
// GPU: gate_up's CTAs bring a shared expert's weights into L2 while the router works, if
// they are few, and down's CTAs take the places of gate_up's as they end.  Each waits for all of the kernel before
// it before it reads what that one wrote: down takes the sorted picks from gate_up, which waited for the router.  (Reading
// the router's picks while gate_up's last tiles were under way, and filling the rings with weights, took 1
// to 2.5 us less, but nothing promises that what the kernel before last has written is visible then.)
//
// Measured (64 experts of 896, 6 picked, 2 shared, hidden 1,280, bf16; CUDA graph): 27.6 / 56.5 / 90.2 us
// for 1 / 8 / 64 tokens, where the weights at the copy rate take 8.4 / 38.7 / 69.2.  While gate_up
// and down stream, they read at 7.1 TB/s; the rest is the order of things.  One token, by the
// global timer: scores 2.5 us, picks 3.8, sorted by expert in every CTA 6.4, the first
// weights 8.2, the last 15; then down, and the sum.
//
// act is kept as the sum of two 16-bit numbers, each multiplied by itself: the products
// are far from bound by the tensor cores, and the layer's error stays the rounding of its output
// (with one number it would be 0.0020 instead of 0.0017 of the output, bf16).  In fp16 the second one is kept
// 2^11 times as large: what the first leaves is at most 2^-12 of it, and below 2^-14 that type has multiples
// of 2^-24 only.
#include <cudaTypedefs.h>

#include <algorithm>
#include <cmath>

#include "dash_common.cuh"
#include "dash_internal.h"

namespace dash {

namespace {

// 4 epilogue warps, and one each that issues the weights' loads, the products and the tokens'
// loads: with one warp for both kinds of loads and one CTA per SM, issuing was the limit
// (64 tokens: 148 us; 20 us less without the tokens' loads, 17 less without products).
constexpr int kThreads = 224;
constexpr int kTile = 128;                  // weight rows of a tile
constexpr int kStep = 64;                   // k elements of a stage (128 bytes)
constexpr int kABytes = kTile * 128;
constexpr int kMaxStages = 8;
constexpr int kExchange = 2 * 16 * 64 * 4;  // gate_up: accumulators that change warps
// Three CTAs per SM.  Two with 113 KB each are as fast at 64 tokens (89 us) and slower at 8
// (56); prefetching stages beyond the ring into L2 was slower (104 us with 4 of them, 131 with 16).
constexpr int kSmem = 75 * 1024;
// Every place of every SM: with fewer CTAs than places some SMs get three and some none, as
// they are dealt out while the kernel before is still there (131 of 148 SMs had work).
constexpr int kCtas = 3 * 148;

// How a call is cut up: the same for equal sizes, whatever the tokens pick, so that a
// token's sums do not depend on the other tokens.
struct Cut {
  int nt;                                   // tokens of a tile at most
  int rows;                                 // gate_up: gate rows of a tile (and as many up rows), 32 .. 64
  int ksteps, kshared;                      // 64-element steps of a part of down's k
  int splits, shared_splits;                // such parts of ffn and of shared_ffn
};

struct Buffers {                            // workspace
  size_t act, sact, part;                   // act: [2][picks by expert][ffn], both parts of the numbers
  size_t sorted;                            // the picks by expert, as they lie in shared memory (Layout)
  size_t bytes;
};

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

Cut cut_of(const DashMoeArgs& a) {
  Cut c;
  c.nt = a.tokens <= 16 ? 16 : 32;
  // gate_up's tiles: as high as lets the CTAs finish together.  `groups`: of tokens of one
  // expert, with a router that picks evenly, and some more.
  const double active = a.experts * (1.0 - std::pow(1.0 - (double)a.topk / a.experts, a.tokens));
  const double groups = 1.05 * std::max(active, (double)a.tokens * a.topk / c.nt);
  const int chunks = ceil_div(a.tokens, c.nt);
  double best = 0.0;
  for (int rows = 64; rows >= 32; rows -= 8) {
    const double tiles = groups * ceil_div(a.ffn, rows) + chunks * ceil_div(a.shared_ffn, rows);
    const double time = std::ceil(tiles / kCtas) * rows;
    if (rows == 64 || time < best) best = time, c.rows = rows;
  }
  // parts of down's k: as long as lets the CTAs finish together (a part costs two steps
  // more than its own), but seven steps at least: more items than CTAs that start beside
  // gate_up's last ones wait for places (one token: 26.8 us with parts of 4, 25.9 with 7)
  const int tiles = ceil_div(a.hidden, kTile), steps = ceil_div(a.ffn, kStep), sh = ceil_div(a.shared_ffn, kStep);
  int k = std::max(steps, 1);
  for (int n = 1; n <= steps; ++n) {
    const int len = ceil_div(steps, n);
    if (len < std::min(7, steps)) break;
    const auto time = [&](int l) {
      return std::ceil((groups * ceil_div(steps, l) + chunks * ceil_div(sh, l)) * tiles / kCtas) * (l + 2);
    };
    if (time(len) < time(k)) k = len;
  }
  c.ksteps = k;
  c.splits = ceil_div(steps, k);
  c.kshared = k;
  c.shared_splits = ceil_div(sh, k);
  return c;
}

// groups of up to nt picks of one expert
__host__ __device__ constexpr int most_units(int nt, int experts, int picks) {
  return picks < experts + picks / nt ? picks : experts + picks / nt;
}
// the sorted picks: each expert's start in the list (one more is the end, and behind it the number of groups), the
// groups, the list
__host__ __device__ constexpr int up16(int n) { return (n + 15) & ~15; }
__host__ __device__ constexpr int base_bytes(int experts) { return up16((experts + 2) * 4); }
__host__ __device__ constexpr int units_bytes(int nt, int experts, int picks) { return up16(most_units(nt, experts, picks) * 4); }
__host__ __device__ constexpr int sorted_bytes(int nt, int experts, int picks) {
  return base_bytes(experts) + units_bytes(nt, experts, picks) + up16(picks * 2);
}

Buffers buffers_of(const DashMoeArgs& a, const Cut& c) {
  Buffers b;
  size_t at = 0;
  const auto take = [&](size_t n) {
    const size_t here = at;
    at += (n + 255) & ~(size_t)255;
    return here;
  };
  const size_t picks = (size_t)a.tokens * a.topk;
  b.act = take(2 * picks * a.ffn * 2);
  b.sact = take(2 * (size_t)a.tokens * a.shared_ffn * 2);
  b.part = take((picks * c.splits + (size_t)a.tokens * c.shared_splits) * a.hidden * 4);
  b.sorted = take(sorted_bytes(c.nt, a.experts, (int)picks));
  b.bytes = at + 256;
  return b;
}

__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------------------
// router: a cluster of CTAs per token, a warp per expert
// ---------------------------------------------------------------------------
constexpr int kRouteThreads = 256;

// lane's share of x . gate[at ..], 8 elements per 256; U such pieces in flight.  A 16-bit gate's products are
// made in fp32, or (WIDE) in 64 bits like those of an fp32 one
template <typename T, bool F32, int U, bool WIDE = F32>
__device__ __forceinline__ double dot64(const T* x, const void* gate, int64_t at, int n, int lane) {
  double s[4] = {};                            // (sums of 64-bit numbers take 20 cycles each)
  for (int i0 = lane * 8; i0 < n; i0 += 256 * U) {
    uint4 xv[U], gv[U], hv[F32 ? U : 1];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + 256 * u;
      xv[u] = gv[u] = hv[F32 ? u : 0] = make_uint4(0, 0, 0, 0);
      if (i < n) {
        xv[u] = *reinterpret_cast<const uint4*>(x + i);
        const uint4* g = reinterpret_cast<const uint4*>(static_cast<const char*>(gate) + (at + i) * (F32 ? 4 : 2));
        gv[u] = g[0];
        if (F32) hv[F32 ? u : 0] = g[1];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t xw[4] = {xv[u].x, xv[u].y, xv[u].z, xv[u].w};
      const uint32_t gw[8] = {gv[u].x, gv[u].y, gv[u].z, gv[u].w, hv[F32 ? u : 0].x, hv[F32 ? u : 0].y, hv[F32 ? u : 0].z, hv[F32 ? u : 0].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack2(xw[j], (T*)nullptr);
        if (F32) {
          s[j] = fma((double)f.x, (double)__uint_as_float(gw[2 * j]), s[j]);
          s[j] = fma((double)f.y, (double)__uint_as_float(gw[2 * j + 1]), s[j]);
        } else {
          const float2 w = unpack2(gw[j], (T*)nullptr);
          if (WIDE) {
            s[j] = fma((double)f.x, (double)w.x, s[j]);
            s[j] = fma((double)f.y, (double)w.y, s[j]);
          } else {
            s[j] += (double)(f.x * w.x);
            s[j] += (double)(f.y * w.y);
          }
        }
      }
    }
  }
  double sum = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return sum;
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t n;
  asm("mov.u32 %0, %cluster_nctaid.x;" : "=r"(n));
  return n;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t n;
  asm("mov.u32 %0, %cluster_ctarank;" : "=r"(n));
  return n;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename T, bool F32>
__global__ void __launch_bounds__(kRouteThreads, 4) moe_route_kernel(const DashMoeArgs a) {
  __shared__ double score[kMoeMaxExperts];
  __shared__ double red[kRouteThreads / 32], best[kMoeMaxTopk];
  __shared__ int id[kMoeMaxTopk];
  launch_next();
  const int C = (int)cluster_size(), rank = (int)cluster_rank();
  const int t = blockIdx.x / C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster_arrive();
  const T* x = static_cast<const T*>(a.x) + t * a.x_stride;
  bool waited = false;
  for (int e = rank * 8 + warp; e - warp < a.experts; e += 8 * C) {
    double s = 0.0;
    if (e < a.experts) {
      s = dot64<T, F32, F32 ? 2 : 5>(x, a.gate, (int64_t)e * a.hidden, a.hidden, lane);
      // Products of two 16-bit numbers have digits for fp32, but those of bf16 can leave its range: above
      // it the sum is no number, and below 2^-126 each is off by 2^-150 at most, which a sum of 2^16
      // products above 2^-80 does not show in 53 bits.  (All in 64 bits: 64 tokens 1.5 us more.)
      if (!F32 && DType<T>::fmt == 1 && !(fabs(s) >= 0x1p-80 && fabs(s) < INFINITY))
        s = dot64<T, F32, 2, true>(x, a.gate, (int64_t)e * a.hidden, a.hidden, lane);
    }
    if (!waited) cluster_wait();                 // the first CTA has started
    waited = true;
    if (e < a.experts && lane == 0) {
      uint32_t to;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(score + e)), "r"(0));
      asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(s) : "memory");
    }
  }
  if (!waited) cluster_wait();
  cluster_arrive();
  cluster_wait();
  if (rank) return;
  // an expert's place among all decides: `share` threads count the experts before it
  const auto value = [&](int e) { return score[e] != score[e] ? -INFINITY : score[e]; };      // NaN: the smallest
  int share = 1;
  while (share < 32 && a.experts * share * 2 <= kRouteThreads) share *= 2;
  for (int x0 = tid / share; x0 - tid / share < a.experts; x0 += kRouteThreads / share) {
    int before = 0;
    if (x0 < a.experts) {
      const double m = value(x0);
      for (int j = tid % share; j < a.experts; j += share) {
        const double v = value(j);
        before += v > m || (v == m && j < x0);
      }
    }
    for (int o = 1; o < share; o <<= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (x0 < a.experts && tid % share == 0 && before < a.topk) id[before] = x0;
  }
  __syncthreads();
  const double top = value(id[0]);
  const auto weight = [&](int e) { return score[e] == top ? 1.0 : exp(score[e] - top); };
  // (a NaN score makes the sum NaN)
  double sum = tid < a.experts ? weight(tid) : 0.0;
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) red[warp] = sum;
  if (tid < a.topk) best[tid] = weight(id[tid]);
  __syncthreads();
  if (tid < a.topk) {
    double total = 0.0, picked = 0.0;
    for (int w = 0; w < kRouteThreads / 32; ++w) total += red[w];
    for (int j = 0; j < a.topk; ++j) picked += best[j];
    a.ids[(int64_t)t * a.topk + tid] = id[tid];
    a.weights[(int64_t)t * a.topk + tid] = (float)(best[tid] / (a.renorm ? picked + 0.0 * total : total) * (double)a.scale);
  }
}

// ---------------------------------------------------------------------------
// gate_up and down
// ---------------------------------------------------------------------------
struct Maps {
  CUtensorMap w, sw;                        // the experts' matrices, the shared one
  CUtensorMap b, sb;                        // gate_up: x by rows, x by 16 rows; down: act, the shared act
};

struct Layout {                             // dynamic shared memory behind the ring
  int stage, stages, bars, exchange, base, units, list, bytes;
};

template <bool DOWN>
__host__ __device__ inline Layout layout_of(int nt, int rows, int experts, int picks) {
  Layout l;
  const int exchange = DOWN ? 0 : kExchange, sorted = sorted_bytes(nt, experts, picks);
  l.stage = (DOWN ? kABytes : 2 * rows * 128) + nt * 128 * (DOWN ? 2 : 1);
  l.stages = (kSmem - 1024 - 512 - exchange - sorted) / l.stage;
  if (l.stages > kMaxStages) l.stages = kMaxStages;
  l.bars = l.stages * l.stage;
  l.exchange = l.bars + 512;
  l.base = l.exchange + exchange;
  l.units = l.base + base_bytes(experts);
  l.list = l.units + units_bytes(nt, experts, picks);
  l.bytes = l.base + sorted + 1024;
  return l;
}

// One tile of work: n tokens from `first` (of the expert's list, or the tokens
// themselves) times rows mt * 128 .. of a matrix, k steps k0 .. k1
struct Item {
  bool shared;
  int expert, first, n, mt, part, k0, k1;
};

template <bool DOWN>
struct Tiles {
  const int* base;                          // per expert: its picks' start in the list
  const uint32_t* units;                    // groups: expert << 16 | first pick
  int nt, tokens, mt, smt, k, sk, kpart, parts, sparts, shared, total;

  __device__ __forceinline__ Item at(int i) const {
    Item it;
    it.shared = i < shared;
    if (!it.shared) i -= shared;
    const int tiles = it.shared ? smt : mt, np = it.shared ? sparts : parts;
    it.mt = i % tiles;
    i /= tiles;
    it.part = i % np;
    i /= np;
    if (it.shared) {
      it.expert = 0;
      it.first = i * nt;
      it.n = min(nt, tokens - it.first);
    } else {
      const uint32_t u = units[i];
      it.expert = (int)(u >> 16);
      it.first = (int)(u & 0xffffu);
      it.n = min(nt, base[it.expert + 1] - it.first);
    }
    it.k0 = it.part * kpart;
    it.k1 = min(it.shared ? sk : k, it.k0 + kpart);
    return it;
  }
};

// 32 lanes x 16 consecutive 32-bit columns
__device__ __forceinline__ void tmem_ld16f(uint32_t taddr, float (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15])
      : "r"(taddr));
}

template <typename T>
constexpr float kLow = DType<T>::fmt == 0 ? 2048.0f : 1.0f;          // of act's second numbers

__device__ __forceinline__ float silu(float g) { return g / (1.0f + expf(-g)); }

// whether `ok` holds in all of the four epilogue warps (a barrier of theirs)
__device__ __forceinline__ bool all_warps(bool ok) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.and.pred q, 1, 128, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)ok)
      : "memory");
  return r != 0;
}

// (bounds of 256 threads: 80 registers, with which three CTAs fit each quarter of an SM)
template <typename T, bool DOWN>
__global__ void __launch_bounds__(256, 3) moe_ffn_kernel(const __grid_constant__ Maps maps, const DashMoeArgs a, const Cut cut,
                                                           const Buffers buf) {
  extern __shared__ __align__(1024) uint8_t raw[];
  uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  const int picks = a.tokens * a.topk;
  const Layout lay = layout_of<DOWN>(cut.nt, cut.rows, a.experts, picks);
  const int NS = lay.stages;
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + lay.bars);      // [stages] TMA -> MMA
  uint64_t* empty = full + kMaxStages;                              // [stages] MMA -> TMA
  uint64_t* acc_full = empty + kMaxStages;                          // [2] MMA -> epilogue
  uint64_t* acc_empty = acc_full + 2;                               // [2] epilogue -> MMA
  uint32_t* holder = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(holder + 1);
  int* base = reinterpret_cast<int*>(sm + lay.base);                // [experts + 1], the number of groups
  uint32_t* units = reinterpret_cast<uint32_t*>(sm + lay.units);    // groups of picks
  uint16_t* list = reinterpret_cast<uint16_t*>(sm + lay.list);      // picks, by expert

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  DeviceError* derr = a.device_error;
  const int cols = DOWN ? 2 * cut.nt : max(32, cut.nt);             // TMEM columns of an accumulator

  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + i, 2);                     // weights and tokens
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc_full + i, 1);
      mbar_init(acc_empty + i, 128);
    }
    *abort_flag = 0;
    mbar_init_fence();
  }
  if (warp == 5) {
    tmem_alloc(holder, 2 * cols);
    tmem_relinquish();
  }
  if (tid == 32) {
    prefetch_tmap(&maps.w);
    prefetch_tmap(&maps.b);
    prefetch_tmap(&maps.sb);
    prefetch_tmap(&maps.sw);
  }
  // The shared expert's weights into L2, while the router works.  14 MB of them (the layer above): 3 to 8 tokens 1 us
  // less.  50 MB: 1 token 47 us, without 44; 402 MB, more than L2 holds: 1 token 126 and 118, 64 tokens 284 and 263.
  constexpr int64_t kFetchMost = (int64_t)24 << 20;
  const int64_t bytes = (int64_t)a.shared_ffn * a.hidden * 2;
  if (!DOWN && 3 * bytes <= kFetchMost) {
    const int64_t piece = 4096;
    for (int64_t at = ((int64_t)tid * gridDim.x + blockIdx.x) * piece; at < 3 * bytes; at += (int64_t)gridDim.x * kThreads * piece) {
      const bool up = at < 2 * bytes;
      const char* p = up ? static_cast<const char*>(a.shared_gate_up) + at : static_cast<const char*>(a.shared_down) + (at - 2 * bytes);
      const int64_t n = min(piece, (up ? 2 * bytes : 3 * bytes) - at);
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"((uint32_t)n) : "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *holder;
  // Both wait here for the kernel before: gate_up for the router's picks, down for
  // the sorted picks and act.  (Nothing is read before this kernel's own wait: only what the kernel
  // directly before has written, or itself waited for and passed on, is sure to be there.)
  uint8_t* sorted = static_cast<uint8_t*>(a.workspace) + buf.sorted;
  const int sorted_end = sorted_bytes(cut.nt, a.experts, picks);
  if constexpr (DOWN) {
    wait_previous();
    launch_next();
    for (int i = tid * 16; i < sorted_end; i += kThreads * 16)
      *reinterpret_cast<uint4*>(sm + lay.base + i) = __ldcg(reinterpret_cast<const uint4*>(sorted + i));
  } else {
    // (in the ring, which is not in use yet)
    uint32_t* tokens = reinterpret_cast<uint32_t*>(sm);               // [experts][words]: who picked it
    const int words = ceil_div(a.tokens, 32);
    uint16_t* expert_of = reinterpret_cast<uint16_t*>(tokens + a.experts * words);
    // (once without the picks while it waits: code that runs for the first time waits for its own
    // instructions; one token 0.9 us less)
#pragma unroll 1
    for (int dry = 1; dry >= 0; --dry) {
      for (int i = tid; i < a.experts * words; i += kThreads) tokens[i] = 0;
      __syncthreads();
      if (!dry) {
        wait_previous();
        launch_next();
      }

      // ---- the picks by expert, in their order (every CTA has to cut an expert's picks into
      // the same groups): a bit per token and expert ----
      for (int p = tid; p < picks; p += kThreads) {
        const int e = dry ? 0 : __ldcg(a.ids + p), t = p / a.topk;
        expert_of[p] = (uint16_t)e;
        atomicOr(tokens + e * words + (t >> 5), 1u << (t & 31));
      }
      __syncthreads();
      if (warp == 0) {
        int run = 0, groups = 0;
        for (int e0 = 0; e0 < a.experts; e0 += 32) {
          const int e = e0 + lane;
          int n = 0;
          if (e < a.experts)
            for (int w = 0; w < words; ++w) n += __popc(tokens[e * words + w]);
          const int own = ceil_div(n, cut.nt);
          int both = n << 16 | own;                   // sums of both at once: picks < 2^13, groups < 2^13
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, both, o);
            if (lane >= o) both += y;
          }
          const int at = run + (both >> 16) - n, g = groups + (both & 0xffff) - own;
          if (e < a.experts) {
            base[e] = at;
            for (int i = 0; i < own; ++i) units[g + i] = (uint32_t)e << 16 | (uint32_t)(at + i * cut.nt);
          }
          both = __shfl_sync(0xffffffffu, both, 31);
          run += both >> 16;
          groups += both & 0xffff;
        }
        if (lane == 0) base[a.experts] = run, base[a.experts + 1] = groups;
      }
      __syncthreads();
      for (int p = tid; p < picks; p += kThreads) {
        const int e = expert_of[p], t = p / a.topk;
        int at = base[e] + __popc(tokens[e * words + (t >> 5)] & ((1u << (t & 31)) - 1));
        for (int w = 0; w < t >> 5; ++w) at += __popc(tokens[e * words + w]);
        list[at] = (uint16_t)p;
      }
      __syncthreads();
    }
    // for down: from the first CTA, as every CTA has the same
    if (blockIdx.x == 0)
      for (int i = tid * 16; i < sorted_end; i += kThreads * 16)
        *reinterpret_cast<uint4*>(sorted + i) = *reinterpret_cast<const uint4*>(sm + lay.base + i);
  }
  // the ring's next writer is the TMA unit
  fence_proxy_async_smem();
  __syncthreads();

  Tiles<DOWN> tiles;
  tiles.base = base;
  tiles.units = units;
  tiles.nt = cut.nt;
  tiles.tokens = a.tokens;
  tiles.mt = ceil_div(DOWN ? a.hidden : a.ffn, DOWN ? kTile : cut.rows);
  tiles.smt = a.shared_ffn ? ceil_div(DOWN ? a.hidden : a.shared_ffn, DOWN ? kTile : cut.rows) : 1;
  tiles.k = ceil_div(DOWN ? a.ffn : a.hidden, kStep);
  tiles.sk = ceil_div(DOWN ? a.shared_ffn : a.hidden, kStep);
  tiles.kpart = DOWN ? cut.ksteps : tiles.k;
  tiles.parts = DOWN ? cut.splits : 1;
  tiles.sparts = DOWN ? max(1, cut.shared_splits) : 1;
  tiles.shared = a.shared_ffn ? ceil_div(a.tokens, cut.nt) * tiles.smt * tiles.sparts : 0;
  tiles.total = tiles.shared + base[a.experts + 1] * tiles.mt * tiles.parts;

  const int a_bytes = DOWN ? kABytes : 2 * cut.rows * 128;
  if (warp == 4) {
    // =================== weights ===================
    if (lane == 0) {
      int st = 0, round = 0, s = 0;
      bool ok = true;
      for (int i = blockIdx.x; i < tiles.total && ok; i += gridDim.x) {
        const Item it = tiles.at(i);
        const CUtensorMap* m = it.shared ? &maps.sw : &maps.w;
        const int row = it.mt * (DOWN ? kTile : cut.rows);
        for (int k = it.k0; k < it.k1; ++k, ++s) {
          if (round && !mbar_wait(empty + st, (round - 1) & 1, abort_flag, derr, 90)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx(full + st, a_bytes);
          // gate_up: gate rows, then their up rows
          tma_load_4d(sm + st * lay.stage, m, full + st, k * kStep, row, DOWN ? it.expert : 0, DOWN ? 0 : it.expert);
          if (++st == NS) st = 0, ++round;
        }
      }
      // never leave with copies in flight
      for (int n = min(s, NS); n > 0; --n) {
        if (--st < 0) st = NS - 1, --round;
        volatile int no_abort = 0;
        mbar_wait(full + st, round & 1, &no_abort, nullptr, 91);
      }
    }
  } else if (warp == 6) {
    // =================== tokens ===================
    int st = 0, round = 0, s = 0;
    bool ok = true;
    if (DOWN) {
      asm volatile("fence.proxy.async;" ::: "memory");             // act is read by the TMA unit
      __syncwarp();
    }
    const bool gather = !DOWN && a.tokens > 16;
    for (int i = blockIdx.x; i < tiles.total && ok; i += gridDim.x) {
      const Item it = tiles.at(i);
      const int n16 = (it.n + 15) & ~15;
      int r[4] = {0, 0, 0, 0};
      if (gather && lane < n16 / 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = it.first + min(lane * 4 + j, it.n - 1);    // columns behind the last: its copies
          r[j] = it.shared ? at : list[at] / a.topk;
        }
      const CUtensorMap* m = DOWN ? (it.shared ? &maps.sb : &maps.b) : &maps.sb;
      for (int k = it.k0; k < it.k1; ++k, ++s) {
        if (round && !mbar_wait_warp(empty + st, (round - 1) & 1, abort_flag, derr, 92)) {
          ok = false;
          break;
        }
        uint8_t* dst = sm + st * lay.stage + a_bytes;
        if (lane == 0) mbar_arrive_expect_tx(full + st, (DOWN ? n16 * 2 : n16) * 128);
        __syncwarp();
        if (DOWN) {
          // 16 rows of the first parts, then of the second
          if (lane < n16 / 16) tma_load_4d(dst + lane * 4096, m, full + st, k * kStep, it.first + lane * 16, 0, 0);
        } else if (gather) {
          if (lane < n16 / 4) tma_gather4(dst + lane * 512, &maps.b, full + st, k * kStep, r[0], r[1], r[2], r[3]);
        } else if (lane == 0) {
          tma_load_4d(dst, m, full + st, k * kStep, 0, 0, 0);        // all tokens
        }
        if (++st == NS) st = 0, ++round;
      }
    }
    for (int n = min(s, NS); n > 0; --n) {
      if (--st < 0) st = NS - 1, --round;
      volatile int no_abort = 0;
      mbar_wait_warp(full + st, round & 1, &no_abort, nullptr, 91);
    }
  } else if (warp == 5) {
    // =================== MMA ===================
    if (lane == 0) {
      int st = 0, round = 0, n_item = 0;
      bool ok = true;
      for (int i = blockIdx.x; i < tiles.total && ok; i += gridDim.x, ++n_item) {
        const Item it = tiles.at(i);
        const uint32_t n16 = (uint32_t)((it.n + 15) & ~15);
        const uint32_t idesc = make_idesc(DType<T>::fmt, 0, 0, kTile, DOWN ? 2 * n16 : n16);
        const int b = n_item & 1;
        if (n_item >= 2 && !mbar_wait(acc_empty + b, ((n_item >> 1) - 1) & 1, abort_flag, derr, 93)) break;
        tc_fence_after();
        for (int k = it.k0; k < it.k1; ++k) {
          if (!mbar_wait(full + st, round & 1, abort_flag, derr, 94)) {
            ok = false;
            break;
          }
          tc_fence_after();
          // (gate_up with narrow tiles: rows 64 and up are whatever lies behind, and nobody reads them)
          const uint32_t sA = smem_u32(sm + st * lay.stage), sB = sA + a_bytes;
          const uint64_t ad = sw128_desc(sA, 16, 1024), bd = sw128_desc(sB, 16, 1024);
#pragma unroll
          for (int kk = 0; kk < kStep / 16; ++kk) umma_ss(tmem + b * cols, ad + kk * 2, bd + kk * 2, idesc, k > it.k0 || kk > 0);
          umma_commit(empty + st);
          if (++st == NS) st = 0, ++round;
        }
        umma_commit(acc_full + b);
      }
      // what was issued is done before TMEM goes back
      for (int k = max(0, n_item - 2); k < n_item; ++k) {
        volatile int no_abort = 0;
        mbar_wait(acc_full + (k & 1), (k >> 1) & 1, &no_abort, nullptr, 95);
      }
    }
  } else {
    // =================== epilogue: thread = weight row = TMEM lane ===================
    float* xs = reinterpret_cast<float*>(sm + lay.exchange);        // [2][16][rows]
    T* act = reinterpret_cast<T*>(static_cast<uint8_t*>(a.workspace) + buf.act);
    T* sact = reinterpret_cast<T*>(static_cast<uint8_t*>(a.workspace) + buf.sact);
    float* part = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + buf.part);
    int n_item = 0;
    for (int i = blockIdx.x; i < tiles.total; i += gridDim.x, ++n_item) {
      const Item it = tiles.at(i);
      const int b = n_item & 1;
      bool ok = mbar_wait_warp(acc_full + b, (n_item >> 1) & 1, abort_flag, derr, 96);
      if (!DOWN) ok = all_warps(ok);              // none goes on to an exchange that another has left
      if (!ok) break;
      tc_fence_after();
      const uint32_t tm = tmem + b * cols + ((uint32_t)(warp * 32) << 16);
      if (DOWN) {
        // 16 tokens at a time: columns of the first parts, then of the second
        for (int c0 = 0; c0 < it.n; c0 += 16) {
          float v[32];
          tmem_ld32f(tm + 2 * c0, v);
          tmem_ld_wait();
          if (c0 + 16 >= it.n) {
            tc_fence_before();
            mbar_arrive(acc_empty + b);
          }
          const int h = it.mt * kTile + warp * 32 + lane;
          if (h < a.hidden)
#pragma unroll
            for (int c = 0; c < 16; ++c)
              if (c0 + c < it.n) {
                const int at = it.first + c0 + c;
                const int64_t row = it.shared ? (int64_t)picks * cut.splits + (int64_t)at * cut.shared_splits + it.part
                                              : (int64_t)list[at] * cut.splits + it.part;
                __stcg(part + row * a.hidden + h, fmaf(v[16 + c], 1.0f / kLow<T>, v[c]));
              }
        }
      } else {
        // 16 columns at a time are exchanged, so that a thread has g and u of a row
        const int r = warp * 32 + lane, which = r >= cut.rows, f = r - which * cut.rows;
        const int width = it.shared ? a.shared_ffn : a.ffn;
        const int64_t rows = it.shared ? a.tokens : picks;
        T* out = it.shared ? sact : act;
        const bool all = !it.shared && a.tokens <= 16;              // columns are the tokens, not the picks
        const int step = kTile / cut.rows, q0 = tid / cut.rows, fc = tid - q0 * cut.rows, col = it.mt * cut.rows + fc;
        for (int c0 = 0; c0 < it.n; c0 += 16) {
          float v[16];
          tmem_ld16f(tm + c0, v);
          tmem_ld_wait();
          const bool end = all || c0 + 16 >= it.n;
          if (end) {
            tc_fence_before();
            mbar_arrive(acc_empty + b);
          }
          if (c0) asm volatile("bar.sync 1, 128;" ::: "memory");    // the last exchange has been read
          if (f < cut.rows)
#pragma unroll
            for (int c = 0; c < 16; ++c) xs[(which * 16 + c) * 64 + f] = v[c];
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (q0 < step && col < width)
            for (int q = c0 + q0; q < it.n && (all || q < c0 + 16); q += step) {
              const int at = it.first + q, n = all ? list[at] / a.topk : q - c0;
              const float x = silu(xs[n * 64 + fc]) * xs[(16 + n) * 64 + fc];
              const T h = (T)x;
              out[(int64_t)at * width + col] = h;
              // (beyond the type's range: infinite, and no infinity less infinity)
              out[(rows + at) * width + col] = isinf((float)h) ? (T)0.0f : (T)((x - (float)h) * kLow<T>);
            }
          if (end) break;
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) tmem_dealloc(tmem, 2 * cols);
}

// ---------------------------------------------------------------------------
// the sum: a CTA per 128 columns of a token, its warps take the parts in turn (little code
// and few loads one after the other: 2 us; a thread for all parts of its columns took 5)
// ---------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) moe_combine_kernel(const DashMoeArgs a, const Cut cut, const Buffers buf) {
  __shared__ float4 sum[8][32];
  const int t = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = ((int)blockIdx.x * 32 + lane) * 4;
  const float* part = reinterpret_cast<const float*>(static_cast<const uint8_t*>(a.workspace) + buf.part);
  const int routed = a.topk * cut.splits, total = routed + cut.shared_splits;
  wait_previous();
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (h < a.hidden)
#pragma unroll 4
    for (int i = warp; i < total; i += 8) {
      const int64_t row = i < routed ? (int64_t)t * routed + i : (int64_t)a.tokens * routed + (int64_t)t * cut.shared_splits + i - routed;
      const float4 p = __ldcg(reinterpret_cast<const float4*>(part + row * a.hidden + h));
      const float w = i < routed ? __ldcg(a.weights + (int64_t)t * a.topk + i / cut.splits) : 1.0f;
      s.x = fmaf(w, p.x, s.x), s.y = fmaf(w, p.y, s.y), s.z = fmaf(w, p.z, s.z), s.w = fmaf(w, p.w, s.w);
    }
  sum[warp][lane] = s;
  __syncthreads();
  if (warp || h >= a.hidden) return;
  s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (a.residual) {
    const uint2 r = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.residual) + t * a.residual_stride + h);
    const float2 x = unpack2(r.x, (T*)nullptr), y = unpack2(r.y, (T*)nullptr);
    s = make_float4(x.x, x.y, y.x, y.y);
  }
#pragma unroll
  for (int w = 0; w < 8; ++w) {
    const float4 p = sum[w][lane];
    s.x += p.x, s.y += p.y, s.z += p.z, s.w += p.w;
  }
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + t * a.out_stride + h) =
      make_uint2(pack2(s.x, s.y, (T*)nullptr), pack2(s.z, s.w, (T*)nullptr));
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// [outer, planes, rows, cols] of 16-bit numbers, packed behind rows of `stride`; boxes of 64 columns (128-byte
// swizzle), box_rows rows and box_planes planes.  box_rows 1: a plain [rows, cols] whose rows are gathered
int encode(CUtensorMap* m, const void* p, bool bf16, int64_t cols, int64_t rows, int64_t stride, int64_t planes, int64_t outer,
           int box_rows, int box_planes) {
  const auto fn = encoder();
  if (!fn) return set_error(DASH_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
  const cuuint64_t dims[4] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes, (cuuint64_t)outer};
  const cuuint64_t strides[3] = {(cuuint64_t)stride * 2, (cuuint64_t)(stride * rows) * 2, (cuuint64_t)(stride * rows * planes) * 2};
  const cuuint32_t box[4] = {kStep, (cuuint32_t)box_rows, (cuuint32_t)box_planes, 1}, one[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, box_rows == 1 ? 2 : 4,
                        const_cast<void*>(p), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? DASH_OK : set_error(DASH_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

template <typename... P, typename... A>
int launch(const char* name, void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool early, int cluster, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  if (early) {
    at[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    at[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    at[cfg.numAttrs].val.clusterDim.x = (unsigned)cluster;
    at[cfg.numAttrs].val.clusterDim.y = at[cfg.numAttrs].val.clusterDim.z = 1;
    ++cfg.numAttrs;
  }
  cfg.attrs = at;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
  if (e != cudaSuccess) return set_error(DASH_ERR_CUDA, "%s launch failed: %s", name, cudaGetErrorString(e));
  count_launch();
  return check_launch(name);
}

template <typename T>
int launch_moe_t(const DashMoeArgs& a, cudaStream_t st) {
  constexpr bool kBf16 = DType<T>::fmt == 1;
  const Cut cut = cut_of(a);
  const Buffers buf = buffers_of(a, cut);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  const int64_t picks = (int64_t)a.tokens * a.topk;
  static std::atomic<uint64_t> done{0};
  const cudaError_t set = once_per_device(done, [] {
    cudaError_t e = cudaSuccess;
    for (const auto k : {moe_ffn_kernel<T, false>, moe_ffn_kernel<T, true>}) {
      if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
      // three CTAs, this kernel's or the next one's
      if (e == cudaSuccess) e = cudaFuncSetAttribute(k, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    }
    return e;
  });
  if (set != cudaSuccess) return set_error(DASH_ERR_CUDA, "moe_ffn_kernel: %s", cudaGetErrorString(set));
  Maps up, down;
  const int64_t xs = a.tokens > 1 ? a.x_stride : a.hidden;
  // an expert's gate rows and up rows are two planes of one box
  int rc = encode(&up.w, a.gate_up, kBf16, a.hidden, a.ffn, a.hidden, 2, a.experts, cut.rows, 2);
  if (!rc) rc = encode(&up.b, a.x, kBf16, a.hidden, a.tokens, xs, 1, 1, 1, 1);
  if (!rc) rc = encode(&up.sb, a.x, kBf16, a.hidden, a.tokens, xs, 1, 1, 16, 1);
  up.sw = up.w;
  if (!rc) rc = encode(&down.w, a.down, kBf16, a.ffn, a.hidden, a.ffn, a.experts, 1, kTile, 1);
  if (!rc) rc = encode(&down.b, ws + buf.act, kBf16, a.ffn, picks, a.ffn, 2, 1, 16, 2);
  down.sw = down.w, down.sb = down.b;
  if (a.shared_ffn) {
    if (!rc) rc = encode(&up.sw, a.shared_gate_up, kBf16, a.hidden, a.shared_ffn, a.hidden, 2, 1, cut.rows, 2);
    if (!rc) rc = encode(&down.sw, a.shared_down, kBf16, a.shared_ffn, a.hidden, a.shared_ffn, 1, 1, kTile, 1);
    if (!rc) rc = encode(&down.sb, ws + buf.sact, kBf16, a.shared_ffn, a.tokens, a.shared_ffn, 2, 1, 16, 2);
  }
  if (rc) return rc;
  int cluster = 8;
  while (cluster > 1 && a.experts <= 4 * cluster) cluster >>= 1;
  rc = launch("moe_route_kernel", a.gate_f32 ? moe_route_kernel<T, true> : moe_route_kernel<T, false>, dim3((unsigned)(a.tokens * cluster)), kRouteThreads, 0, st, false, cluster, a);
  const Layout lu = layout_of<false>(cut.nt, cut.rows, a.experts, (int)picks),
               ld = layout_of<true>(cut.nt, cut.rows, a.experts, (int)picks);
  if (!rc) rc = launch("moe_up_kernel", moe_ffn_kernel<T, false>, dim3(kCtas), kThreads, lu.bytes, st, true, 1, up, a, cut, buf);
  if (!rc) rc = launch("moe_down_kernel", moe_ffn_kernel<T, true>, dim3(kCtas), kThreads, ld.bytes, st, true, 1, down, a, cut, buf);
  const dim3 grid((unsigned)ceil_div(a.hidden, 128), (unsigned)a.tokens);
  if (!rc) rc = launch("moe_combine_kernel", moe_combine_kernel<T>, grid, 256, 0, st, true, 1, a, cut, buf);
  return rc;
}

}  // namespace

size_t moe_workspace(const DashMoeArgs& a) { return buffers_of(a, cut_of(a)).bytes; }

int launch_moe(const DashMoeArgs& a, cudaStream_t st) {
  return a.dtype == DASH_DTYPE_BF16 ? launch_moe_t<__nv_bfloat16>(a, st) : launch_moe_t<__half>(a, st);
}

}  // namespace dash
