// dash_verify.cu -- verification of drafted tokens (speculative sampling over a
// tree, or greedy matching) and the next token.
//
// A cluster of CTAs takes a sequence; each CTA owns a contiguous slice of the
// vocabulary and each warp a contiguous part of the slice, so running sums
// follow the vocabulary's order.  Every CTA walks the drafted tokens with the
// same numbers (the probabilities of the drafted tokens themselves are
// gathered once, at the start); only a sum per CTA is shared, written into the
// other CTAs' shared memory.  A pass over a row is bound by latency (a few
// microseconds for 1 MB of two fp32 rows by 8 CTAs), so each warp has
// kVerUnroll loads per row in flight, and with many sequences four CTAs of 256
// threads share an SM.
//
// Residuals: with c_0 = 0, W_0 = 1 the residual after k rejections among the
// children of a row is R_k = max(p - c_k q, 0) / W_k, because
//   R_{k+1} ~ max(R_k - q, 0) = max(p - (c_k + W_k) q, 0) / W_k   (q >= 0)
// so c_{k+1} = c_k + W_k and W_{k+1} = sum max(p - c_{k+1} q, 0): one pass over
// the row per rejection that is followed by another child, none for an
// acceptance, and one for the token drawn at the end (its part of the row is
// read again to find the place).  All sums are 64-bit: a 32-bit running sum
// over a vocabulary of 10^5 moves the borders between tokens by more than a rare
// token's probability.
//
// Measured (CUDA graph, vocabulary 129,280): 64 sequences of 16 fp32 rows, drawn
// drafts, 33 us.  By the global timer: set-up 2.3; a first pass that all 512 CTAs
// make at once, at memory rate, to 10-14 (66 MB), its exchange to 16; a second by
// half of the sequences to 24 and a third by a third of them to 30; the search for
// the token's place 0.7, and up to 10 where many CTAs still read.  One sequence of 4
// rows 12.4 us, greedy 16 of 8 18.6 us (up to four passes of 3-4 us, one after the
// other).  Certain drafts 18.5 us (1 x 4) and 43 (64 x 16): one pass, in which every
// element is compared with the rejected tokens.
#include <cooperative_groups.h>
#include "dash_tree.cuh"

namespace cg = cooperative_groups;

namespace dash {
namespace {

constexpr int kVerThreads = 512;
constexpr int kVerWarps = kVerThreads / 32;      // at most
constexpr int kVerNodes = 256;
constexpr int kVerMaxCluster = 8;
constexpr int kVerUnroll = 4;

struct VerSmem {
  int par[kVerNodes];
  int64_t tok[kVerNodes];
  float pv[kVerNodes], qv[kVerNodes], ua[kVerNodes];
  int rejected[kVerNodes];
  int path[kVerNodes];
  double part[kVerWarps];                        // this CTA's sums, by warp
  unsigned long long wkey[kVerWarps];
  // what every CTA of the cluster wrote here (sums or argmax keys), two
  // buffers: a pass fills one while a slower CTA may still read the other
  double sum[2][kVerMaxCluster];
  unsigned long long key[2][kVerMaxCluster];
};

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

// E consecutive elements as they are stored: 16 bytes, or one element
template <typename T, int E>
struct Raw {
  uint4 u;
  __device__ __forceinline__ void load(const T* p) { u = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ float at(int e) const {
    union { uint4 u; T t[E]; } w;
    w.u = u;
    return to_f(w.t[e]);
  }
};
template <typename T>
struct Raw<T, 1> {
  T t;
  __device__ __forceinline__ void load(const T* p) { t = *p; }
  __device__ __forceinline__ float at(int) const { return to_f(t); }
};

// order-preserving image of a float: NaN above everything, -0 equal to +0
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  x += 0.0f;
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

}  // namespace

// E elements per load: 16 bytes where every row starts on 16 bytes, else 1.
template <typename T, int E, int MODE>
__global__ void __launch_bounds__(kVerThreads, 2) verify_kernel(const __grid_constant__ DashVerifyArgs a) {
  __shared__ VerSmem S;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int s = blockIdx.x / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, warps = blockDim.x >> 5;
  // the other CTAs' shared memory is written once they run: waited for in the first pass
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int r0 = a.q_start[s];
  const int n = r0 < 0 ? 0 : max(0, min(min(a.q_start[s + 1], a.rows) - r0, a.max_nodes));
  if (tid == 0 && rank == 0 && a.q_start[s + 1] - r0 > a.max_nodes)
    record_error(a.device_error, DASH_DEV_BAD_TREE, 80, a.q_start[s + 1] - r0);
  const T* target = reinterpret_cast<const T*>(a.target);
  const T* draft = reinterpret_cast<const T*>(a.draft);
  const int V = a.vocab;
  for (int i = tid; i < n; i += blockDim.x) {
    int p = a.parents ? a.parents[r0 + i] : i - 1;
    if (i == 0) p = -1;
    if (i > 0 && (p < 0 || p >= i)) {
      if (rank == 0) record_error(a.device_error, DASH_DEV_BAD_TREE, 81, p);
      p = -1;
    }
    const int64_t x = a.tokens[r0 + i];
    const bool in = x >= 0 && x < V;
    S.par[i] = in ? p : -1;
    S.tok[i] = x;
    if (in && p >= 0) {
      S.pv[i] = to_f(target[(int64_t)(r0 + p) * a.target_stride + x]);
      S.qv[i] = MODE == 0 ? to_f(draft[(int64_t)(r0 + p) * a.draft_stride + x]) : 0.0f;
      S.ua[i] = MODE < 2 ? a.u_accept[r0 + i] : 0.0f;
    }
  }
  __syncthreads();

  // this warp's part of the vocabulary: whole groups of 32 E elements
  constexpr int STEP = 32 * E;
  const int64_t parts = (int64_t)C * warps;
  const int64_t per = ((V + parts - 1) / parts + STEP - 1) / STEP * STEP;
  const int64_t v0 = min((int64_t)V, (rank * warps + warp) * per), v1 = min((int64_t)V, v0 + per);

  int cur = 0, kept = 0, n_rej = 0, pass = 0;
  auto wait_started = [&]() {
    if (pass == 0) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  };
  double c = 0.0, W = 1.0;
  // the residual of element v (probabilities as stored, 64-bit arithmetic)
  auto residual = [&](int64_t v, double r, double q, int rej) -> double {
    if constexpr (MODE == 0) {
      r = fma(-c, q, r);
    } else {
      for (int k = 0; k < rej; ++k)
        if (S.rejected[k] == (int)v) r = 0.0;
    }
    return r > 0.0 ? r : 0.0;
  };
  // f(v, p, q) for the elements of this warp's part, lane by lane, kVerUnroll
  // loads of a row in flight
  auto scan_part = [&](const T* pr, const T* qr, bool two, auto f) {
    int64_t v = v0 + lane * E;
    for (; v + (kVerUnroll - 1) * STEP + E <= v1; v += kVerUnroll * STEP) {
      Raw<T, E> p[kVerUnroll], q[kVerUnroll];
#pragma unroll
      for (int k = 0; k < kVerUnroll; ++k) p[k].load(pr + v + k * STEP);
      if (two) {
#pragma unroll
        for (int k = 0; k < kVerUnroll; ++k) q[k].load(qr + v + k * STEP);
      }
#pragma unroll
      for (int k = 0; k < kVerUnroll; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) f(v + k * STEP + e, p[k].at(e), two ? q[k].at(e) : 0.0f);
    }
#pragma unroll 1
    for (; v + E <= v1; v += STEP) {
      Raw<T, E> p, q;
      p.load(pr + v);
      if (two) q.load(qr + v);
#pragma unroll
      for (int e = 0; e < E; ++e) f(v + e, p.at(e), two ? q.at(e) : 0.0f);
    }
#pragma unroll 1
    for (int e = 0; e < E && v + e < v1; ++e) f(v + e, to_f(pr[v + e]), two ? to_f(qr[v + e]) : 0.0f);
  };
  // the residual's sum: S.part of this CTA's warps, S.sum of every CTA; returns all
  auto vocab_sum = [&](int rej) -> double {
    const T* pr = target + (int64_t)(r0 + cur) * a.target_stride;
    const bool two = MODE == 0 && c != 0.0;
    double acc = 0.0;
    scan_part(pr, two ? draft + (int64_t)(r0 + cur) * a.draft_stride : pr, two,
              [&](int64_t v, float p, float q) { acc += residual(v, p, q, rej); });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) S.part[warp] = acc;
    wait_started();
    __syncthreads();
    if (warp == 0 && lane < C) {
      double t = 0.0;
      for (int w = 0; w < warps; ++w) t += S.part[w];
      *cluster.map_shared_rank(&S.sum[pass & 1][rank], lane) = t;
    }
    cluster.sync();
    double t = 0.0;
    for (int r = 0; r < C; ++r) t += S.sum[pass & 1][r];
    ++pass;
    return t;
  };
  auto row_argmax = [&]() -> int {
    const T* pr = target + (int64_t)(r0 + cur) * a.target_stride;
    unsigned long long best = 0;
    scan_part(pr, pr, false, [&](int64_t v, float x, float) {
      const unsigned long long k = ((unsigned long long)order_key(x) << 32) | (0xffffffffu - (uint32_t)v);
      best = k > best ? k : best;
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
      best = k > best ? k : best;
    }
    if (lane == 0) S.wkey[warp] = best;
    wait_started();
    __syncthreads();
    if (warp == 0 && lane < C) {
      best = 0;
      for (int w = 0; w < warps; ++w) best = S.wkey[w] > best ? S.wkey[w] : best;
      *cluster.map_shared_rank(&S.key[pass & 1][rank], lane) = best;
    }
    cluster.sync();
    best = 0;
    for (int r = 0; r < C; ++r) {
      const unsigned long long k = S.key[pass & 1][r];
      best = k > best ? k : best;
    }
    ++pass;
    return (int)(0xffffffffu - (uint32_t)best);
  };

  int arg = -1;                        // mode 2: argmax behind cur, -1 = not known yet
  bool fresh = true;                   // mode 0: W belongs to c
  if (tid == 0) S.path[0] = 0;
  for (int i = 1; i < n; ++i) {
    if (S.par[i] != cur) continue;
    const int x = (int)S.tok[i];
    bool take;
    if (MODE == 2) {
      if (arg < 0) arg = row_argmax();
      take = x == arg;
    } else if (MODE == 0) {
      if (!fresh) {
        W = vocab_sum(0);
        fresh = true;
      }
      const double q = S.qv[i], p = S.pv[i];
      take = (double)S.ua[i] * W * q < fma(-c, q, p);
      if (!take) {
        c += W;
        fresh = false;
      }
    } else {
      bool again = false;
      for (int k = 0; k < n_rej; ++k) again |= S.rejected[k] == x;
      const double p = again ? 0.0 : (double)S.pv[i];
      take = (double)S.ua[i] * W < p;
      if (!take && !again) {
        W -= p;
        __syncthreads();               // rejected is read by all threads above
        if (tid == 0) S.rejected[n_rej] = x;
        ++n_rej;
        __syncthreads();
      }
    }
    if (take) {
      cur = i;
      ++kept;
      if (tid == 0) S.path[kept] = i;
      c = 0.0;
      W = 1.0;
      fresh = true;
      n_rej = 0;
      arg = -1;
    }
  }

  // ---- the next token ----
  int64_t* out = a.out_tokens + (int64_t)s * a.max_nodes;
  if (n > 0 && MODE == 2) {
    if (arg < 0) arg = row_argmax();
    if (rank == 0 && tid == 0) {
      a.next_token[s] = arg;
      out[kept] = arg;
    }
  } else if (n > 0) {
    double t = vocab_sum(n_rej);
    if (!(t > 0.0)) {                  // empty residual: the row itself
      c = 0.0;
      n_rej = 0;
      t = vocab_sum(0);
    }
    const double at = (double)a.u_sample[s] * t;
    // the part that holds the place: the first whose running sum passes it
    // (rounding can leave none: then the last one with any mass); first the
    // CTA, then the warp
    auto find = [&](const double* x, int n, double& before) -> int {
      int hit = -1, last = -1;
      double run = before, last_before = before;
      for (int i = 0; i < n; ++i) {
        if (x[i] > 0.0) {
          last = i;
          last_before = run;
          if (run + x[i] > at) { hit = i; break; }
        }
        run += x[i];
      }
      before = last_before;
      return hit >= 0 ? hit : last;
    };
    double hit_before = 0.0;
    int hit = find(S.sum[(pass - 1) & 1], C, hit_before);
    const bool mine = hit == rank;
    if (mine) hit = find(S.part, warps, hit_before);
    if (hit < 0) {
      if (rank == 0 && tid == 0) { a.next_token[s] = -1; out[kept] = -1; }
    } else if (mine && hit == warp) {
      const T* pr = target + (int64_t)(r0 + cur) * a.target_stride;
      const T* qr = MODE == 0 ? draft + (int64_t)(r0 + cur) * a.draft_stride : pr;
      const bool two = MODE == 0 && c != 0.0;
      double run = hit_before;
      int64_t found = -1, some = -1;   // the place, the last element with mass
      float pn[E], qn[E];              // the next elements, read a step ahead
      auto read = [&](int64_t v) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t i = v + lane * E + e;
          pn[e] = i < v1 ? to_f(pr[i]) : 0.0f;
          qn[e] = two && i < v1 ? to_f(qr[i]) : 0.0f;
        }
      };
      read(v0);
      for (int64_t v = v0; v < v1 && found < 0; v += STEP) {
        double x[E], own = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          x[e] = residual(v + lane * E + e, pn[e], qn[e], n_rej);
          own += x[e];
        }
        if (v + STEP < v1) read(v + STEP);
        double incl = own;             // running sum over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        double b = run + (incl - own);
        int64_t got = -1, any = -1;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          b += x[e];
          if (x[e] > 0.0) {
            any = v + lane * E + e;
            if (got < 0 && b > at) got = any;
          }
        }
        const uint32_t m = __ballot_sync(0xffffffffu, got >= 0), ma = __ballot_sync(0xffffffffu, any >= 0);
        if (ma) some = __shfl_sync(0xffffffffu, any, 31 - __clz(ma));
        if (m) found = __shfl_sync(0xffffffffu, got, __ffs(m) - 1);
        run += __shfl_sync(0xffffffffu, incl, 31);
      }
      if (found < 0) found = some;
      if (lane == 0) {
        a.next_token[s] = found;
        out[kept] = found;
      }
    }
  }
  wait_started();                      // no drafted token, no pass
  if (rank == 0) {
    __syncthreads();
    if (tid == 0) {
      a.n_accept[s] = kept;
      if (n == 0) a.next_token[s] = -1;
    }
    for (int i = tid; i < a.max_nodes; i += blockDim.x) {
      a.path[(int64_t)s * a.max_nodes + i] = i < n && i <= kept ? S.path[i] : -1;
      if (n > 0 && i < kept) out[i] = S.tok[S.path[i + 1]];
      else if (n == 0 || i > kept) out[i] = -1;
    }
  }
  // every write to another CTA's shared memory came before a barrier of the
  // cluster that both have passed
}

template <typename T, int E, int MODE>
static int launch_verify_t(const DashVerifyArgs& a, cudaStream_t st) {
  // Eight CTAs per sequence while that fills the GPU's slots once (four CTAs of 256
  // threads per SM); 512 threads where the GPU is far from full.
  int C = kVerMaxCluster;
  while (C > 1 && (a.n_seq * (C / 2) >= 592 || a.vocab <= 32 * E * (C / 2))) C >>= 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_seq * C));
  cfg.blockDim = dim3(a.n_seq * C <= 148 ? kVerThreads : kVerThreads / 2);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<T, E, MODE>, a);
  if (e != cudaSuccess) return set_error(DASH_ERR_CUDA, "verify_kernel launch failed: %s", cudaGetErrorString(e));
  count_launch();
  return check_launch("verify_kernel");
}

template <typename T>
static int launch_verify_e(const DashVerifyArgs& a, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const bool vec = (reinterpret_cast<uintptr_t>(a.target) & 15) == 0 && a.target_stride % E == 0 &&
                   (a.mode != 0 || ((reinterpret_cast<uintptr_t>(a.draft) & 15) == 0 && a.draft_stride % E == 0));
  if (a.mode == 0) return vec ? launch_verify_t<T, E, 0>(a, st) : launch_verify_t<T, 1, 0>(a, st);
  if (a.mode == 1) return vec ? launch_verify_t<T, E, 1>(a, st) : launch_verify_t<T, 1, 1>(a, st);
  return vec ? launch_verify_t<T, E, 2>(a, st) : launch_verify_t<T, 1, 2>(a, st);
}

int launch_verify(const DashVerifyArgs& a, cudaStream_t st) {
  if (a.dtype == DASH_DTYPE_F32) return launch_verify_e<float>(a, st);
  if (a.dtype == DASH_DTYPE_BF16) return launch_verify_e<__nv_bfloat16>(a, st);
  return launch_verify_e<__half>(a, st);
}

}  // namespace dash
