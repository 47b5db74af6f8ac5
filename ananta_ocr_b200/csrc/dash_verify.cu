// dash_verify.cu -- verification of drafted tokens (speculative sampling over a
// tree, or greedy matching) and the next token.
//
// A cluster of CTAs takes a sequence; each CTA owns a contiguous slice of the
// vocabulary and each warp a contiguous part of the slice, so running sums
// follow the vocabulary's order.  Every CTA walks the drafted tokens with the
// same numbers (the probabilities of the drafted tokens themselves are
// gathered once, at the start); only the sums over the vocabulary are shared,
// by reads of the other CTAs' shared memory.
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
#include <cooperative_groups.h>
#include "dash_tree.cuh"

namespace cg = cooperative_groups;

namespace dash {
namespace {

constexpr int kVerThreads = 512;
constexpr int kVerWarps = kVerThreads / 32;
constexpr int kVerNodes = 256;
constexpr int kVerMaxCluster = 8;

struct VerSmem {
  int par[kVerNodes];
  int64_t tok[kVerNodes];
  float pv[kVerNodes], qv[kVerNodes], ua[kVerNodes];
  int rejected[kVerNodes];
  int path[kVerNodes];
  // sums (or argmax keys) of this CTA's warps, two buffers: a pass writes one
  // while a slower CTA may still read the other
  double sum[2][kVerWarps];
  unsigned long long key[2];
  unsigned long long wkey[kVerWarps];
};

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

template <typename T, int E>
struct Vec { T v[E]; };

// element i of the row as stored, E at a time
template <typename T, int E>
__device__ __forceinline__ void load_e(const T* row, int64_t i, float (&x)[E]) {
  if constexpr (E == 1) {
    x[0] = to_f(row[i]);
  } else {
    union { uint4 u; Vec<T, E> t; } w;
    w.u = __ldg(reinterpret_cast<const uint4*>(row + i));
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = to_f(w.t.v[e]);
  }
}

// order-preserving image of a float: NaN above everything, -0 equal to +0
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  x += 0.0f;
  const uint32_t u = __float_as_uint(x);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

}  // namespace

// E elements per load: 16 bytes where every row starts on 16 bytes, else 1.
template <typename T, int E>
__global__ void __launch_bounds__(kVerThreads) verify_kernel(const __grid_constant__ DashVerifyArgs a) {
  __shared__ VerSmem S;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int s = blockIdx.x / C;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int r0 = a.q_start[s];
  const int n = max(0, min(min(a.q_start[s + 1], a.rows) - r0, a.max_nodes));
  if (tid == 0 && rank == 0 && a.q_start[s + 1] - r0 > a.max_nodes)
    record_error(a.device_error, DASH_DEV_BAD_TREE, 80, a.q_start[s + 1] - r0);
  const T* target = reinterpret_cast<const T*>(a.target);
  const T* draft = reinterpret_cast<const T*>(a.draft);
  const int V = a.vocab;
  for (int i = tid; i < n; i += kVerThreads) {
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
      S.qv[i] = a.mode == 0 ? to_f(draft[(int64_t)(r0 + p) * a.draft_stride + x]) : 0.0f;
      S.ua[i] = a.mode < 2 ? a.u_accept[r0 + i] : 0.0f;
    }
  }
  __syncthreads();

  // this warp's part of the vocabulary: whole groups of 32 E elements
  constexpr int STEP = 32 * E;
  const int64_t parts = (int64_t)C * kVerWarps;
  const int64_t per = ((V + parts - 1) / parts + STEP - 1) / STEP * STEP;
  const int64_t v0 = min((int64_t)V, (rank * kVerWarps + warp) * per), v1 = min((int64_t)V, v0 + per);

  int cur = 0, kept = 0, n_rej = 0, pass = 0;
  double c = 0.0, W = 1.0;
  // the residual of element v (probabilities as stored, 64-bit arithmetic)
  auto residual = [&](int64_t v, float p, float q, int rej) -> double {
    double r = (double)p;
    if (a.mode == 0) {
      r = __dsub_rn(r, __dmul_rn(c, (double)q));
    } else {
      for (int k = 0; k < rej; ++k)
        if (S.rejected[k] == (int)v) r = 0.0;
    }
    return r > 0.0 ? r : 0.0;
  };
  // sums of the residual over every warp's part -> S.sum of all CTAs
  auto vocab_sum = [&](int rej) {
    const T* pr = target + (int64_t)(r0 + cur) * a.target_stride;
    const T* qr = a.mode == 0 ? draft + (int64_t)(r0 + cur) * a.draft_stride : pr;
    const bool two = a.mode == 0 && c != 0.0;
    double acc = 0.0;
    for (int64_t v = v0 + lane * E; v < v1; v += STEP) {
      float p[E], q[E];
      if (E == 1 || v + E <= v1) {
        load_e<T, E>(pr, v, p);
        if (two) load_e<T, E>(qr, v, q);
#pragma unroll
        for (int e = 0; e < E; ++e) acc += residual(v + e, p[e], two ? q[e] : 0.0f, rej);
      } else {
        for (int e = 0; v + e < v1; ++e)
          acc += residual(v + e, to_f(pr[v + e]), two ? to_f(qr[v + e]) : 0.0f, rej);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) S.sum[pass & 1][warp] = acc;
    cluster.sync();
  };
  auto total = [&]() -> double {       // every thread: all parts in vocabulary order
    double t = 0.0;
    for (int r = 0; r < C; ++r) {
      const double* ps = cluster.map_shared_rank(&S.sum[pass & 1][0], r);
      for (int w = 0; w < kVerWarps; ++w) t += ps[w];
    }
    return t;
  };
  auto row_argmax = [&]() -> int {
    const T* pr = target + (int64_t)(r0 + cur) * a.target_stride;
    unsigned long long best = 0;
    auto see = [&](float x, int64_t v) {
      const unsigned long long k = ((unsigned long long)order_key(x) << 32) | (0xffffffffu - (uint32_t)v);
      best = k > best ? k : best;
    };
    for (int64_t v = v0 + lane * E; v < v1; v += STEP) {
      if (E == 1 || v + E <= v1) {
        float p[E];
        load_e<T, E>(pr, v, p);
#pragma unroll
        for (int e = 0; e < E; ++e) see(p[e], v + e);
      } else {
        for (int e = 0; v + e < v1; ++e) see(to_f(pr[v + e]), v + e);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, best, o);
      best = k > best ? k : best;
    }
    if (lane == 0) S.wkey[warp] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kVerWarps; ++w) best = S.wkey[w] > best ? S.wkey[w] : best;
      S.key[pass & 1] = best;
    }
    cluster.sync();
    best = 0;
    for (int r = 0; r < C; ++r) {
      const unsigned long long k = *cluster.map_shared_rank(&S.key[pass & 1], r);
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
    if (a.mode == 2) {
      if (arg < 0) arg = row_argmax();
      take = x == arg;
    } else if (a.mode == 0) {
      if (!fresh) {
        vocab_sum(0);
        W = total();
        ++pass;
        fresh = true;
      }
      const double q = S.qv[i], p = S.pv[i];
      take = (double)S.ua[i] * W * q < __dsub_rn(p, __dmul_rn(c, q));
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
  if (n > 0 && a.mode == 2) {
    if (arg < 0) arg = row_argmax();
    if (rank == 0 && tid == 0) {
      a.next_token[s] = arg;
      out[kept] = arg;
    }
  } else if (n > 0) {
    vocab_sum(n_rej);
    double t = total();
    if (!(t > 0.0)) {                  // empty residual: the row itself
      ++pass;
      c = 0.0;
      n_rej = 0;
      vocab_sum(0);
      t = total();
    }
    const double at = (double)a.u_sample[s] * t;
    // the warp whose part holds the place: the first whose running sum
    // passes it (rounding can leave none: then the last one with any mass)
    int hit = -1, last = -1;
    double before = 0.0, hit_before = 0.0, last_before = 0.0;
    for (int r = 0; r < C; ++r) {
      const double* ps = cluster.map_shared_rank(&S.sum[pass & 1][0], r);
      for (int w = 0; w < kVerWarps; ++w) {
        const double x = ps[w];
        if (x > 0.0) {
          last = r * kVerWarps + w;
          last_before = before;
          if (hit < 0 && before + x > at) { hit = last; hit_before = before; }
        }
        before += x;
      }
    }
    if (hit < 0) { hit = last; hit_before = last_before; }
    if (hit < 0) {
      if (rank == 0 && tid == 0) { a.next_token[s] = -1; out[kept] = -1; }
    } else if (hit == rank * kVerWarps + warp) {
      const T* pr = target + (int64_t)(r0 + cur) * a.target_stride;
      const T* qr = a.mode == 0 ? draft + (int64_t)(r0 + cur) * a.draft_stride : pr;
      double run = hit_before;
      int64_t found = -1, some = -1;   // the place, the last element with mass
      for (int64_t v = v0; v < v1 && found < 0; v += STEP) {
        double x[E], mine = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int64_t i = v + lane * E + e;
          x[e] = i < v1 ? residual(i, to_f(pr[i]), to_f(qr[i]), n_rej) : 0.0;
          mine += x[e];
        }
        double incl = mine;            // running sum over the lanes
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        double b = run + (incl - mine);
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
  if (rank == 0) {
    __syncthreads();
    if (tid == 0) {
      a.n_accept[s] = kept;
      if (n == 0) a.next_token[s] = -1;
    }
    for (int i = tid; i < a.max_nodes; i += kVerThreads) {
      a.path[(int64_t)s * a.max_nodes + i] = i < n && i <= kept ? S.path[i] : -1;
      if (n > 0 && i < kept) out[i] = S.tok[S.path[i + 1]];
      else if (n == 0 || i > kept) out[i] = -1;
    }
  }
  cluster.sync();                      // no CTA leaves while another reads its sums
}

template <typename T, int E>
static int launch_verify_t(const DashVerifyArgs& a, cudaStream_t st) {
  // enough CTAs to fill the GPU; one cluster of 8 reads a row of 10^5 fp32
  // probabilities in 16 parts of 8 KB per CTA
  int C = kVerMaxCluster;
  while (C > 1 && (a.n_seq * (C / 2) >= 592 || a.vocab <= 32 * E * kVerWarps * (C / 2))) C >>= 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.n_seq * C));
  cfg.blockDim = dim3(kVerThreads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<T, E>, a);
  if (e != cudaSuccess) return set_error(DASH_ERR_CUDA, "verify_kernel launch failed: %s", cudaGetErrorString(e));
  count_launch();
  return check_launch("verify_kernel");
}

template <typename T>
static int launch_verify_e(const DashVerifyArgs& a, cudaStream_t st) {
  constexpr int E = 16 / sizeof(T);
  const bool vec = (reinterpret_cast<uintptr_t>(a.target) & 15) == 0 && a.target_stride % E == 0 &&
                   (a.mode != 0 || ((reinterpret_cast<uintptr_t>(a.draft) & 15) == 0 && a.draft_stride % E == 0));
  return vec ? launch_verify_t<T, E>(a, st) : launch_verify_t<T, 1>(a, st);
}

int launch_verify(const DashVerifyArgs& a, cudaStream_t st) {
  if (a.dtype == DASH_DTYPE_F32) return launch_verify_e<float>(a, st);
  if (a.dtype == DASH_DTYPE_BF16) return launch_verify_e<__nv_bfloat16>(a, st);
  return launch_verify_e<__half>(a, st);
}

}  // namespace dash
