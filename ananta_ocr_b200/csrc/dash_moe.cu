// dash_moe.cu -- a whole mixture-of-experts layer for a few tokens.
//
// Four kernels: the router (scores exact to 64 bits, the picks, their weights), gate_up
// and SwiGLU of every pick and of the shared expert, down, and the weighted sum in the
// picks' order.  Bound by the weights of the experts that the tokens picked.
#include "dash_common.cuh"
#include "dash_internal.h"

namespace dash {

namespace {

template <typename T>
__device__ __forceinline__ float load(const void* p, int64_t i) { return (float)static_cast<const T*>(p)[i]; }

// one CTA per token
template <typename T>
__global__ void __launch_bounds__(256) moe_route_kernel(const DashMoeArgs a) {
  __shared__ double score[kMoeMaxExperts];
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = warp; e < a.experts; e += 8) {
    double s = 0.0;
    for (int i = lane; i < a.hidden; i += 32) {
      const double g = a.gate_f32 ? (double)static_cast<const float*>(a.gate)[(int64_t)e * a.hidden + i]
                                  : (double)load<T>(a.gate, (int64_t)e * a.hidden + i);
      s = fma((double)load<T>(a.x, t * a.x_stride + i), g, s);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) score[e] = s;
  }
  __syncthreads();
  if (warp) return;
  double top = -INFINITY, sum = 0.0;
  for (int e = 0; e < a.experts; ++e) top = fmax(top, score[e]);
  for (int e = lane; e < a.experts; e += 32) sum += exp(score[e] - top);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  double mine = 0.0, picked = 0.0;
  int id = 0;
  uint32_t used = 0;                         // this lane's experts that are taken
  for (int j = 0; j < a.topk; ++j) {
    double best = 0.0;
    int at = -1;
    for (int e = lane, i = 0; e < a.experts; e += 32, ++i) {
      const double s = score[e] == score[e] ? score[e] : -INFINITY;
      if (!(used >> i & 1u) && (at < 0 || s > best)) best = s, at = e;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const double s = __shfl_xor_sync(0xffffffffu, best, o);
      const int e = __shfl_xor_sync(0xffffffffu, at, o);
      if (e >= 0 && (at < 0 || s > best || (s == best && e < at))) best = s, at = e;
    }
    if ((at & 31) == lane) used |= 1u << (at >> 5);
    const double p = exp(score[at] - top) / sum;
    if (lane == j) mine = p, id = at;
    picked += p;
  }
  if (lane < a.topk) {
    a.ids[t * a.topk + lane] = id;
    a.weights[t * a.topk + lane] = (float)(mine / (a.renorm ? picked : 1.0) * (double)a.scale);
  }
}

// act[row][f]: a warp per feature; rows: the picks, then the tokens' shared expert
template <typename T>
__global__ void __launch_bounds__(256) moe_up_kernel(const DashMoeArgs a, float* act) {
  const int lane = threadIdx.x & 31;
  const int64_t picks = (int64_t)a.tokens * a.topk;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const bool shared = w >= picks * a.ffn;
  const int64_t v = shared ? w - picks * a.ffn : w;
  const int n = shared ? a.shared_ffn : a.ffn;
  if (n == 0 || v >= (shared ? (int64_t)a.tokens : picks) * n) return;
  const int64_t r = v / n;
  const int f = (int)(v % n);
  const int64_t t = shared ? r : r / a.topk;
  const T* g = shared ? static_cast<const T*>(a.shared_gate_up)
                      : static_cast<const T*>(a.gate_up) + (int64_t)a.ids[r] * 2 * a.ffn * a.hidden;
  float x = 0.0f, y = 0.0f;
  for (int i = lane; i < a.hidden; i += 32) {
    const float h = load<T>(a.x, t * a.x_stride + i);
    x = fmaf(h, (float)g[(int64_t)f * a.hidden + i], x);
    y = fmaf(h, (float)g[(int64_t)(n + f) * a.hidden + i], y);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o), y += __shfl_xor_sync(0xffffffffu, y, o);
  if (lane == 0) act[w] = x / (1.0f + expf(-x)) * y;
}

// out: a warp per (token, feature)
template <typename T>
__global__ void __launch_bounds__(256) moe_down_kernel(const DashMoeArgs a, const float* act) {
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (w >= (int64_t)a.tokens * a.hidden) return;
  const int64_t t = w / a.hidden, h = w % a.hidden;
  float s = a.residual ? load<T>(a.residual, t * a.residual_stride + h) : 0.0f;
  for (int j = 0; j <= a.topk; ++j) {
    const bool shared = j == a.topk;
    const int n = shared ? a.shared_ffn : a.ffn;
    const int64_t r = t * a.topk + j;
    const float* x = shared ? act + (int64_t)a.tokens * a.topk * a.ffn + t * n : act + r * n;
    const T* d = shared ? static_cast<const T*>(a.shared_down)
                        : static_cast<const T*>(a.down) + (int64_t)a.ids[r] * a.hidden * n;
    float y = 0.0f;
    for (int i = lane; i < n; i += 32) y = fmaf(x[i], (float)d[h * n + i], y);
#pragma unroll
    for (int o = 16; o; o >>= 1) y += __shfl_xor_sync(0xffffffffu, y, o);
    if (n) s = fmaf(y, shared ? 1.0f : a.weights[r], s);
  }
  if (lane == 0) static_cast<T*>(a.out)[t * a.out_stride + h] = (T)s;
}

template <typename T>
int launch_moe_t(const DashMoeArgs& a, cudaStream_t st) {
  float* act = static_cast<float*>(a.workspace);
  moe_route_kernel<T><<<a.tokens, 256, 0, st>>>(a);
  const int64_t rows = (int64_t)a.tokens * ((int64_t)a.topk * a.ffn + a.shared_ffn);
  moe_up_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(a, act);
  moe_down_kernel<T><<<(unsigned)(((int64_t)a.tokens * a.hidden + 7) / 8), 256, 0, st>>>(a, act);
  for (int i = 0; i < 3; ++i) count_launch();
  return check_launch("moe kernels");
}

}  // namespace

size_t moe_workspace(const DashMoeArgs& a) {
  return (size_t)a.tokens * ((size_t)a.topk * a.ffn + a.shared_ffn) * sizeof(float) + 16;
}

int launch_moe(const DashMoeArgs& a, cudaStream_t st) {
  return a.dtype == DASH_DTYPE_BF16 ? launch_moe_t<__nv_bfloat16>(a, st) : launch_moe_t<__half>(a, st);
}

}  // namespace dash
